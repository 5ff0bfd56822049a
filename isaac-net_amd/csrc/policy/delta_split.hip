// The gated delta rule over long windows of few robots (the mathematics: delta.h), where a workgroup a robot and head would
// leave most of the chip idle: what does not need the state is computed for every chunk at once, and only the state goes
// from chunk to chunk.
//
//     before   forward    U = (I + L')^-1 V,            W = -(I + L')^-1 (a K),   f = c beta
//              backward   U = (I + L)^-T P^T dO,        W = (I + L)^-T (c K),     f = -a beta,   G = Q^T (scale a dO)
//     scan     X = U + W S,   S <- a_C S + G + K^T (f X)          (forward: X = E; backward: X = Z, S the gradient's)
//     after    forward    O = scale a Q S + P X;        backward: delta_chunk_kernel
//
// The scan is the only part that is serial: two products a chunk, its operands double-buffered in LDS; it is bound by the
// latency of that chain, the other parts by their own products. 2 robots x 4096 steps x 8 heads of 64 x 64, bfloat16, 64 chunks,
// us: before 25, scan 174 (2.7 a chunk), after 20; backward 46, 198 (3.1 a chunk) and the chunks' gradients 52. In one pass
// the forward takes 607. 4 x 2048 x 8 heads of 128 x 128: 74, 140, 45; 101, 191, 194.
#include "delta.h"
#include "delta_launch.h"

namespace pol {

// the workspace of one direction: W in three planes [robot, head][chunk][3][C][KP], f and the rows' a (forward) or c
// (backward) [robot, head][chunk][2 C + 4] with a_C, and G [robot, head][chunk][K][V]
struct SplitWork {
    __bf16* w;
    float *f, *G;
    static size_t up(size_t x) { return (x + 255) & ~(size_t)255; }
    static int kp(int K) { return K <= 32 ? 32 : K <= 64 ? 64 : 128; }
    static size_t w_bytes(const InetDelta& d, int64_t units) { return up((size_t)units * 3 * d.chunk * kp(d.K) * 2); }
    static size_t f_bytes(const InetDelta& d, int64_t units) { return up((size_t)units * (2 * d.chunk + 4) * 4); }
    static size_t bytes(const InetDelta& d, bool back) {
        const int64_t units = (int64_t)d.B * d.H * ((d.T + d.chunk - 1) / d.chunk);
        return w_bytes(d, units) + f_bytes(d, units) + (back ? up((size_t)units * d.K * d.V * 4) : 0);
    }
    explicit SplitWork(const InetDelta& d) {
        const int64_t units = (int64_t)d.B * d.H * ((d.T + d.chunk - 1) / d.chunk);
        w = (__bf16*)d.work;
        f = (float*)((char*)d.work + w_bytes(d, units));
        G = (float*)((char*)f + f_bytes(d, units));
    }
};

template <typename T, int C, int KP, bool BACK> struct BeforeLds {
    static constexpr int NP = Elem<T>::planes, LK = KP + 8, LC = C + 8, LL = C + 4;
    Gates<C> gates;
    alignas(16) __bf16 k[NP * C * LK], q[BACK ? NP * C * LK : 8], p[BACK ? 3 * C * LC : 8];
    alignas(16) float ln[C * LL];
    alignas(16) __bf16 v[NP * C * LV], w[3 * C * LK];
};

// One workgroup a chunk, robot, head and 64 columns; the first of the columns' workgroups computes W too.
template <typename T, int C, int KP, bool BACK, bool VEC>
__global__ __launch_bounds__(DELTA_WG, 2) void delta_before_kernel(InetDelta d, const T* __restrict__ rhs, int64_t rhs_b,
                                                                   int64_t rhs_t, int64_t rhs_h, float* __restrict__ U,
                                                                   SplitWork work) {
    constexpr int NP = Elem<T>::planes, RT = C / 16, KT = KP / 16;
    extern __shared__ char lds_raw[];
    typedef BeforeLds<T, C, KP, BACK> Lds;
    Lds& s = *(Lds*)lds_raw;
    const Planes<NP> Kr{s.k, Lds::LK, C * Lds::LK}, Qr{s.q, Lds::LK, C * Lds::LK}, R{s.v, LV, C * LV};
    const Planes<3> P{s.p, Lds::LC, C * Lds::LC}, W{s.w, Lds::LK, C * Lds::LK};
    const int chunks = (d.T + C - 1) / C, ch = blockIdx.x % chunks, t0 = ch * C;
    const int64_t bh = blockIdx.x / chunks, unit = blockIdx.x, row_s = (int64_t)d.H * d.V;
    const int b = (int)(bh / d.H), h = (int)(bh % d.H), hk = h / (d.H / d.Hk);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.y * 64, width = d.V - c0 < 64 ? d.V - c0 : 64;
    {
        Rows<T, C, KP, VEC> kr, qr;
        Rows<T, C, 64, VEC> vr;
        Gate gate;
        kr.load((const T*)d.k + b * d.k_s[0] + hk * d.k_s[2], d.k_s[1], t0, d.T, d.K);
        if (BACK) qr.load((const T*)d.q + b * d.q_s[0] + hk * d.q_s[2], d.q_s[1], t0, d.T, d.K);
        vr.load(rhs + b * rhs_b + h * rhs_h + c0, rhs_t, t0, rhs ? d.T : 0, width);
        if (w == 0) {
            gate.load<C>(d, b, h, t0);
            put_gates<C>(s.gates, gate);
        }
        kr.put(Kr);
        if (BACK) qr.put(Qr);
        vr.put_natural(R);
    }
    __syncthreads();
    if (BACK) {
        triangles<C, KP, NP, 3, true>(Kr, Qr, P, s.gates, s.ln, Lds::LL, d.scale, w, n, g);
    } else {
        if (w < RT) triangle_l<C, KP, NP, false>(Kr, s.gates, s.ln, Lds::LL, w, n, g);
        __syncthreads();
        if (w == 0) invert_blocks<C>(s.ln, Lds::LL);
        __syncthreads();
    }
    const float* rowf = BACK ? s.gates.c : s.gates.a;
    auto solve = [&](f32x4 (&x)[RT]) {
        if (BACK) solve_up<C>(x, s.ln, Lds::LL, n, g);
        else solve_down<C>(x, s.ln, Lds::LL, n, g);
    };
    if (w * 16 < width) {
        f32x4 x[RT] = {};
        if (BACK) {
            f32x4 u[RT], G[KT] = {};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) u[rt] = plane_tile(R, rt * 16, w * 16, n, g);
#pragma unroll
            for (int kp = 0; kp < RT / 2; ++kp) {
                const Frag<NP> uf = split_tiles<NP>(u[2 * kp], u[2 * kp + 1]);
#pragma unroll
                for (int rt = 0; rt < 2 * kp + 2; ++rt) x[rt] = mma<2>(P.tr_frag(rt, kp, n, g), uf, x[rt]);
            }
#pragma unroll
            for (int kp = 0; kp < RT / 2; ++kp) {
                const f32x4 a0 = *(const f32x4*)(s.gates.a + kp * 32 + 4 * g) * d.scale,
                            a1 = *(const f32x4*)(s.gates.a + kp * 32 + 16 + 4 * g) * d.scale;
                const Frag<3> of = split_tiles<3>(u[2 * kp] * a0, u[2 * kp + 1] * a1);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) G[kt] = mma<2>(Qr.tr_frag(kt, kp, n, g), of, G[kt]);
            }
            if (w * 16 + n < width)
                state_store(G, work.G + unit * d.K * d.V + c0, 4 * (uint32_t)(4 * g * d.V + w * 16 + n), d.V, d.K, g);
        } else {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) x[rt] = plane_tile(R, rt * 16, w * 16, n, g);
        }
        solve(x);
        if (w * 16 + n < width) {
            rows_store(x, U + ((int64_t)b * d.T + t0) * row_s + h * d.V + c0, 4 * (uint32_t)(4 * g * row_s + w * 16 + n), row_s,
                       d.T - t0, g);
        }
    }
    if (blockIdx.y) return;
#pragma unroll
    for (int kt = w; kt < KT; kt += 4) {
        f32x4 x[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const f32x4 m = *(const f32x4*)(rowf + rt * 16 + 4 * g);
            x[rt] = Kr.tr_tile(kt, rt, n, g) * (BACK ? m : -m);
        }
        solve(x);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e) W.put1(rt * 16 + 4 * g + e, perm(kt * 16 + n), x[rt][e]);
    }
    if (threadIdx.x < C) {
        const int i = threadIdx.x;
        float* f = work.f + unit * (2 * C + 4);
        f[i] = BACK ? -s.gates.a[i] * s.gates.beta[i] : s.gates.c[i] * s.gates.beta[i];
        f[C + i] = rowf[i];
        if (i == 0) f[2 * C] = s.gates.a_end;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 3 * C * (KP / 8); i += DELTA_WG) {
        const int r = i / (KP / 8), c = i % (KP / 8) * 8;
        *(bf16x8*)(work.w + (unit * 3 * C + r) * KP + c) = *(const bf16x8*)(s.w + r * Lds::LK + c);
    }
}

// chunk operands of the scan, in LDS twice: W's planes, K by rows, f and the rows' factors
template <typename T, int C, int KP> struct ScanBuf {
    static constexpr int NP = Elem<T>::planes, LK = KP + 8;
    alignas(16) __bf16 w[3 * C * LK], k[NP * C * LK];
    alignas(16) float f[2 * C + 4];
};

// One workgroup of eight waves a robot, head and 64 columns: waves 0 .. 3 own 16 columns of the state each, waves 4 .. 7 bring
// the next chunk's operands to LDS (the one wave a SIMD that computes is a single chain; what it need not do shortens it).
// X overwrites U.
template <typename T, int C, int KP, bool BACK, bool VEC>
__global__ __launch_bounds__(2 * DELTA_WG, 2) void delta_serial_kernel(InetDelta d, const float* __restrict__ first,
                                                                   float* __restrict__ last, float* __restrict__ between,
                                                                   float* __restrict__ U, SplitWork work,
                                                                   const T* __restrict__ d_o) {
    constexpr int NP = Elem<T>::planes, RT = C / 16, KT = KP / 16, LK = KP + 8, WG8 = 3 * C * (KP / 8),
                  NW = (WG8 + DELTA_WG - 1) / DELTA_WG;
    extern __shared__ char lds_raw[];
    typedef ScanBuf<T, C, KP> Buf;
    Buf* buf = (Buf*)lds_raw;
    const int chunks = (d.T + C - 1) / C;
    const int64_t bh = blockIdx.x, row_s = (int64_t)d.H * d.V;
    const int b = (int)(bh / d.H), h = (int)(bh % d.H), hk = h / (d.H / d.Hk);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.y * 64, width = d.V - c0 < 64 ? d.V - c0 : 64;
    const bool mine = w * 16 + n < width;
    uint32_t at = 4 * (uint32_t)(4 * g * d.V + w * 16 + n), at_row = 4 * (uint32_t)(4 * g * row_s + w * 16 + n);
    const T* k = (const T*)d.k + b * d.k_s[0] + hk * d.k_s[2];
    float* rows = U + b * (int64_t)d.T * row_s + h * d.V + c0;
    const int64_t kv = (int64_t)d.K * d.V;

    auto chunk_at = [&](int i) { return BACK ? chunks - 1 - i : i; };
    const int tid = threadIdx.x & (DELTA_WG - 1);
    Rows<T, C, KP, VEC> kr;
    kr.tid = tid;
    bf16x8 wr[NW];
    float fr = 0.0f;
    auto fetch = [&](int ch) {
        const int64_t unit = bh * chunks + ch;
#pragma unroll
        for (int m = 0; m < NW; ++m) {
            const int i = tid + m * DELTA_WG;
            if (WG8 % DELTA_WG == 0 || i < WG8)
                wr[m] = *(const bf16x8*)(work.w + (unit * 3 * C + i / (KP / 8)) * KP + i % (KP / 8) * 8);
        }
        kr.load(k, d.k_s[1], ch * C, d.T, d.K);
        if (tid < 2 * C + 4) fr = work.f[unit * (2 * C + 4) + tid];
    };
    auto put = [&](Buf& s) {
#pragma unroll
        for (int m = 0; m < NW; ++m) {
            const int i = tid + m * DELTA_WG;
            if (WG8 % DELTA_WG == 0 || i < WG8) *(bf16x8*)(s.w + i / (KP / 8) * LK + i % (KP / 8) * 8) = wr[m];
        }
        kr.put(Planes<NP>{s.k, LK, C * LK});
        if (tid < 2 * C + 4) s.f[tid] = fr;
    };
    if (w >= 4) {
        fetch(chunk_at(0));
        put(buf[0]);
        if (chunks > 1) fetch(chunk_at(1));
        __syncthreads();
        for (int i = 0; i < chunks; ++i) {
            if (i + 1 < chunks) put(buf[(i + 1) & 1]);
            if (i + 2 < chunks) fetch(chunk_at(i + 2));
            __syncthreads();
        }
        return;
    }
    f32x4 un[RT] = {}, gn[KT] = {};
    auto fetch_own = [&](int ch) {                  // the wave's own columns
        if (mine) rows_load(un, rows + ch * C * row_s, at_row, row_s, d.T - ch * C, g);
        if (BACK) {
            if (mine) state_load(gn, work.G + (bh * chunks + ch) * kv + c0, at, d.V, d.K, g);
        }
    };
    f32x4 S[KT] = {};
    if (mine && first) state_load(S, first + bh * kv + c0, at, d.V, d.K, g);
    fetch_own(chunk_at(0));
    __syncthreads();
    for (int i = 0; i < chunks; ++i) {
        const int ch = chunk_at(i);
        const Buf& s = buf[i & 1];
        keep(at), keep(at_row);
        f32x4 x[RT];
        // (what was fetched for this chunk is waited for here, not with what is fetched next)
        auto arrived = [](f32x4& v) { asm volatile("" : "+v"(v)); };
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            x[rt] = un[rt];
            arrived(x[rt]);
        }
        f32x4 G[KT];
        if (BACK)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                G[kt] = gn[kt];
                arrived(G[kt]);
            }
        if (i + 1 < chunks) fetch_own(chunk_at(i + 1));
        if (w * 16 < width) {
            const Planes<3> W{(__bf16*)s.w, LK, C * LK};
            const Planes<NP> Kr{(__bf16*)s.k, LK, C * LK};
            // the state before the chunk, or its gradient after it: [robot, head][chunks - 1]
            if (i && mine)
                state_store(S, between + (bh * (chunks - 1) + (BACK ? ch : ch - 1)) * kv + c0, at, d.V, d.K, g);
            f32x4 y[RT] = {};
#pragma unroll
            for (int kp = 0; kp < KT / 2; ++kp) {
                const Frag<3> sf = split_tiles<3>(S[2 * kp], S[2 * kp + 1]);
                Frag<3> wf[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) wf[rt] = W.frag(rt * 16 + n, kp * 32 + 8 * g);
                mma_rows<2>(wf, sf, y);
            }
            const float a_end = s.f[2 * C];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const f32x4 m = *(const f32x4*)(s.f + C + rt * 16 + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[rt][e] += m[e] != 0.0f ? y[rt][e] : 0.0f;
                }
            }
            if (mine) rows_store(x, rows + ch * C * row_s, at_row, row_s, d.T - ch * C, g);
            f32x4 old[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                old[kt] = S[kt];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    S[kt][e] = (a_end != 0.0f ? a_end * S[kt][e] : 0.0f) + (BACK ? G[kt][e] : 0.0f);
            }
#pragma unroll
            for (int kp = 0; kp < RT / 2; ++kp) {
                const f32x4 f0 = *(const f32x4*)(s.f + kp * 32 + 4 * g), f1 = *(const f32x4*)(s.f + kp * 32 + 16 + 4 * g);
                const Frag<3> xf = split_tiles<3>(x[2 * kp] * f0, x[2 * kp + 1] * f1);
                Frag<NP> kf[KT];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) kf[kt] = Kr.tr_frag(kt, kp, n, g);
                mma_rows<2>(kf, xf, S);
            }
            if (__builtin_expect(!all_finite(x, s.f, g), 0)) {       // (asked at the end: the chain does not wait for it)
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // (X is stored once more)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) S[kt] = old[kt];
                SameDelta& a = same_delta();
                const int col = w * 16 + n;
                auto give = [&](int t, float e, float = 0.0f) {
                    if (mine) rows[(ch * C + t) * row_s + col] = e;
                };
                const T* q = (const T*)a.q + b * a.q_s[0] + hk * a.q_s[2];
                if (BACK) {
                    const T* u = d_o + b * (int64_t)a.T * row_s + h * a.V + c0;
                    steps_backward<C>(a, b, h, ch * C, k, q, u, row_s, col, mine && d_o, S, g, give);
                } else {
                    const T* v = (const T*)a.v + b * a.v_s[0] + h * a.v_s[2] + c0;
                    steps_forward<C, false>(a, b, h, ch * C, k, q, v, a.v_s[1], col, mine, S, g, give);
                }
            }
        }
        __syncthreads();
    }
    if (mine && last) state_store(S, last + bh * kv + c0, at, d.V, d.K, g);
}

template <typename T, int C, int KP> struct AfterLds {
    static constexpr int NP = Elem<T>::planes, NO = Elem<T>::ord + 1, LK = KP + 8, LC = C + 8;
    Gates<C> gates;
    alignas(16) __bf16 k[NP * C * LK], q[NP * C * LK], p[NO * C * LC];
    alignas(16) T o[C * LV];
};

// O of one chunk, robot, head and 64 columns
template <typename T, int C, int KP, bool VEC>
__global__ __launch_bounds__(DELTA_WG, 2) void delta_after_kernel(InetDelta d) {
    constexpr int NP = Elem<T>::planes, ORD = Elem<T>::ord, NO = ORD + 1, RT = C / 16, KT = KP / 16;
    extern __shared__ char lds_raw[];
    typedef AfterLds<T, C, KP> Lds;
    Lds& s = *(Lds*)lds_raw;
    const Planes<NP> Kr{s.k, Lds::LK, C * Lds::LK}, Qr{s.q, Lds::LK, C * Lds::LK};
    const Planes<NO> P{s.p, Lds::LC, C * Lds::LC};
    const int chunks = (d.T + C - 1) / C, ch = blockIdx.x % chunks, t0 = ch * C;
    const int64_t bh = blockIdx.x / chunks, row_s = (int64_t)d.H * d.V, kv = (int64_t)d.K * d.V;
    const int b = (int)(bh / d.H), h = (int)(bh % d.H), hk = h / (d.H / d.Hk);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.y * 64, width = d.V - c0 < 64 ? d.V - c0 : 64;
    const bool mine = w * 16 + n < width;
    const int64_t row0 = ((int64_t)b * d.T + t0) * row_s + h * d.V + c0;
    Rows<T, C, KP, VEC> kr, qr;
    Gate gate;
    kr.load((const T*)d.k + b * d.k_s[0] + hk * d.k_s[2], d.k_s[1], t0, d.T, d.K);
    qr.load((const T*)d.q + b * d.q_s[0] + hk * d.q_s[2], d.q_s[1], t0, d.T, d.K);
    f32x4 S[KT] = {}, x[RT] = {};
    const float* from = ch ? d.chunk_state + (bh * (chunks - 1) + ch - 1) * kv : d.state ? d.state + bh * kv : nullptr;
    if (mine && from) state_load(S, from + c0, 4 * (uint32_t)(4 * g * d.V + w * 16 + n), d.V, d.K, g);
    if (mine) rows_load(x, d.err + row0, 4 * (uint32_t)(4 * g * row_s + w * 16 + n), row_s, d.T - t0, g);
    if (w == 0) {
        gate.load<C>(d, b, h, t0);
        put_gates<C>(s.gates, gate);
    }
    kr.put(Kr);
    qr.put(Qr);
    __syncthreads();
    if (w < RT) triangle_p<C, KP, NP, NO>(Kr, Qr, P, s.gates, d.scale, w, n, g);
    __syncthreads();
    if (w * 16 < width) {
        f32x4 o[RT] = {};
#pragma unroll
        for (int kp = 0; kp < KT / 2; ++kp) {
            const Frag<NO> sf = split_tiles<NO>(S[2 * kp], S[2 * kp + 1]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt] = mma<ORD>(Qr.frag(rt * 16 + n, kp * 32 + 8 * g), sf, o[rt]);
        }
        const bool sound = all_finite(x, s.gates.beta, g);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const f32x4 a = *(const f32x4*)(s.gates.a + rt * 16 + 4 * g);
            x[rt] *= *(const f32x4*)(s.gates.beta + rt * 16 + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[rt][e] = a[e] != 0.0f ? d.scale * a[e] * o[rt][e] : 0.0f;
        }
#pragma unroll
        for (int kp = 0; kp < RT / 2; ++kp) {
            const Frag<NO> xf = split_tiles<NO>(x[2 * kp], x[2 * kp + 1]);
#pragma unroll
            for (int rt = 2 * kp; rt < RT; ++rt) o[rt] = mma<ORD>(P.frag(rt * 16 + n, kp * 32 + 8 * g), xf, o[rt]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) tile_put(s.o + rt * 16 * LV + w * 16, LV, n, g, o[rt]);
        if (__builtin_expect(!sound, 0)) {
            const int col = w * 16 + n;
            SameDelta& a = same_delta();
            steps_forward<C, true>(a, b, h, t0, (const T*)a.k + b * a.k_s[0] + hk * a.k_s[2],
                                   (const T*)a.q + b * a.q_s[0] + hk * a.q_s[2],
                                   (const T*)a.v + b * a.v_s[0] + h * a.v_s[2] + c0, a.v_s[1], col, mine, S, g,
                                   [&](int t, float, float out) { s.o[t * LV + col] = (T)out; });
        }
    }
    __syncthreads();
    store_rows<T, C, VEC>(s.o, (T*)d.o + row0, row_s, d.T - t0, width);
}

template <typename T, int C, int KP, bool BACK, bool VEC>
static int launch(const InetDelta& d, const InetDeltaGrad* g, hipStream_t st) {
    const int chunks = (d.T + C - 1) / C, cols = (d.V + 63) / 64;
    const SplitWork work(d);
    static_assert(sizeof(BeforeLds<T, C, KP, BACK>) <= LDS_MAX && 2 * sizeof(ScanBuf<T, C, KP>) <= LDS_MAX &&
                      sizeof(AfterLds<T, C, KP>) <= LDS_MAX, "LDS");
    auto before = delta_before_kernel<T, C, KP, BACK, VEC>;
    auto serial = delta_serial_kernel<T, C, KP, BACK, VEC>;
    const size_t bl = sizeof(BeforeLds<T, C, KP, BACK>), sl = 2 * sizeof(ScanBuf<T, C, KP>);
    if (allow_lds((const void*)before, bl) || allow_lds((const void*)serial, sl)) return INET_POLICY_ELAUNCH;
    const T* rhs = BACK ? (const T*)g->d_o : (const T*)d.v;
    const int64_t rs[3] = {BACK ? (int64_t)d.T * d.H * d.V : d.v_s[0], BACK ? (int64_t)d.H * d.V : d.v_s[1],
                           BACK ? (int64_t)d.V : d.v_s[2]};
    float* U = BACK ? g->err_grad : d.err;
    hipLaunchKernelGGL(before, dim3(d.B * d.H * chunks, cols), dim3(DELTA_WG), bl, st, d, rhs, rs[0], rs[1], rs[2], U,
                       work);
    if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH;
    hipLaunchKernelGGL(serial, dim3(d.B * d.H, cols), dim3(2 * DELTA_WG), sl, st, d, BACK ? g->d_state_out : d.state,
                       BACK ? g->d_state : d.state_out, BACK ? g->chunk_grad : d.chunk_state, U, work,
                       BACK ? rhs : nullptr);
    if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH;
    if (!BACK) {
        auto after = delta_after_kernel<T, C, KP, VEC>;
        const size_t al = sizeof(AfterLds<T, C, KP>);
        if (allow_lds((const void*)after, al)) return INET_POLICY_ELAUNCH;
        hipLaunchKernelGGL(after, dim3(d.B * d.H * chunks, cols), dim3(DELTA_WG), al, st, d);
    }
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

size_t delta_split_bytes(const InetDelta& d, bool back) { return SplitWork::bytes(d, back); }

// a forward pass, or the serial part of a backward one
int delta_split(const InetDelta& d, const InetDeltaGrad* g, bool vec, hipStream_t st) {
    return delta_dispatch(d, [&](auto t, auto c, auto kp) {
        typedef typename decltype(t)::type T;
        constexpr int C = decltype(c)::value, KP = decltype(kp)::value;
        if (g) return vec ? launch<T, C, KP, true, true>(d, g, st) : launch<T, C, KP, true, false>(d, g, st);
        return vec ? launch<T, C, KP, false, true>(d, g, st) : launch<T, C, KP, false, false>(d, g, st);
    });
}

}  // namespace pol
