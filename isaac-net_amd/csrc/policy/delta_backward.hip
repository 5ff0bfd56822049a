// Backward pass of the gated delta rule over windows (the mathematics: delta.h). A window of one chunk is one kernel's
// (delta_window_kernel). Longer ones take two: the state's gradient goes backwards through a window chunk by chunk, column
// tile by column tile, as the forward pass goes forwards, and leaves each chunk's dS and Z (delta_scan_kernel); with
// those, every chunk's gradients of q, k and the gates are independent, and one workgroup a chunk computes them
// (delta_chunk_kernel).
#include "delta.h"
#include "delta_launch.h"

namespace pol {

// the kernels' second argument, as same_delta()
typedef const __attribute__((address_space(4))) InetDeltaGrad SameGrad;
DEV SameGrad& same_grad() {
    static_assert(sizeof(InetDelta) % alignof(InetDeltaGrad) == 0, "the arguments lie one behind the other");
    return *(SameGrad*)(&same_delta() + 1);
}

// rows of values [steps][V] into planes in their own order, zeros up to vp columns
template <typename T, int C, bool VEC, int N>
DEV void stage_rows(const T* __restrict__ x, int64_t row0, int64_t row_s, int steps, int V, int vp, const Planes<N>& s) {
    for (int i = threadIdx.x; i < C * (vp / 8); i += DELTA_WG) {
        const int r = i / (vp / 8), c = i % (vp / 8) * 8;
        float o[8] = {};
        if (x && r < steps && c < V) load8(x + row0 + r * row_s + c, V - c, VEC, o);
        s.put4(r, c, o[0], o[1], o[2], o[3]);
        s.put4(r, c + 4, o[4], o[5], o[6], o[7]);
    }
}

// 16 columns of a chunk: Z from the gradient S of the state after the chunk (has_s; else zero) and dO (u, read here)
template <int C, int KP, int NP>
DEV void column_gradients(const f32x4 (&S)[KP / 16], bool has_s, f32x4 (&z)[C / 16], f32x4 (&u)[C / 16],
                          const Gates<C>& gates, const float* ln, int ld, const Planes<NP>& Kr, const Planes<3>& P,
                          const Planes<NP>& O, int c0, int n, int g) {
    constexpr int RT = C / 16, KT = KP / 16;
    // dX = c K dS + P^T dO
    if (has_s) {
#pragma unroll
        for (int kp = 0; kp < KT / 2; ++kp) {
            const Frag<3> sf = split_tiles<3>(S[2 * kp], S[2 * kp + 1]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) z[rt] = mma<2>(Kr.frag(rt * 16 + n, kp * 32 + 8 * g), sf, z[rt]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const f32x4 c = *(const f32x4*)(gates.c + rt * 16 + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[rt][e] = c[e] != 0.0f ? c[e] * z[rt][e] : 0.0f;
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) u[rt] = plane_tile(O, rt * 16, c0, n, g);
#pragma unroll
    for (int kp = 0; kp < RT / 2; ++kp) {
        const Frag<NP> uf = split_tiles<NP>(u[2 * kp], u[2 * kp + 1]);
#pragma unroll
        for (int rt = 0; rt < 2 * kp + 2; ++rt) z[rt] = mma<2>(P.tr_frag(rt, kp, n, g), uf, z[rt]);
    }
    solve_up<C>(z, ln, ld, n, g);                   // Z
}

// S, the gradient of the state after a chunk, to that of the state before it: a_C S + Q^T (scale a dO) - K^T (a beta Z)
template <int C, int KP, int NP>
DEV void state_gradient(f32x4 (&S)[KP / 16], const f32x4 (&z)[C / 16], const f32x4 (&u)[C / 16], const Gates<C>& gates,
                        float scale, const Planes<NP>& Kr, const Planes<NP>& Qr, int n, int g) {
    constexpr int RT = C / 16, KT = KP / 16;
    const float a_end = gates.a_end;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[kt][e] = a_end != 0.0f ? a_end * S[kt][e] : 0.0f;
#pragma unroll
    for (int kp = 0; kp < RT / 2; ++kp) {
        f32x4 o[2], y[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const f32x4 a = *(const f32x4*)(gates.a + kp * 32 + 16 * m + 4 * g),
                        bt = *(const f32x4*)(gates.beta + kp * 32 + 16 * m + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[m][e] = scale * a[e] * u[2 * kp + m][e];
                y[m][e] = a[e] != 0.0f ? -bt[e] * a[e] * z[2 * kp + m][e] : 0.0f;
            }
        }
        const Frag<3> of = split_tiles<3>(o[0], o[1]), yf = split_tiles<3>(y[0], y[1]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            S[kt] = mma<2>(Qr.tr_frag(kt, kp, n, g), of, S[kt]);
            S[kt] = mma<2>(Kr.tr_frag(kt, kp, n, g), yf, S[kt]);
        }
    }
}

template <typename T, int C, int KP> struct ScanLds {
    static constexpr int NP = Elem<T>::planes, LK = KP + 8, LC = C + 8, LL = C + 4;
    Gates<C> gates;
    alignas(16) __bf16 k[NP * C * LK], q[NP * C * LK], p[3 * C * LC];
    alignas(16) float ln[C * LL];
    alignas(16) __bf16 u[NP * C * LV];
};

// The state's gradient. One workgroup of four waves per robot, head and 64 columns; wave w owns 16 columns. Bound as the
// forward pass is, by its chain of products a chunk. 300 robots x 77 steps x 6 heads of 40 x 56, float32: 113 us.
template <typename T, int C, int KP, bool VEC>
__global__ __launch_bounds__(DELTA_WG, 3 * sizeof(ScanLds<T, C, KP>) <= LDS_MAX && KP <= 64 ? 3 : 2)
void delta_scan_kernel(InetDelta d, InetDeltaGrad gr) {
    constexpr int NP = Elem<T>::planes, RT = C / 16, KT = KP / 16;
    extern __shared__ char lds_raw[];
    typedef ScanLds<T, C, KP> Lds;
    Lds& s = *(Lds*)lds_raw;
    const Planes<NP> Kr{s.k, Lds::LK, C * Lds::LK}, Qr{s.q, Lds::LK, C * Lds::LK};
    const Planes<3> P{s.p, Lds::LC, C * Lds::LC};
    const Planes<NP> O{s.u, LV, C * LV};
    const int b = blockIdx.x / d.H, h = blockIdx.x % d.H, hk = h / (d.H / d.Hk);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.y * 64, width = d.V - c0 < 64 ? d.V - c0 : 64;      // the workgroup's columns
    const bool cols = w * 16 < width, mine = w * 16 + n < width;
    const T* q = (const T*)d.q + b * d.q_s[0] + hk * d.q_s[2];
    const T* k = (const T*)d.k + b * d.k_s[0] + hk * d.k_s[2];
    const int chunks = (d.T + C - 1) / C;
    const int64_t bh = (int64_t)b * d.H + h, row_s = (int64_t)d.H * d.V, rows0 = b * (int64_t)d.T * row_s + h * d.V + c0;

    Rows<T, C, KP, VEC> kr, qr;
    Rows<T, C, 64, VEC> ur;                              // dO
    Gate gate;
    auto fetch = [&](int t0) {
        kr.load(k, d.k_s[1], t0, d.T, d.K);
        qr.load(q, d.q_s[1], t0, d.T, d.K);
        ur.load((const T*)gr.d_o + rows0, row_s, t0, gr.d_o ? d.T : 0, width);
        if (w == 0) gate.load<C>(d, b, h, t0);
    };
    if (chunks) fetch((chunks - 1) * C);

    uint32_t at = 4 * (uint32_t)(4 * g * d.V + w * 16 + n), at_err = 4 * (uint32_t)(4 * g * row_s + w * 16 + n);
    f32x4 S[KT] = {};                               // the gradient of the state, 16 columns
    if (mine && gr.d_state_out) state_load(S, gr.d_state_out + bh * d.K * d.V + c0, at, d.V, d.K, g);

    for (int ch = chunks - 1; ch >= 0; --ch) {
        const int t0 = ch * C;
        kr.put(Kr);
        qr.put(Qr);
        ur.put_natural(O);
        if (w == 0) put_gates<C>(s.gates, gate);
        __syncthreads();
        keep(at), keep(at_err);
        triangles<C, KP, NP, 3, true>(Kr, Qr, P, s.gates, s.ln, Lds::LL, d.scale, w, n, g);
        if (ch) fetch(t0 - C);
        if (cols) {
            f32x4 z[RT] = {}, u[RT];
            column_gradients<C, KP, NP>(S, true, z, u, s.gates, s.ln, Lds::LL, Kr, P, O, w * 16, n, g);
            const bool sound = all_finite(z, s.gates.beta, g);
            if (mine) {
                rows_store(z, gr.err_grad + rows0 + t0 * row_s, at_err, row_s, d.T - t0, g);
                if (ch + 1 < chunks)
                    state_store(S, gr.chunk_grad + (bh * (chunks - 1) + ch) * d.K * d.V + c0, at, d.V, d.K, g);
            }
            f32x4 old[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) old[kt] = S[kt];
            if (ch || gr.d_state) state_gradient<C, KP, NP>(S, z, u, s.gates, d.scale, Kr, Qr, n, g);
            if (__builtin_expect(!sound, 0)) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // (Z is stored once more)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) S[kt] = old[kt];
                SameDelta& a = same_delta();
                const T* d_o = (const T*)same_grad().d_o;
                const int col = w * 16 + n;
                float* to = same_grad().err_grad + rows0 + t0 * row_s + col;
                steps_backward<C>(a, b, h, t0, k, q, d_o + rows0, row_s, col, mine && d_o, S, g,
                                  [&](int t, float x) { if (mine) to[t * row_s] = x; });
            }
        }
        __syncthreads();
    }
    if (mine && gr.d_state) state_store(S, gr.d_state + bh * d.K * d.V + c0, at, d.V, d.K, g);
}

// the rows' sums that the log-decays' gradients are made of, by the key rows' part: q . dQ, k . dK+, k . dK-, the state's
// share of k . dK- (in the triangles' place when those are done with); and E . Z, and <S, dS> by wave
template <int C> struct Parts {
    float q[4][C], kp[4][C], km[4][C], ks[4][C];
};
template <int C> struct alignas(16) Sums {
    float ez[C], ss[4];
    int odd[4];                                          // whether a wave's errors or Z are not all finite
};

// The planes that the gradients' products hold X, Z, S, dS, D and M in: as many as the outputs of q's type ask for, but three
// (WIDE) where 16-bit q, k and v have float32 gates, whose gradients are then of 32-bit grade too. 1008 x 2774 x 1 head of 24 x
// 24, bfloat16: chunk kernel 750 us, wide 878; 16384 x 24 x 2 heads of 64 x 64: window kernel 627, wide 790 (in turn, in
// one run).
template <typename T, bool WIDE> struct Grade {
    static constexpr int ord = WIDE ? 2 : Elem<T>::ord, planes = ord + 1;
};

// D and M of a chunk in LDS (as P: columns in the order perm()), in the place of X, Z and dO when those are done with
template <int NO, int C> struct Inner {
    static constexpr int LC = C + 8, SIZE = 2 * NO * C * LC;
    Planes<NO> D, M;
    DEV explicit Inner(__bf16* p) : D{p, LC, C * LC}, M{p + NO * C * LC, LC, C * LC} {}
};

// LDS of the chunk kernel in bytes: gates and sums, K and Q, and the rows X, Z and dO (of vp + 8) with the triangles in
// their place at the end, Z and dO in the order in which the one-chunk kernel can have its own triangles in X's place
template <typename T, int C, int NO> constexpr size_t rows_lds(int vp, size_t triangles) {
    const size_t row = sizeof(__bf16) * C * (vp + 8), NP = Elem<T>::planes, x = NO * row,
                 all = (NO + NP) * row + (x > triangles ? x : triangles), in = sizeof(__bf16) * Inner<NO, C>::SIZE;
    return all > in ? all : in;
}
template <typename T, int C, int KP, int NO> constexpr size_t chunk_lds(int vp, size_t triangles = 0) {
    return sizeof(Gates<C>) + sizeof(Sums<C>) + sizeof(__bf16) * 2 * Elem<T>::planes * C * (KP + 8) +
           rows_lds<T, C, NO>(vp, triangles);
}

// X = beta E, dbeta's E . Z and dV = beta Z by rows; Z from memory (err_grad) where z_in, else as it is in LDS already
template <typename T, int C, bool VEC, int NO>
DEV void stage_errors(const InetDelta& d, const float* z_in, T* dv, int64_t row0, int64_t row_s, int steps, int vp,
                      const Gates<C>& gates, const Planes<NO>& X, const Planes<NO>& Z, Sums<C>& sums) {
    const int lanes = vp <= 32 ? 4 : vp <= 64 ? 8 : 16;             // a row
    float sound = 0.0f;                                             // 0, or NaN
    for (int i = threadIdx.x; i < C * lanes; i += DELTA_WG) {
        const int r = i / lanes, c = i % lanes * 8;
        float e[8] = {}, z[8] = {}, x = 0.0f;
        if (r < steps && c < d.V) load8(d.err + row0 + r * row_s + c, d.V - c, VEC, e);
        const float beta = gates.beta[r];
        if (c < vp) {
            if (z_in) {
                if (r < steps && c < d.V) load8(z_in + row0 + r * row_s + c, d.V - c, VEC, z);
                Z.put4(r, c, z[0], z[1], z[2], z[3]);
                Z.put4(r, c + 4, z[4], z[5], z[6], z[7]);
            } else {
                const Frag<NO> f = Z.frag(r, c);
#pragma unroll
                for (int m = 0; m < NO; ++m)
#pragma unroll
                    for (int u = 0; u < 8; ++u) z[u] += (float)f.p[m][u];
            }
            if (r < steps && c < d.V) {
                const float lo[4] = {beta * z[0], beta * z[1], beta * z[2], beta * z[3]},
                            hi[4] = {beta * z[4], beta * z[5], beta * z[6], beta * z[7]};
                store4(dv + row0 + r * row_s + c, d.V - c, VEC, lo);
                store4(dv + row0 + r * row_s + c + 4, d.V - c - 4, VEC, hi);
            }
            X.put4(r, c, beta * e[0], beta * e[1], beta * e[2], beta * e[3]);
            X.put4(r, c + 4, beta * e[4], beta * e[5], beta * e[6], beta * e[7]);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            x += e[u] * z[u];
            sound += beta * e[u] * 0.0f + beta * z[u] * 0.0f;
        }
        for (int o = 1; o < lanes; o <<= 1) x += __shfl_xor(x, o);
        if (c == 0) sums.ez[r] = x;
    }
    const bool odd = __builtin_amdgcn_ballot_w64(sound != sound) != 0;
    if ((threadIdx.x & 63) == 0) sums.odd[threadIdx.x >> 6] = odd;
}

// eight consecutive values of a 32-bit matrix's row
DEV void row8(const float* __restrict__ p, bool in, int v, int V, bool vec, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    if (in && v < V) load8(p + v, V - v, vec, x);
}

// dg and dbeta of step t, the chunk's step i, in the gates' type (D, G: InetDelta and InetDeltaGrad wherever they lie)
template <int C, typename D, typename G>
DEV void put_gate_gradients(D& d, G& gr, int b, int h, int t, int i, const Gates<C>& gates, float dg, float db) {
    const int64_t at = ((int64_t)b * d.T + t) * d.H + h;
    if (i ? gates.seg[i] != gates.seg[i - 1] : gates.seg[0] != 0) dg = 0.0f;         // (the memory was emptied)
    if (d.gate_dtype == INET_POLICY_F32) {
        ((float*)gr.d_g)[at] = dg;
        ((float*)gr.d_beta)[at] = db;
    } else if (d.gate_dtype == INET_POLICY_BF16) {
        ((__bf16*)gr.d_g)[at] = (__bf16)dg;
        ((__bf16*)gr.d_beta)[at] = (__bf16)db;
    } else {
        ((_Float16*)gr.d_g)[at] = (_Float16)dg;
        ((_Float16*)gr.d_beta)[at] = (_Float16)db;
    }
}

// The gradients of q, k and the gates of one chunk, from K, Q, X, Z and dO in LDS and the state S before the chunk and its
// gradient dS after it (NULL: zero). A wave takes key rows' tiles (and, where there are fewer than four of those, its share
// of the steps' tiles), so that S and dS are read and split once; the triangles D and M wait in registers until X, Z and
// dO, at `place`, are done with.
template <typename T, int C, int KP, bool VEC, int NP, int NO>
DEV void chunk_gradients(const InetDelta& d, const InetDeltaGrad& gr, int b, int h, int t0, const float* __restrict__ S,
                         const float* __restrict__ dS, const Gates<C>& gates, Sums<C>& sums, const Planes<NP>& Kr,
                         const Planes<NP>& Qr, const Planes<NO>& X, const Planes<NO>& Z, const Planes<NP>& O,
                         __bf16* place, int vp) {
    constexpr int ORD = NO - 1, RT = C / 16, KT = KP / 16, KW = KT < 4 ? KT : 4, TW = 4 / KW, TN = RT / TW;
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, hk = h / (d.H / d.Hk);
    const T* q = (const T*)d.q + b * d.q_s[0] + hk * d.q_s[2];
    const T* k = (const T*)d.k + b * d.k_s[0] + hk * d.k_s[2];
    // row tile it of D (from dO) and of M (from Z): the lane's step i, steps j = 4 g + e of an earlier tile
    constexpr int PASSES = C == 64 ? 2 : 1;
    const int it = C == 64 ? w : w & 1;
    f32x4 tri[PASSES][RT] = {};
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        const int i = it * 16 + n;
        const bool m = C == 64 ? pass : w >> 1;
        for (int v = 0; v < vp; v += 32) {
            if (m) {
                const Frag<NO> z = Z.frag(i, v + 8 * g);
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    if (r <= it) tri[pass][r] = mma<ORD>(X.frag(r * 16 + n, v + 8 * g), z, tri[pass][r]);
            } else {
                const Frag<NP> o = O.frag(i, v + 8 * g);
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    if (r <= it) tri[pass][r] = mma<ORD>(X.frag(r * 16 + n, v + 8 * g), o, tri[pass][r]);
            }
        }
        const float f = m ? -gates.beta[i] : d.scale;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int j = r * 16 + 4 * g;
            if (r <= it) {
                const f32x4 dec = (r == it ? decay4<C, true>(gates, i, j) : decay4<C, false>(gates, i, j)) * f;
                tri[pass][r] *= dec;
                if (m && r == it)
#pragma unroll
                    for (int e = 0; e < 4; ++e) tri[pass][r][e] = j + e < i ? tri[pass][r][e] : 0.0f;
            }
        }
    }
    // the state's shares; part: the wave's key rows, its steps' tiles: first, first + TW, ...
    constexpr int KN = KT / KW;
    const int part = w % KW, first = w / KW;
    float sq[TN] = {}, sp[TN] = {}, sn[TN] = {}, sc[TN] = {}, ss = 0.0f;
    f32x4 dq[KN][TN] = {}, dp[KN][TN] = {}, dm[KN][TN] = {};
#pragma unroll
    for (int kn = 0; kn < KN; ++kn) {
        const int kt = kn * KW + part, row = kt * 16 + n;
        if (kt * 16 >= d.K) continue;
        for (int v = 0; v < vp; v += 32) {
            float x[8], y[8];
            if (S) {
                row8(S + (int64_t)row * d.V, row < d.K, v + 8 * g, d.V, VEC, x);
                const Frag<NO> sf = split8<NO>(x);
#pragma unroll
                for (int u = 0; u < TN; ++u) {
                    const int i = (first + u * TW) * 16 + n;
                    dq[kn][u] = mma<ORD>(sf, O.frag(i, v + 8 * g), dq[kn][u]);
                    dp[kn][u] = mma<ORD>(sf, Z.frag(i, v + 8 * g), dp[kn][u]);
                }
            }
            if (dS) {
                row8(dS + (int64_t)row * d.V, row < d.K, v + 8 * g, d.V, VEC, y);
                const Frag<NO> df = split8<NO>(y);
#pragma unroll
                for (int u = 0; u < TN; ++u)
                    dm[kn][u] = mma<ORD>(df, X.frag((first + u * TW) * 16 + n, v + 8 * g), dm[kn][u]);
                if (S && first == 0)
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss += x[e] * y[e];
            }
        }
    }
    __syncthreads();                                    // X, Z and dO are done with
    const Inner<NO, C> in(place);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        const int i = it * 16 + n;
        const bool m = C == 64 ? pass : w >> 1;
        const Planes<NO> to{in.D.p + (m ? NO * C * in.D.ld : 0), in.D.ld, in.D.plane};     // (an offset: LDS to the compiler)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const f32x4 x = tri[pass][r];
            if (r <= it || (r == it + 1 && (r & 1))) to.put4(i, perm(r * 16 + 4 * g), x[0], x[1], x[2], x[3]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int kn = 0; kn < KN; ++kn) {
        const int kt = kn * KW + part;
        if (kt * 16 >= d.K) continue;
#pragma unroll
        for (int u = 0; u < TN; ++u) {
            const int tt = first + u * TW, i = tt * 16 + n;
            const float a = gates.a[i], c = gates.c[i], ya = -gates.beta[i] * a, oa = d.scale * a;
            f32x4 q4 = dq[kn][u], p4 = dp[kn][u], m4 = dm[kn][u], dc;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q4[e] = a != 0.0f ? q4[e] * oa : 0.0f;
                p4[e] = a != 0.0f ? p4[e] * ya : 0.0f;
                m4[e] = c != 0.0f ? m4[e] * c : 0.0f;
                dc[e] = m4[e];
            }
#pragma unroll
            for (int p = 0; p < RT / 2; ++p) {
                const Frag<NP> kf = Kr.tr_frag(kt, p, n, g);
                if (2 * p <= tt) {                          // earlier steps
                    q4 = mma<ORD>(kf, in.D.frag(i, p * 32 + 8 * g), q4);
                    p4 = mma<ORD>(kf, in.M.frag(i, p * 32 + 8 * g), p4);
                }
                if (2 * p + 1 >= tt) {                      // later ones
                    m4 = mma<ORD>(Qr.tr_frag(kt, p, n, g), in.D.tr_frag(tt, p, n, g), m4);
                    m4 = mma<ORD>(kf, in.M.tr_frag(tt, p, n, g), m4);
                }
            }
            const int kd = kt * 16 + 4 * g, t = t0 + i;
            if (t < d.T && kd < d.K) {
                float qv[4], kv[4], dk[4], dqv[4];
                load4(q + t * d.q_s[1] + kd, d.K - kd, VEC, qv);
                load4(k + t * d.k_s[1] + kd, d.K - kd, VEC, kv);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sq[u] += q4[e] * qv[e];
                    sp[u] += p4[e] * kv[e];
                    sn[u] += m4[e] * kv[e];
                    sc[u] += dc[e] * kv[e];
                    dk[e] = p4[e] + m4[e];
                    dqv[e] = q4[e];
                }
                const int64_t at = (((int64_t)b * d.T + t) * d.H + h) * d.K + kd;
                if (d.H == d.Hk) {
                    store4((T*)gr.d_q + at, d.K - kd, VEC, dqv);
                    store4((T*)gr.d_k + at, d.K - kd, VEC, dk);
                } else {
                    store4(gr.head_grad + at, d.K - kd, VEC, dqv);
                    store4(gr.head_grad + (int64_t)d.B * d.T * d.H * d.K + at, d.K - kd, VEC, dk);
                }
            }
        }
    }
    static_assert(sizeof(Parts<C>) <= sizeof(__bf16) * Inner<NO, C>::SIZE, "the triangles' place");
    Parts<C>& parts = *(Parts<C>*)place;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < TN; ++u) {
        const int i0 = (first + u * TW) * 16 + n;
        auto give = [&](float x, float (&to)[4][C]) {
            x += __shfl_xor(x, 16);
            x += __shfl_xor(x, 32);
            if (g == 0) to[part][i0] = x;
        };
        give(sq[u], parts.q), give(sp[u], parts.kp), give(sn[u], parts.km), give(sc[u], parts.ks);
    }
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
    if (lane == 0) sums.ss[w] = ss;
    __syncthreads();
    if (w == 0) {
        const int step = t0 + lane;
        float x = 0.0f, e = 0.0f;
        int seg = -1;
        if (lane < C) {
            seg = gates.seg[lane];
#pragma unroll
            for (int m = 0; m < KW; ++m) {
                x += parts.q[m][lane] + parts.kp[m][lane] - parts.km[m][lane];
                e += parts.ks[m][lane];
            }
        }
        // the state's share, at the last step
        for (int o = 32; o; o >>= 1) e += __shfl_xor(e, o);
        if (lane == C - 1)
            x += e + (gates.a_end != 0.0f ? gates.a_end * (sums.ss[0] + sums.ss[1] + sums.ss[2] + sums.ss[3]) : 0.0f);
        for (int o = 1; o < C; o <<= 1) {
            const float u = __shfl_down(x, o);
            const int sg = __shfl_down(seg, o);
            if (lane + o < C && sg == seg) x += u;
        }
        if (lane < C && step < d.T) put_gate_gradients<C>(d, gr, b, h, step, lane, gates, x, sums.ez[lane]);
    }
}

// eight columns of a row from c on (past the last: 0), without branches
template <typename T> DEV void columns8(const T* p, bool in, uint32_t c, int V, float (&x)[8]) {
    keep(c);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const bool at = in && c + u < (uint32_t)V;
        const float v = (float)p[at ? c + u : 0u];
        x[u] = at ? v : 0.0f;
    }
}

// The same by single steps, where the errors or Z are not finite (what a product would carry to steps that see nothing of them):
// the state before each step is taken anew from that before the chunk, 16 lanes a key row, eight columns each. rows: six rows
// of C in LDS.
template <typename T, int C, int NO>
DEV void chunk_steps(int b, int h, int t0, const Planes<NO>& Z, const Gates<C>& gates, const Sums<C>& sums, float* rows) {
    SameDelta& d = same_delta();
    SameGrad& gr = same_grad();
    const int chunks = (d.T + C - 1) / C, ch = t0 / C, steps = d.T - t0 < C ? d.T - t0 : C, hk = h / (d.H / d.Hk), K = d.K, V = d.V;
    const int64_t bh = (int64_t)b * d.H + h, kv = (int64_t)d.K * V, at = bh * (chunks - 1) + ch, row_s = (int64_t)d.H * V;
    const float* S0 = ch ? d.chunk_state + (at - 1) * kv : d.state ? d.state + bh * kv : nullptr;
    const float* dS0 = ch + 1 < chunks ? gr.chunk_grad + at * kv : gr.d_state_out ? gr.d_state_out + bh * kv : nullptr;
    const T *k = (const T*)d.k + b * d.k_s[0] + hk * d.k_s[2] + t0 * d.k_s[1],
            *q = (const T*)d.q + b * d.q_s[0] + hk * d.q_s[2] + t0 * d.q_s[1];
    const int64_t row0 = ((int64_t)b * d.T + t0) * row_s + h * V, k_s = d.k_s[1], q_s = d.q_s[1];
    const float scale = d.scale;
    const float* err = d.err + row0;
    const T* d_o = gr.d_o ? (const T*)gr.d_o + row0 : nullptr;
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, c0 = (threadIdx.x & 15) * 8;
    float *keeps = rows + 4 * C, *betas = rows + 5 * C;
    for (int i = threadIdx.x; i < 4 * C; i += DELTA_WG) rows[i] = 0.0f;
    if ((int)threadIdx.x < steps) {
        const StepGate gate(d, b, h, t0 + threadIdx.x);
        keeps[threadIdx.x] = gate.keep;
        betas[threadIdx.x] = gate.beta;
    }
    __syncthreads();
#pragma nounroll
    for (int r0 = 0; r0 < K; r0 += DELTA_WG / 16) {
        const int row = r0 + (threadIdx.x >> 4);
        const bool in = row < K;
        float S[8], dS[8], e[8], o[8];
        columns8(dS0 ? dS0 + (int64_t)(in ? row : 0) * V : err, in && dS0, c0, V, dS);
#pragma nounroll
        for (int t = steps - 1; t >= 0; --t) {
            columns8(S0 ? S0 + (int64_t)(in ? row : 0) * V : err, in && S0, c0, V, S);
#pragma nounroll
            for (int j = 0; j < t; ++j) {                 // to the state before step t
                const float keep = keeps[j], kb = in ? (float)k[j * k_s + row] : 0.0f, beta = betas[j];
                columns8(err + j * row_s, true, c0, V, e);
#pragma unroll
                for (int u = 0; u < 8; ++u) S[u] = (keep != 0.0f ? keep * S[u] : 0.0f) + kb * (beta * e[u]);
            }
            const float keep = keeps[t], beta = betas[t], key = in ? (float)k[t * k_s + row] : 0.0f,
                        query = in ? scale * (float)q[t * q_s + row] : 0.0f;
            columns8(err + t * row_s, true, c0, V, e);
            columns8(d_o ? d_o + t * row_s : (const T*)err, d_o, c0, V, o);
            float dq = 0.0f, dk = 0.0f, dg = 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float z = 0.0f;
#pragma unroll
                for (int m = 0; m < NO; ++m) z += (float)Z.p[m * Z.plane + t * Z.ld + (c0 < V ? c0 : 0) + u];
                z = c0 + u < V ? z : 0.0f;
                S[u] = keep != 0.0f ? keep * S[u] : 0.0f;
                const float x = beta * e[u], y = beta * z, after = dS[u] + query * o[u], before = after - key * y;
                dq += (S[u] + key * x) * o[u];
                dk += after * x - S[u] * y;
                dg += S[u] * before;
                dS[u] = keep != 0.0f ? keep * before : 0.0f;
            }
            dq *= scale;
            if (!in) dg = 0.0f;
#pragma unroll
            for (int s = 1; s < 16; s <<= 1) {
                dq += __shfl_xor(dq, s);
                dk += __shfl_xor(dk, s);
            }
            for (int s = 1; s < 64; s <<= 1) dg += __shfl_xor(dg, s);
            if (lane == 0) rows[w * C + t] += dg;
            if (in && c0 == 0) {
                SameDelta& d = same_delta();
                SameGrad& gr = same_grad();
                const int64_t to = (((int64_t)b * d.T + t0 + t) * d.H + h) * K + row;
                if (d.H == d.Hk) {
                    ((T*)gr.d_q)[to] = (T)dq;
                    ((T*)gr.d_k)[to] = (T)dk;
                } else {
                    gr.head_grad[to] = dq;
                    gr.head_grad[(int64_t)d.B * d.T * d.H * K + to] = dk;
                }
            }
        }
    }
    __syncthreads();
    if (w == 0 && lane < steps) {
        const float dg = (rows[lane] + rows[C + lane]) + (rows[2 * C + lane] + rows[3 * C + lane]);
        put_gate_gradients<C>(same_delta(), same_grad(), b, h, t0 + lane, lane, gates, dg, sums.ez[lane]);
    }
}

// The gradients of q, k and the gates, one workgroup a chunk, robot and head: X, Z and dO as planes in LDS, D and M by tiles
// of 16 x 16, then a wave a tile of 16 key columns at a time. Bound by its matrix products and the LDS reads that feed them (the
// planes of 32-bit grade make three to six products of one). 300 x 77 x 6 heads of 40 x 56, float32: 169 us; 2 x 4096 x 8
// heads of 64 x 64, bfloat16: 52 us.
template <typename T, int C, int KP, bool VEC, bool WIDE>
__global__ __launch_bounds__(DELTA_WG, C == 32 && KP <= 64 ? (sizeof(T) == 2 && !WIDE ? 5 : 3) : 2)
void delta_chunk_kernel(InetDelta d, InetDeltaGrad gr) {
    constexpr int NP = Elem<T>::planes, NO = Grade<T, WIDE>::planes, LK = KP + 8;
    extern __shared__ char lds_raw[];
    const int vp = (d.V + 31) & ~31, lv = vp + 8;
    Gates<C>& gates = *(Gates<C>*)lds_raw;
    Sums<C>& sums = *(Sums<C>*)(lds_raw + sizeof(Gates<C>));
    __bf16* pool = (__bf16*)(lds_raw + sizeof(Gates<C>) + sizeof(Sums<C>));
    const Planes<NP> Kr{pool, LK, C * LK}, Qr{pool + NP * C * LK, LK, C * LK};
    __bf16* rows = pool + 2 * NP * C * LK;
    const Planes<NO> X{rows, lv, C * lv}, Z{rows + NO * C * lv, lv, C * lv};
    const Planes<NP> O{rows + 2 * NO * C * lv, lv, C * lv};
    const int chunks = (d.T + C - 1) / C, ch = blockIdx.x % chunks, t0 = ch * C;
    const int64_t bh = blockIdx.x / chunks, row_s = (int64_t)d.H * d.V;
    const int b = (int)(bh / d.H), h = (int)(bh % d.H), hk = h / (d.H / d.Hk), steps = d.T - t0;
    const int64_t row0 = ((int64_t)b * d.T + t0) * row_s + h * d.V;
    {
        Rows<T, C, KP, VEC> kr, qr;
        Gate gate;
        kr.load((const T*)d.k + b * d.k_s[0] + hk * d.k_s[2], d.k_s[1], t0, d.T, d.K);
        qr.load((const T*)d.q + b * d.q_s[0] + hk * d.q_s[2], d.q_s[1], t0, d.T, d.K);
        if (threadIdx.x < 64) {
            gate.load<C>(d, b, h, t0);
            put_gates<C>(gates, gate);
        }
        kr.put(Kr);
        qr.put(Qr);
    }
    stage_rows<T, C, VEC, NP>((const T*)gr.d_o, row0, row_s, steps, d.V, vp, O);
    __syncthreads();
    stage_errors<T, C, VEC, NO>(d, gr.err_grad, (T*)gr.d_v, row0, row_s, steps, vp, gates, X, Z, sums);
    __syncthreads();
    if (__builtin_expect(sums.odd[0] | sums.odd[1] | sums.odd[2] | sums.odd[3], 0)) {
        chunk_steps<T, C>(b, h, t0, Z, gates, sums, (float*)X.p);
        return;
    }
    const int64_t kv = (int64_t)d.K * d.V, at = bh * (chunks - 1) + ch;
    const float* S = ch ? d.chunk_state + (at - 1) * kv : d.state ? d.state + bh * kv : nullptr;
    const float* dS = ch + 1 < chunks ? gr.chunk_grad + at * kv : gr.d_state_out ? gr.d_state_out + bh * kv : nullptr;
    chunk_gradients<T, C, KP, VEC, NP, NO>(d, gr, b, h, t0, S, dS, gates, sums, Kr, Qr, X, Z, O, rows, vp);
}

// the one-chunk kernel's triangles P and L, in X's place until that is staged
template <int C> constexpr size_t triangles_lds() { return sizeof(__bf16) * 3 * C * (C + 8) + sizeof(float) * C * (C + 4); }
template <typename T, int C, int KP, int NO> constexpr size_t window_lds(int vp) {
    return chunk_lds<T, C, KP, NO>(vp, triangles_lds<C>());
}

// The whole backward pass of a window of at most C steps, one workgroup a robot and head: Z and what the scan would leave
// stay in LDS and registers, so S, dS, q, k, v and dO are read once. 16384 robots x 24 steps x 2 heads of 64 x 64, bfloat16: 700 us
// for 1.44 GB (2.1 TB/s); its waves wait for LDS and for each other's parts, four workgroups a compute unit.
template <typename T, int C, int KP, bool VEC, bool WIDE>
__global__ __launch_bounds__(DELTA_WG, C == 32 && KP <= 64 ? 3 : 2)
void delta_window_kernel(InetDelta d, InetDeltaGrad gr) {
    constexpr int NP = Elem<T>::planes, NO = Grade<T, WIDE>::planes, LK = KP + 8, LC = C + 8, LL = C + 4, RT = C / 16,
                  KT = KP / 16;
    extern __shared__ char lds_raw[];
    const int vp = (d.V + 31) & ~31, lv = vp + 8;
    Gates<C>& gates = *(Gates<C>*)lds_raw;
    Sums<C>& sums = *(Sums<C>*)(lds_raw + sizeof(Gates<C>));
    __bf16* pool = (__bf16*)(lds_raw + sizeof(Gates<C>) + sizeof(Sums<C>));
    const Planes<NP> Kr{pool, LK, C * LK}, Qr{pool + NP * C * LK, LK, C * LK};
    __bf16* rows = pool + 2 * NP * C * LK;
    const Planes<NO> Z{rows, lv, C * lv}, X{rows + (NO + NP) * C * lv, lv, C * lv};
    const Planes<NP> O{rows + NO * C * lv, lv, C * lv};
    const Planes<3> P{X.p, LC, C * LC};             // (X's place and after, until it is staged)
    float* ln = (float*)(P.p + 3 * C * LC);
    const int64_t bh = blockIdx.x, row_s = (int64_t)d.H * d.V, kv = (int64_t)d.K * d.V;
    const int b = blockIdx.x / d.H, h = blockIdx.x % d.H, hk = h / (d.H / d.Hk);
    const int64_t row0 = (int64_t)b * d.T * row_s + h * d.V;
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    {
        Rows<T, C, KP, VEC> kr, qr;
        Gate gate;
        kr.load((const T*)d.k + b * d.k_s[0] + hk * d.k_s[2], d.k_s[1], 0, d.T, d.K);
        qr.load((const T*)d.q + b * d.q_s[0] + hk * d.q_s[2], d.q_s[1], 0, d.T, d.K);
        if (w == 0) {
            gate.load<C>(d, b, h, 0);
            put_gates<C>(gates, gate);
        }
        kr.put(Kr);
        qr.put(Qr);
    }
    stage_rows<T, C, VEC, NP>((const T*)gr.d_o, row0, row_s, d.T, d.V, vp, O);
    __syncthreads();
    triangles<C, KP, NP, 3, true>(Kr, Qr, P, gates, ln, LL, d.scale, w, n, g);
    for (int c0 = 0; c0 < d.V; c0 += 64) {
        const int width = d.V - c0 < 64 ? d.V - c0 : 64;
        const bool mine = w * 16 + n < width;
        const uint32_t at = 4 * (uint32_t)(4 * g * d.V + w * 16 + n);
        if (c0 + w * 16 < vp) {                     // (columns from V up to vp: zeros)
            f32x4 z[RT] = {}, u[RT], S[KT] = {};
            if (mine && gr.d_state_out) state_load(S, gr.d_state_out + bh * kv + c0, at, d.V, d.K, g);
            column_gradients<C, KP, NP>(S, gr.d_state_out != nullptr, z, u, gates, ln, LL, Kr, P, O, c0 + w * 16, n, g);
            const bool sound = all_finite(z, gates.beta, g);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 4; ++e) Z.put1(rt * 16 + 4 * g + e, c0 + w * 16 + n, z[rt][e]);
            f32x4 old[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) old[kt] = S[kt];
            if (gr.d_state) state_gradient<C, KP, NP>(S, z, u, gates, d.scale, Kr, Qr, n, g);
            if (__builtin_expect(!sound, 0)) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) S[kt] = old[kt];
                SameDelta& a = same_delta();
                const T* d_o = (const T*)same_grad().d_o;
                const int col = w * 16 + n;
                for (int r = a.T + g; r < C; r += 4) Z.put1(r, c0 + col, 0.0f);
                steps_backward<C>(a, b, h, 0, (const T*)a.k + b * a.k_s[0] + hk * a.k_s[2],
                                  (const T*)a.q + b * a.q_s[0] + hk * a.q_s[2], d_o + row0 + c0, row_s, col, mine && d_o, S, g,
                                  [&](int t, float x) { Z.put1(t, c0 + col, x); });
            }
            if (mine && gr.d_state) state_store(S, gr.d_state + bh * kv + c0, at, d.V, d.K, g);
        }
    }
    __syncthreads();
    stage_errors<T, C, VEC, NO>(d, nullptr, (T*)gr.d_v, row0, row_s, d.T, vp, gates, X, Z, sums);
    __syncthreads();
    if (__builtin_expect(sums.odd[0] | sums.odd[1] | sums.odd[2] | sums.odd[3], 0)) {
        chunk_steps<T, C>(b, h, 0, Z, gates, sums, (float*)X.p);
        return;
    }
    chunk_gradients<T, C, KP, VEC, NP, NO>(d, gr, b, h, 0, d.state ? d.state + bh * kv : nullptr,
                                           gr.d_state_out ? gr.d_state_out + bh * kv : nullptr, gates, sums, Kr, Qr, X,
                                           Z, O, rows, vp);
}

// gradients of shared query and key heads: the value heads' own, summed in head order. Memory bounds it: 12 us for 59 MB
// (300 x 77 x 6 heads of 40 over 2, float32: 4.9 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void delta_heads_kernel(const float* __restrict__ x, T* __restrict__ q,
                                                          T* __restrict__ k, int64_t rows, int K, int rep) {
    const int64_t total = rows * K;                     // rows: B T Hk
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / K, c = i % K;
        float sq = 0.0f, sk = 0.0f;
        for (int r = 0; r < rep; ++r) {
            sq += x[(row * rep + r) * K + c];
            sk += x[total * rep + (row * rep + r) * K + c];
        }
        q[i] = (T)sq;
        k[i] = (T)sk;
    }
}

template <typename T, int C, int KP, bool VEC, bool WIDE>
static int launch(const InetDelta& d, const InetDeltaGrad& g, hipStream_t st) {
    constexpr int NO = Grade<T, WIDE>::planes;
    const int chunks = (d.T + C - 1) / C, vp = (d.V + 31) & ~31;
    static_assert(chunk_lds<T, C, KP, NO>(INET_POLICY_MAX_HEAD) <= LDS_MAX, "LDS");
    if (d.work) {
        if (int rc = delta_split(d, &g, VEC, st)) return rc;
    } else if constexpr (C == 32) {               // (chunks of 64 are for delta_split alone)
        static_assert(sizeof(ScanLds<T, C, KP>) <= LDS_MAX && window_lds<T, C, KP, NO>(INET_POLICY_MAX_HEAD) <= LDS_MAX, "LDS");
        if (chunks == 1) {
            auto window = delta_window_kernel<T, C, KP, VEC, WIDE>;
            const size_t lds = window_lds<T, C, KP, NO>(vp);
            if (allow_lds((const void*)window, lds)) return INET_POLICY_ELAUNCH;
            hipLaunchKernelGGL(window, dim3(d.B * d.H), dim3(DELTA_WG), lds, st, d, g);
        } else {
            auto scan = delta_scan_kernel<T, C, KP, VEC>;
            const size_t lds = sizeof(ScanLds<T, C, KP>);
            if (allow_lds((const void*)scan, lds)) return INET_POLICY_ELAUNCH;
            hipLaunchKernelGGL(scan, dim3(d.B * d.H, (d.V + 63) / 64), dim3(DELTA_WG), lds, st, d, g);
        }
        if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH;
    } else {
        return INET_POLICY_EINVAL;
    }
    if (!chunks) return INET_POLICY_OK;
    if (chunks > 1) {
        auto chunk = delta_chunk_kernel<T, C, KP, VEC, WIDE>;
        const size_t lds = chunk_lds<T, C, KP, NO>(vp);
        if (allow_lds((const void*)chunk, lds)) return INET_POLICY_ELAUNCH;
        hipLaunchKernelGGL(chunk, dim3(d.B * d.H * chunks), dim3(DELTA_WG), lds, st, d, g);
        if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH;
    }
    if (d.H != d.Hk) {
        const int64_t rows = (int64_t)d.B * d.T * d.Hk;
        hipLaunchKernelGGL(delta_heads_kernel<T>, dim3(blocks256(rows * d.K)), dim3(256), 0, st, g.head_grad, (T*)g.d_q,
                           (T*)g.d_k, rows, d.K, d.H / d.Hk);
    }
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

int delta_backward(const InetDelta& d, const InetDeltaGrad& g, bool vec, hipStream_t st) {
    return delta_dispatch(d, [&](auto t, auto c, auto kp) {
        typedef typename decltype(t)::type T;
        constexpr int C = decltype(c)::value, KP = decltype(kp)::value;
        if constexpr (!std::is_same<T, float>::value)
            if (d.gate_dtype == INET_POLICY_F32)
                return vec ? launch<T, C, KP, true, true>(d, g, st) : launch<T, C, KP, false, true>(d, g, st);
        return vec ? launch<T, C, KP, true, false>(d, g, st) : launch<T, C, KP, false, false>(d, g, st);
    });
}

}  // namespace pol
