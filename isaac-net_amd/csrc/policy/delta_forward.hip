// Forward pass of the gated delta rule over windows (the mathematics: delta.h).
#include "delta.h"
#include "delta_launch.h"

namespace pol {

template <typename T, int C, int KP> struct ForwardLds {
    static constexpr int NP = Elem<T>::planes, NO = Elem<T>::ord + 1, LK = KP + 8, LC = C + 8, LL = C + 4;
    Gates<C> gates;
    alignas(16) __bf16 k[NP * C * LK], q[NP * C * LK], p[NO * C * LC];
    alignas(16) float ln[C * LL];
    alignas(16) T v[C * LV], o[C * LV];
};

// One workgroup of four waves per robot, head and 64 columns; wave w owns 16 columns. Per chunk: K, Q and the gates to LDS,
// the triangles and the diagonal blocks' inverses by the waves in parts, then each wave's own columns through products whose
// results are the next one's operands in its registers. Chunks are short chains, so what bounds it is how many workgroups
// share a compute unit and wait in turn: three, within 168 registers (four, within 128, spill: 608 us for the 485 below), but
// two where float32's planes of 64 keys fill the LDS.
// 16384 robots x 24 steps x 2 heads of 64 x 64, bfloat16, state in and out: 485 us for the 1.48 GB it has to move (3.1 TB/s,
// where a copy makes 4.8) and 0.2 GB of errors kept; 300 x 77 x 6 heads of 40 x 56, float32: 116 us.
template <typename T, int C, int KP, bool VEC>
__global__ __launch_bounds__(DELTA_WG, 3 * sizeof(ForwardLds<T, C, KP>) <= LDS_MAX && KP <= 64 ? 3 : 2)
void delta_forward_kernel(InetDelta d) {
    constexpr int NP = Elem<T>::planes, ORD = Elem<T>::ord, NO = ORD + 1, RT = C / 16, KT = KP / 16;
    extern __shared__ char lds_raw[];
    typedef ForwardLds<T, C, KP> Lds;
    Lds& s = *(Lds*)lds_raw;
    const Planes<NP> Kr{s.k, Lds::LK, C * Lds::LK}, Qr{s.q, Lds::LK, C * Lds::LK};
    const Planes<NO> P{s.p, Lds::LC, C * Lds::LC};
    const int b = blockIdx.x / d.H, h = blockIdx.x % d.H, hk = h / (d.H / d.Hk);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.y * 64, width = d.V - c0 < 64 ? d.V - c0 : 64;      // the workgroup's columns
    const bool cols = w * 16 < width, mine = w * 16 + n < width;
    const T* q = (const T*)d.q + b * d.q_s[0] + hk * d.q_s[2];
    const T* k = (const T*)d.k + b * d.k_s[0] + hk * d.k_s[2];
    const T* v = (const T*)d.v + b * d.v_s[0] + h * d.v_s[2] + c0;
    const int chunks = (d.T + C - 1) / C;
    const int64_t bh = (int64_t)b * d.H + h, row_s = (int64_t)d.H * d.V, rows0 = b * (int64_t)d.T * row_s + h * d.V + c0;

    Rows<T, C, KP, VEC> kr, qr;
    Rows<T, C, 64, VEC> vr;
    Gate gate;
    auto fetch = [&](int t0) {
        kr.load(k, d.k_s[1], t0, d.T, d.K);
        qr.load(q, d.q_s[1], t0, d.T, d.K);
        vr.load(v, d.v_s[1], t0, d.T, width);
        if (w == 0) gate.load<C>(d, b, h, t0);
    };
    if (chunks) fetch(0);

    uint32_t at = 4 * (uint32_t)(4 * g * d.V + w * 16 + n), at_err = 4 * (uint32_t)(4 * g * row_s + w * 16 + n);
    f32x4 S[KT] = {};
    if (mine && d.state) state_load(S, d.state + bh * d.K * d.V + c0, at, d.V, d.K, g);

    for (int ch = 0; ch < chunks; ++ch) {
        const int t0 = ch * C;
        kr.put(Kr);
        qr.put(Qr);
        vr.put(s.v, LV);
        if (w == 0) put_gates<C>(s.gates, gate);
        __syncthreads();
        keep(at), keep(at_err);
        triangles<C, KP, NP, NO, false>(Kr, Qr, P, s.gates, s.ln, Lds::LL, d.scale, w, n, g);
        if (ch + 1 < chunks) fetch(t0 + C);
        if (cols) {
            if (d.chunk_state && ch && mine)
                state_store(S, d.chunk_state + (bh * (chunks - 1) + ch - 1) * d.K * d.V + c0, at, d.V, d.K, g);
            // K S to the last bits of 32, since the state goes on with it; Q S to the output's
            f32x4 x[RT] = {}, o[RT] = {};
#pragma unroll
            for (int kp = 0; kp < KT / 2; ++kp) {
                const Frag<3> sf = split_tiles<3>(S[2 * kp], S[2 * kp + 1]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    x[rt] = mma<2>(Kr.frag(rt * 16 + n, kp * 32 + 8 * g), sf, x[rt]);
                    o[rt] = mma<ORD>(Qr.frag(rt * 16 + n, kp * 32 + 8 * g), sf, o[rt]);
                }
            }
            // the errors; then X = beta E
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const f32x4 a = *(const f32x4*)(s.gates.a + rt * 16 + 4 * g), vt = tile_at(s.v + rt * 16 * LV + w * 16, LV, n, g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[rt][e] = vt[e] - (a[e] != 0.0f ? a[e] * x[rt][e] : 0.0f);
                    o[rt][e] = a[e] != 0.0f ? d.scale * a[e] * o[rt][e] : 0.0f;
                }
            }
            solve_down<C>(x, s.ln, Lds::LL, n, g);
            const bool sound = all_finite(x, s.gates.beta, g);
            if (d.err && mine) rows_store(x, d.err + rows0 + t0 * row_s, at_err, row_s, d.T - t0, g);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) x[rt] *= *(const f32x4*)(s.gates.beta + rt * 16 + 4 * g);
#pragma unroll
            for (int kp = 0; kp < RT / 2; ++kp) {
                const Frag<NO> xf = split_tiles<NO>(x[2 * kp], x[2 * kp + 1]);
#pragma unroll
                for (int rt = 2 * kp; rt < RT; ++rt)
                    o[rt] = mma<ORD>(P.frag(rt * 16 + n, kp * 32 + 8 * g), xf, o[rt]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) tile_put(s.o + rt * 16 * LV + w * 16, LV, n, g, o[rt]);
            const float a_end = s.gates.a_end;
            f32x4 old[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                old[kt] = S[kt];
#pragma unroll
                for (int e = 0; e < 4; ++e) S[kt][e] = a_end != 0.0f ? a_end * S[kt][e] : 0.0f;
            }
#pragma unroll
            for (int kp = 0; kp < RT / 2; ++kp) {
                const f32x4 c0 = *(const f32x4*)(s.gates.c + kp * 32 + 4 * g),
                            c1 = *(const f32x4*)(s.gates.c + kp * 32 + 16 + 4 * g);
                const Frag<3> xf = split_tiles<3>(x[2 * kp] * c0, x[2 * kp + 1] * c1);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) S[kt] = mma<2>(Kr.tr_frag(kt, kp, n, g), xf, S[kt]);
            }
            if (__builtin_expect(!sound, 0)) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // (the errors are stored once more)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) S[kt] = old[kt];
                const int col = w * 16 + n;
                SameDelta& a = same_delta();
                steps_forward<C, true>(a, b, h, t0, k, q, v, a.v_s[1], col, mine, S, g, [&](int t, float err, float out) {
                    s.o[t * LV + col] = (T)out;
                    if (a.err && mine) a.err[rows0 + (t0 + t) * row_s + col] = err;
                });
            }
        }
        __syncthreads();
        store_rows<T, C, VEC>(s.o, (T*)d.o + rows0 + t0 * row_s, row_s, d.T - t0, width);
    }
    if (mine) state_store(S, d.state_out + bh * d.K * d.V + c0, at, d.V, d.K, g);
}

template <typename T, int C, int KP, bool VEC> static int launch(const InetDelta& d, hipStream_t st) {
    const size_t lds = sizeof(ForwardLds<T, C, KP>);
    static_assert(sizeof(ForwardLds<T, C, KP>) <= LDS_MAX, "LDS");
    auto k = delta_forward_kernel<T, C, KP, VEC>;
    if (allow_lds((const void*)k, lds)) return INET_POLICY_ELAUNCH;
    hipLaunchKernelGGL(k, dim3(d.B * d.H, (d.V + 63) / 64), dim3(DELTA_WG), lds, st, d);
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

int delta_forward(const InetDelta& d, bool vec, hipStream_t st) {
    if (d.work) return delta_split(d, nullptr, vec, st);
    return delta_dispatch(d, [&](auto t, auto c, auto kp) {
        typedef typename decltype(t)::type T;
        constexpr int C = decltype(c)::value, KP = decltype(kp)::value;
        if constexpr (C == 32) return vec ? launch<T, C, KP, true>(d, st) : launch<T, C, KP, false>(d, st);
        return INET_POLICY_EINVAL;                // (chunks of 64 are for delta_split alone)
    });
}

}  // namespace pol
