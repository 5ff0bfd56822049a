// Forward pass of the gated delta rule over windows (the mathematics: delta.h).
#include "delta.h"
#include "delta_launch.h"

namespace pol {

template <typename T, int C, int KP> struct ForwardLds {
    static constexpr int NP = Elem<T>::planes, NO = Elem<T>::ord + 1, LK = KP + 8, LC = C + 8, LL = C + 4;
    Gates<C> gates;
    alignas(16) __bf16 k[NP * C * LK], q[NP * C * LK], kt[NP * KP * LC], p[NO * C * LC];
    alignas(16) float ln[C * LL];
};

// One workgroup of four waves per robot, head and 64 NV columns; wave w owns NV tiles of 16 columns.
template <typename T, int C, int KP, int NV>
__global__ __launch_bounds__(DELTA_WG) void delta_forward_kernel(InetDelta d, int vec) {
    constexpr int NP = Elem<T>::planes, ORD = Elem<T>::ord, NO = ORD + 1, RT = C / 16, KT = KP / 16;
    extern __shared__ char lds_raw[];
    typedef ForwardLds<T, C, KP> Lds;
    Lds& s = *(Lds*)lds_raw;
    const Planes<NP> Kr{s.k, Lds::LK, C * Lds::LK}, Qr{s.q, Lds::LK, C * Lds::LK}, Kt{s.kt, Lds::LC, KP * Lds::LC};
    const Planes<NO> P{s.p, Lds::LC, C * Lds::LC};
    const int b = blockIdx.x / d.H, h = blockIdx.x % d.H, hk = h / (d.H / d.Hk);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int col0 = (blockIdx.y * 4 + w) * NV * 16 + n;
    const bool cols = (blockIdx.y * 4 + w) * NV * 16 < d.V;
    const T* q = (const T*)d.q + b * d.q_s[0] + hk * d.q_s[2];
    const T* k = (const T*)d.k + b * d.k_s[0] + hk * d.k_s[2];
    const T* v = (const T*)d.v + b * d.v_s[0] + h * d.v_s[2];
    const int chunks = (d.T + C - 1) / C;
    const int64_t bh = (int64_t)b * d.H + h;

    f32x4 S[KT][NV] = {};
    if (cols && d.state)
        for (int kt = 0; kt < KT; ++kt)
            for (int nv = 0; nv < NV; ++nv)
                for (int e = 0; e < 4; ++e) {
                    const int row = kt * 16 + 4 * g + e, col = col0 + 16 * nv;
                    if (row < d.K && col < d.V) S[kt][nv][e] = d.state[(bh * d.K + row) * d.V + col];
                }

    for (int ch = 0; ch < chunks; ++ch) {
        const int t0 = ch * C;
        stage<T, C, KP, NP, true, true>(k, d.k_s[1], t0, d.T, d.K, vec & 1, Kr, Kt);
        stage<T, C, KP, NP, true, false>(q, d.q_s[1], t0, d.T, d.K, vec & 2, Qr, Qr);
        if (w == 0) load_gates<C>(s.gates, d, b, h, t0);
        __syncthreads();
        // the triangles: row tile rt of K K^T (jobs 0 .. RT - 1) and of Q K^T (RT .. 2 RT - 1, in the opposite order,
        // so that a wave has as many tiles of the one as it lacks of the other)
        for (int job = w; job < 2 * RT; job += 4) {
            const bool qk = job >= RT;
            const int rt = qk ? 2 * RT - 1 - job : job;
#pragma unroll
            for (int ct = 0; ct < RT; ++ct) {
                if (ct > rt && !(qk && ct == rt + 1 && (ct & 1))) continue;
                f32x4 acc = {};
                if (ct <= rt)
                    for (int k8 = 0; k8 < KP; k8 += 32)
                        acc = mma<2>((qk ? Qr : Kr).frag(rt * 16 + n, k8 + 8 * g), Kr.frag(ct * 16 + n, k8 + 8 * g),
                                     acc);
                const int j = ct * 16 + n;
                for (int e = 0; e < 4; ++e) {
                    const int i = rt * 16 + 4 * g + e;
                    if (qk) P.put(i, perm(j), i >= j ? acc[e] * d.scale * decay(s.gates, i, j) : 0.0f);
                    else s.ln[i * Lds::LL + j] = i > j ? -acc[e] * s.gates.beta[j] * decay(s.gates, i, j) : 0.0f;
                }
            }
        }
        __syncthreads();
        invert_blocks<C>(s.ln, Lds::LL);
        __syncthreads();
        if (cols) {
            if (d.chunk_state)
                for (int kt = 0; kt < KT; ++kt)
                    for (int nv = 0; nv < NV; ++nv)
                        for (int e = 0; e < 4; ++e) {
                            const int row = kt * 16 + 4 * g + e, col = col0 + 16 * nv;
                            if (row < d.K && col < d.V)
                                d.chunk_state[((bh * chunks + ch) * d.K + row) * d.V + col] = S[kt][nv][e];
                        }
            // K S to the last bits of 32, since the state goes on with it; Q S to the output's
            f32x4 ks[RT][NV] = {}, qs[RT][NV] = {};
#pragma unroll
            for (int kp = 0; kp < KT / 2; ++kp)
#pragma unroll
                for (int nv = 0; nv < NV; ++nv) {
                    const Frag<3> sf = split_tiles<3>(S[2 * kp][nv], S[2 * kp + 1][nv]);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        ks[rt][nv] = mma<2>(Kr.frag(rt * 16 + n, kp * 32 + 8 * g), sf, ks[rt][nv]);
                        qs[rt][nv] = mma<ORD>(Qr.frag(rt * 16 + n, kp * 32 + 8 * g), sf, qs[rt][nv]);
                    }
                }
            // the errors, block row by block row
            f32x4 x[RT][NV];
#pragma unroll
            for (int nv = 0; nv < NV; ++nv) {
                const int col = col0 + 16 * nv;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    f32x4 acc;
                    for (int e = 0; e < 4; ++e) {
                        const int i = rt * 16 + 4 * g + e, t = t0 + i;
                        const float vv = t < d.T && col < d.V ? (float)v[t * d.v_s[1] + col] : 0.0f, a = s.gates.a[i];
                        acc[e] = a != 0.0f ? vv - a * ks[rt][nv][e] : vv;
                    }
#pragma unroll
                    for (int m = 0; m < rt; ++m)
                        acc = mma32(*(const f32x4*)(s.ln + (rt * 16 + n) * Lds::LL + m * 16 + 4 * g), x[m][nv], acc);
                    x[rt][nv] = mma32(*(const f32x4*)(s.ln + (rt * 16 + n) * Lds::LL + rt * 16 + 4 * g), acc, f32x4{});
                }
                if (d.err)
                    for (int rt = 0; rt < RT; ++rt)
                        for (int e = 0; e < 4; ++e) {
                            const int t = t0 + rt * 16 + 4 * g + e;
                            if (t < d.T && col < d.V)
                                d.err[(((int64_t)b * d.T + t) * d.H + h) * d.V + col] = x[rt][nv][e];
                        }
            }
            // (X = beta E from here on)
            for (int rt = 0; rt < RT; ++rt)
                for (int nv = 0; nv < NV; ++nv)
                    for (int e = 0; e < 4; ++e) x[rt][nv][e] *= s.gates.beta[rt * 16 + 4 * g + e];
#pragma unroll
            for (int nv = 0; nv < NV; ++nv) {
                const int col = col0 + 16 * nv;
                Frag<NO> xf[RT / 2];
                for (int kp = 0; kp < RT / 2; ++kp) xf[kp] = split_tiles<NO>(x[2 * kp][nv], x[2 * kp + 1][nv]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    f32x4 acc;
                    for (int e = 0; e < 4; ++e) {
                        const float a = s.gates.a[rt * 16 + 4 * g + e];
                        acc[e] = a != 0.0f ? d.scale * a * qs[rt][nv][e] : 0.0f;
                    }
#pragma unroll
                    for (int kp = 0; kp <= rt / 2; ++kp)
                        acc = mma<ORD>(P.frag(rt * 16 + n, kp * 32 + 8 * g), xf[kp], acc);
                    for (int e = 0; e < 4; ++e) {
                        const int t = t0 + rt * 16 + 4 * g + e;
                        if (t < d.T && col < d.V)
                            ((T*)d.o)[(((int64_t)b * d.T + t) * d.H + h) * d.V + col] = (T)acc[e];
                    }
                }
            }
            const float a_end = s.gates.a_end;
#pragma unroll
            for (int nv = 0; nv < NV; ++nv) {
                Frag<3> xf[RT / 2];
                for (int kp = 0; kp < RT / 2; ++kp) {
                    f32x4 u = x[2 * kp][nv], l = x[2 * kp + 1][nv];
                    for (int e = 0; e < 4; ++e) {
                        u[e] *= s.gates.c[kp * 32 + 4 * g + e];
                        l[e] *= s.gates.c[kp * 32 + 16 + 4 * g + e];
                    }
                    xf[kp] = split_tiles<3>(u, l);
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    for (int e = 0; e < 4; ++e) S[kt][nv][e] = a_end != 0.0f ? a_end * S[kt][nv][e] : 0.0f;
#pragma unroll
                    for (int kp = 0; kp < RT / 2; ++kp)
                        S[kt][nv] = mma<2>(Kt.frag(kt * 16 + n, kp * 32 + 8 * g), xf[kp], S[kt][nv]);
                }
            }
        }
        __syncthreads();
    }
    if (cols)
        for (int kt = 0; kt < KT; ++kt)
            for (int nv = 0; nv < NV; ++nv)
                for (int e = 0; e < 4; ++e) {
                    const int row = kt * 16 + 4 * g + e, col = col0 + 16 * nv;
                    if (row < d.K && col < d.V) d.state_out[(bh * d.K + row) * d.V + col] = S[kt][nv][e];
                }
}

template <typename T, int C, int KP, int NV> static int launch(const InetDelta& d, int vec, hipStream_t st) {
    const size_t lds = sizeof(ForwardLds<T, C, KP>);
    static_assert(sizeof(ForwardLds<T, C, KP>) <= LDS_MAX, "LDS");
    auto k = delta_forward_kernel<T, C, KP, NV>;
    if (allow_lds((const void*)k, lds)) return INET_POLICY_ELAUNCH;
    hipLaunchKernelGGL(k, dim3(d.B * d.H, (d.V + 64 * NV - 1) / (64 * NV)), dim3(DELTA_WG), lds, st, d, vec);
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

int delta_forward(const InetDelta& d, int vec, hipStream_t st) {
    return delta_dispatch(d, [&](auto t, auto c, auto kp) {
        typedef typename decltype(t)::type T;
        return launch<T, decltype(c)::value, decltype(kp)::value, 1>(d, vec, st);
    });
}

}  // namespace pol
