// The gated delta rule over windows: chunk mathematics shared by the forward and the backward kernels.
//
// Within a chunk of C steps, with G_i the sum of the log-decays to step i, Gam_ij = e^{G_i - G_j} (0 across a reset),
// a_i = e^{G_i} from the chunk's start (0 after a reset), c_i = e^{G_C - G_i} to its end (0 before a reset), and S the
// state at its start:
//     forward    (I + L') E = V - a K S,   L'_ij = (k_i . k_j) Gam_ij beta_j  (i > j)      the prediction errors
//                X = beta E,  P_ij = scale (q_i . k_j) Gam_ij (i >= j)
//                O = scale a Q S + P X,    S <- a_C S + K^T (c X)
//     backward   dX = P^T dO + c K dS,     (I + L)^T Z = dX,   L_ij = beta_i (k_i . k_j) Gam_ij
//                dV = beta Z,  Y = -a dV,  dS <- a_C dS + Q^T (scale a dO) + K^T Y
//                D_ij = scale Gam_ij (dO_i . X_j) (i >= j),  M_ij = -beta_i Gam_ij (Z_i . X_j) (i > j)
//                dQ = scale a dO S^T + D K
//                dK = [Y S^T + M K] + [c X dS^T + D^T Q + M^T K] = dK+ + dK-
//                dbeta_i = E_i . Z_i,   dG_i = q_i . dQ_i + k_i . dK+_i - k_i . dK-_i  (+ at the chunk's last step the
//                state's share sum_i c_i k_i . (dS X_i) + a_C <S, dS>),  dg_t = the sum of dG_i over i >= t up to the
//                next reset
// (the triangular system in the errors rather than in X keeps dbeta free of a division by beta).
//
// The columns of S, E, X, Z and dS are independent of each other: a wave owns tiles of 16 columns and takes the state
// through the whole window in its registers, as matrix-instruction results that are the next product's operands in
// place. What the waves share per chunk, K, Q and the C x C triangles, is in LDS. The triangular systems go by blocks of
// 16: the diagonal blocks are inverted by substitution (stable where a robot's keys hardly change from step to step),
// the blocks below enter by 32-bit matrix instructions.
//
// The log-decays' sums are held in 64 bits: their differences stay exact to 32 bits whatever the chunk has decayed by.
#pragma once
#include "policy_dev.h"
#include "../../../include/inet_policy.h"

namespace pol {

constexpr int DELTA_WG = 256;
constexpr double DECAY_MIN = -104.0;     // e^-104 is 0 in 32 bits: the memory is emptied

// per chunk and head: the gates, in LDS
template <int C> struct alignas(16) Gates {
    double G[C];
    int seg[C];
    float a[C], c[C], beta[C];
    float a_end;
};

template <typename T> DEV float gate_at(const void* p, int64_t i) { return (float)((const T*)p)[i]; }
DEV float gate_load(const void* p, int64_t i, int dtype) {
    return dtype == INET_POLICY_F32 ? gate_at<float>(p, i) : dtype == INET_POLICY_BF16 ? gate_at<__bf16>(p, i)
                                                                                       : gate_at<_Float16>(p, i);
}

// wave 0: the chunk's gates from step t0 on (steps from T on: no decay, nothing written)
template <int C> DEV void load_gates(Gates<C>& s, const InetDelta& d, int b, int h, int t0) {
    const int lane = threadIdx.x & 63, t = t0 + lane;
    double g = 0.0;
    float beta = 0.0f;
    int cut = 0;
    if (lane < C && t < d.T) {
        const float gf = gate_load(d.g, b * d.g_s[0] + t * d.g_s[1] + h * d.g_s[2], d.gate_dtype);
        beta = gate_load(d.beta, b * d.beta_s[0] + t * d.beta_s[1] + h * d.beta_s[2], d.gate_dtype);
        cut = (d.reset && d.reset[b * d.reset_s[0] + t * d.reset_s[1]]) || (double)gf < DECAY_MIN;
        g = cut ? 0.0 : (double)gf;
    }
    for (int o = 1; o < C; o <<= 1) {
        const double u = __shfl_up(g, o);
        const int v = __shfl_up(cut, o);
        if (lane >= o) { g += u; cut += v; }
    }
    const double g_end = __shfl(g, C - 1);
    const int seg_end = __shfl(cut, C - 1);
    if (lane < C) {
        s.G[lane] = g;
        s.seg[lane] = cut;
        s.beta[lane] = beta;
        s.a[lane] = cut == 0 ? expf((float)g) : 0.0f;
        s.c[lane] = cut == seg_end ? expf((float)(g_end - g)) : 0.0f;
        if (lane == 0) s.a_end = seg_end == 0 ? expf((float)g_end) : 0.0f;
    }
}

// Gam_ij
template <int C> DEV float decay(const Gates<C>& s, int i, int j) {
    return s.seg[i] == s.seg[j] ? expf((float)(s.G[i] - s.G[j])) : 0.0f;
}

// rows t0 .. t0 + C - 1 of x [steps][K] (row stride st) into planes in the order perm(), and, where TR, transposed
template <typename T, int C, int KP, int N, bool ROWS, bool TR>
DEV void stage(const T* __restrict__ x, int64_t st, int t0, int t_end, int K, bool vec, const Planes<N>& rows,
               const Planes<N>& tr) {
    for (int i = threadIdx.x; i < C * (KP / 8); i += DELTA_WG) {
        const int r = i / (KP / 8), c = i % (KP / 8) * 8;
        float v[8] = {};
        if (t0 + r < t_end && c < K) load8(x + (t0 + r) * st + c, K - c, vec, v);
        if (ROWS) {
            rows.put4(r, perm(c), v[0], v[1], v[2], v[3]);
            rows.put4(r, perm(c + 4), v[4], v[5], v[6], v[7]);
        }
        if (TR)
            for (int e = 0; e < 8; ++e) tr.put(c + e, perm(r), v[e]);
    }
}

// the 16 x 16 diagonal blocks of I + L (L's negative in Ln, row-major, rows of ld) replaced by their inverses: wave w
// takes block w; lane n of each 16 solves for column n by forward substitution
template <int C> DEV void invert_blocks(float* Ln, int ld) {
    const int w = threadIdx.x >> 6, n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    if (w >= C / 16) return;
    float* B = Ln + (w * 16) * ld + w * 16;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float s = i == n ? 1.0f : 0.0f;
#pragma unroll
        for (int m4 = 0; m4 < (i + 3) / 4; ++m4) {
            const f32x4 l = *(const f32x4*)(B + i * ld + 4 * m4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * m4 + e < i) s += l[e] * x[4 * m4 + e];
        }
        x[i] = s;
    }
    // (the wave's lanes have read the block before any of them writes: one wave, in order)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if ((i >> 2) == g) B[i * ld + n] = x[i];
}

}  // namespace pol
