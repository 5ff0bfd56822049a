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
//
// A chunk's products take every step with every other, those that may not see each other by a factor of zero, which an
// infinity or NaN passes (0 x NaN). So where a chunk's rows X or Z are not finite, its 16 columns go by single steps
// (steps_forward, steps_backward): what is wrong stays with its episode, and with the steps that follow it.
#pragma once
#include "policy_dev.h"
#include "../../../include/inet_policy.h"

namespace pol {

constexpr int DELTA_WG = 256;
constexpr double DECAY_MIN = -104.0;     // e^-104 is 0 in 32 bits: the memory is emptied

// per chunk and head: the gates, in LDS. Gam_ij of a step i and a step j of an earlier tile of 16 is in[i] out[tile of
// i][j], through the last step before i's tile (for decays both factors are at most 1).
template <int C> struct alignas(16) Gates {
    double G[C];
    float a[C], c[C], beta[C], in[C], out[C / 16][C];
    int seg[C];
    float a_end;
};

template <typename T> DEV float gate_at(const void* p, int64_t i) { return (float)((const T*)p)[i]; }
DEV float gate_load(const void* p, int64_t i, int dtype) {
    return dtype == INET_POLICY_F32 ? gate_at<float>(p, i) : dtype == INET_POLICY_BF16 ? gate_at<__bf16>(p, i)
                                                                                       : gate_at<_Float16>(p, i);
}

// lane i's step of a chunk, as loaded (steps from T on: no decay, nothing written)
struct Gate {
    float g = 0.0f, beta = 0.0f;
    int cut = 0;
    template <int C> DEV void load(const InetDelta& d, int b, int h, int t0) {
        const int lane = threadIdx.x & 63, t = t0 + lane;
        g = beta = 0.0f;
        cut = 0;
        if (lane < C && t < d.T) {
            g = gate_load(d.g, b * d.g_s[0] + t * d.g_s[1] + h * d.g_s[2], d.gate_dtype);
            beta = gate_load(d.beta, b * d.beta_s[0] + t * d.beta_s[1] + h * d.beta_s[2], d.gate_dtype);
            if (d.reset) cut = d.reset[b * d.reset_s[0] + t * d.reset_s[1]];
        }
    }
};

// one wave: the chunk's gates
template <int C> DEV void put_gates(Gates<C>& s, const Gate& x) {
    const int lane = threadIdx.x & 63;
    const bool empty = x.cut != 0 || (double)x.g < DECAY_MIN;
    const double g = lane_scan(empty ? 0.0 : (double)x.g);
    const int seg = lane_scan(empty ? 1 : 0);
    const double g_end = __shfl(g, C - 1);
    const int seg_end = __shfl(seg, C - 1), to = (lane & ~15) - 1;
    const double g_in = __shfl(g, to);                            // (of the first tile: not used)
    const int seg_in = __shfl(seg, to);
#pragma unroll
    for (int r = 1; r < C / 16; ++r) {
        const double g_r = __shfl(g, 16 * r - 1);
        const int seg_r = __shfl(seg, 16 * r - 1);
        if (lane < 16 * r) s.out[r][lane] = seg == seg_r ? expf((float)(g_r - g)) : 0.0f;
    }
    if (lane < C) {
        s.G[lane] = g;
        s.seg[lane] = seg;
        s.beta[lane] = x.beta;
        s.a[lane] = seg == 0 ? expf((float)g) : 0.0f;
        s.c[lane] = seg == seg_end ? expf((float)(g_end - g)) : 0.0f;
        s.in[lane] = lane >= 16 && seg == seg_in ? expf((float)(g - g_in)) : 0.0f;
        if (lane == 0) s.a_end = seg_end == 0 ? expf((float)g_end) : 0.0f;
    }
}

// Gam_ij for step i and steps j .. j + 3, 4 g + e of a tile; DIAG: of the same tile of 16, j <= i alone
template <int C, bool DIAG> DEV f32x4 decay4(const Gates<C>& s, int i, int j) {
    f32x4 x;
    if constexpr (DIAG) {
        const double gi = s.G[i];
        const int si = s.seg[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = j + e <= i && s.seg[j + e] == si ? expf((float)(gi - s.G[j + e])) : 0.0f;
    } else {
        x = *(const f32x4*)(s.out[i >> 4] + j) * s.in[i];
    }
    return x;
}

// C rows of x [steps][K] (row stride st) on their way from memory to LDS: load() and, when the rows of the chunk before
// are done with, put()
// (VEC: rows start on 16 bytes and hold whole groups of eight)
template <typename T, int C, int KP, bool VEC> struct Rows {
    static constexpr int GR = C * (KP / 8), NL = (GR + DELTA_WG - 1) / DELTA_WG;
    typedef T V8 __attribute__((ext_vector_type(8)));
    V8 v[NL];
    int tid = threadIdx.x;                               // (of the DELTA_WG that load together)
    DEV void load(const T* __restrict__ x, int64_t st, int t0, int t_end, int K) {
#pragma unroll
        for (int m = 0; m < NL; ++m) {
            const int i = tid + m * DELTA_WG, r = i / (KP / 8), c = i % (KP / 8) * 8;
            v[m] = V8{};
            if (i < GR && t0 + r < t_end && c < K) {
                const T* p = x + (t0 + r) * st + c;
                if constexpr (VEC) v[m] = *(const V8*)p;
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c + e < K) v[m][e] = p[e];
            }
        }
    }
    DEV void put(T* s, int ld) const {                            // as they are
#pragma unroll
        for (int m = 0; m < NL; ++m) {
            const int i = tid + m * DELTA_WG, r = i / (KP / 8), c = i % (KP / 8) * 8;
            if (GR % DELTA_WG == 0 || i < GR) *(V8*)(s + r * ld + c) = v[m];
        }
    }
    template <int N> DEV void put_natural(const Planes<N>& s) const {       // columns in their own order
#pragma unroll
        for (int m = 0; m < NL; ++m) {
            const int i = tid + m * DELTA_WG, r = i / (KP / 8), c = i % (KP / 8) * 8;
            if (GR % DELTA_WG == 0 || i < GR) {
                s.put4(r, c, (float)v[m][0], (float)v[m][1], (float)v[m][2], (float)v[m][3]);
                s.put4(r, c + 4, (float)v[m][4], (float)v[m][5], (float)v[m][6], (float)v[m][7]);
            }
        }
    }
    template <int N> DEV void put(const Planes<N>& s) const {
#pragma unroll
        for (int m = 0; m < NL; ++m) {
            const int i = tid + m * DELTA_WG, r = i / (KP / 8), c = i % (KP / 8) * 8;
            if (GR % DELTA_WG == 0 || i < GR) {
                s.put4(r, perm(c), (float)v[m][0], (float)v[m][1], (float)v[m][2], (float)v[m][3]);
                s.put4(r, perm(c + 4), (float)v[m][4], (float)v[m][5], (float)v[m][6], (float)v[m][7]);
            }
        }
    }
};

// a 16 x 16 tile of values in LDS (rows of ld, the tile at s) as a matrix instruction's result: lane column n, rows 4 g + e
template <typename T> DEV f32x4 tile_at(const T* s, int ld, int n, int g) {
    f32x4 x;
    if constexpr (sizeof(T) == 2) {
        typedef T V4 __attribute__((ext_vector_type(4)));
        const V4 v = __builtin_bit_cast(V4, read_tr((const __bf16*)s + (4 * g + (n >> 2)) * ld + (n & 3) * 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = s[(4 * g + e) * ld + n];
    }
    return x;
}

// 16 x 16 values from planes (columns in their own order) as a result's tile
template <int N> DEV f32x4 plane_tile(const Planes<N>& s, int row0, int c0, int n, int g) {
    f32x4 x = {};
#pragma unroll
    for (int m = N - 1; m >= 0; --m)
        x += tile_at<__bf16>(s.p + m * s.plane + row0 * s.ld + c0, s.ld, n, g);
    return x;
}

// such a result to LDS, rounded to T
template <typename T> DEV void tile_put(T* s, int ld, int n, int g, f32x4 x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[(4 * g + e) * ld + n] = (T)x[e];
}

// C rows of 64 columns from LDS (rows of LV) to out [steps][heads][V], out at the first step, this head and these columns
constexpr int LV = 64 + 8;
template <typename T, int C, bool VEC> DEV void store_rows(const T* s, T* __restrict__ out, int64_t st, int steps, int cols) {
    typedef T V8 __attribute__((ext_vector_type(8)));
    for (int i = threadIdx.x; i < C * 8; i += DELTA_WG) {
        const int r = i / 8, c = i % 8 * 8;
        if (r < steps && c < cols) {
            const V8 v = *(const V8*)(s + r * LV + c);
            T* p = out + r * st + c;
            if constexpr (VEC) *(V8*)p = v;
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < cols) p[e] = v[e];
        }
    }
}

// the state's tiles of 16 columns, from and to [K][V] at the first of the columns; off: row 4 g, column n, in bytes.
// (p and what is added to it is the same in all lanes, so an access is a base, one offset for all, and no arithmetic)
template <typename P> DEV P at_byte(P p, uint32_t off) { return (P)((uintptr_t)p + off); }
template <int KT> DEV void state_load(f32x4 (&S)[KT], const float* __restrict__ p, uint32_t off, int V, int K, int g) {
    if (K == KT * 16) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[kt][e] = *at_byte(p + (kt * 16 + e) * V, off);
    } else {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[kt][e] = kt * 16 + 4 * g + e < K ? *at_byte(p + (kt * 16 + e) * V, off) : 0.0f;
    }
}
template <int KT> DEV void state_store(const f32x4 (&S)[KT], float* __restrict__ p, uint32_t off, int V, int K, int g) {
    if (K == KT * 16) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) *at_byte(p + (kt * 16 + e) * V, off) = S[kt][e];
    } else {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (kt * 16 + 4 * g + e < K) *at_byte(p + (kt * 16 + e) * V, off) = S[kt][e];
    }
}
// the same for 16 columns of a chunk's rows (row_s apart), `left` of them inside the window
template <int RT> DEV void rows_load(f32x4 (&x)[RT], const float* __restrict__ p, uint32_t off, int64_t row_s, int left, int g) {
    if (left >= RT * 16) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[rt][e] = *at_byte(p + (rt * 16 + e) * row_s, off);
    } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[rt][e] = rt * 16 + 4 * g + e < left ? *at_byte(p + (rt * 16 + e) * row_s, off) : 0.0f;
    }
}
template <int RT> DEV void rows_store(const f32x4 (&x)[RT], float* __restrict__ p, uint32_t off, int64_t row_s, int left, int g) {
    if (left >= RT * 16) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e) *at_byte(p + (rt * 16 + e) * row_s, off) = x[rt][e];
    } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (rt * 16 + 4 * g + e < left) *at_byte(p + (rt * 16 + e) * row_s, off) = x[rt][e];
    }
}

// keeps what is computed from x inside the loop: addresses are cheaper to compute again than to hold in registers
DEV void keep(uint32_t& x) { asm volatile("" : "+v"(x)); }
// the same for what is equal in all lanes
template <typename X> DEV void keep_same(X& x) { asm volatile("" : "+s"(x)); }

// tile row it of the triangles: -L (in Ln, f32, rows of ld) from K K^T, or P from Q K^T. The products are taken
// transposed (K's rows as A), so that a lane holds four steps j of one step i. ROWS_BETA: L_ij takes beta_i, else beta_j.
template <int C, int KP, int NP, bool ROWS_BETA>
DEV void triangle_l(const Planes<NP>& Kr, const Gates<C>& gt, float* ln, int ld, int it, int n, int g) {
    const int i = it * 16 + n;
#pragma unroll
    for (int jt = 0; jt < C / 16; ++jt) {
        if (jt > it) continue;
        f32x4 acc = {};
#pragma unroll
        for (int k8 = 0; k8 < KP; k8 += 32)
            acc = mma<2>(Kr.frag(jt * 16 + n, k8 + 8 * g), Kr.frag(i, k8 + 8 * g), acc);
        const int j = jt * 16 + 4 * g;
        const f32x4 dec = jt == it ? decay4<C, true>(gt, i, j) : decay4<C, false>(gt, i, j);
        f32x4 b = *(const f32x4*)(gt.beta + j);
        if (ROWS_BETA) b = f32x4{1, 1, 1, 1} * gt.beta[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = j + e < i ? -acc[e] * dec[e] * b[e] : 0.0f;
        *(f32x4*)(ln + i * ld + j) = acc;
    }
}
template <int C, int KP, int NP, int NO>
DEV void triangle_p(const Planes<NP>& Kr, const Planes<NP>& Qr, const Planes<NO>& P, const Gates<C>& gt, float scale,
                    int it, int n, int g) {
    const int i = it * 16 + n;
#pragma unroll
    for (int jt = 0; jt < C / 16; ++jt) {
        const int j = jt * 16 + 4 * g;
        if (jt <= it) {
            f32x4 acc = {};
#pragma unroll
            for (int k8 = 0; k8 < KP; k8 += 32)
                acc = mma<2>(Kr.frag(jt * 16 + n, k8 + 8 * g), Qr.frag(i, k8 + 8 * g), acc);
            const f32x4 dec = (jt == it ? decay4<C, true>(gt, i, j) : decay4<C, false>(gt, i, j)) * scale;
            P.put4(i, perm(j), acc[0] * dec[0], acc[1] * dec[1], acc[2] * dec[2], acc[3] * dec[3]);
        } else if (jt == it + 1 && (jt & 1)) {       // the later tile of a pair that the products take together
            P.put4(i, perm(j), 0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
}

// the 16 x 16 diagonal blocks of I + L (-L in Ln, rows of ld) replaced by their inverses, by one wave: lanes 16 b .. 16 b
// + 15 take block b, lane n holds row n and solves for column n by forward substitution, row i's values from lane i
// s + sum of l[m .. m + 3] of lane I of each 16, times x[m .. m + 3]. (The compiler would take the 120 lane moves of a
// block first, in as many registers; the wait states are those between a write of l and its read from another lane.)
template <int I> DEV float sum4(const float (&l)[16], const float (&x)[16], int m, float s) {
    asm volatile("s_nop 1\n\t"
                 "v_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
                 "v_fmac_f32_dpp %0, %2, %6 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
                 "v_fmac_f32_dpp %0, %3, %7 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
                 "v_fmac_f32_dpp %0, %4, %8 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
                 : "+v"(s)
                 : "v"(l[m]), "v"(l[m + 1]), "v"(l[m + 2]), "v"(l[m + 3]), "v"(x[m]), "v"(x[m + 1]), "v"(x[m + 2]),
                   "v"(x[m + 3]), "n"(I));
    return s;
}
// (x[m] is 0 for m >= I, where l holds zeros too)
template <int I> DEV void substitute(const float (&l)[16], float (&x)[16], int n) {
    if constexpr (I < 16) {
        float s = I == n ? 1.0f : 0.0f;
#pragma unroll
        for (int m = 0; m < I; m += 4) s = sum4<I>(l, x, m, s);
        x[I] = s;
        substitute<I + 1>(l, x, n);
    }
}
template <int C> DEV void invert_blocks(float* ln, int ld) {
    const int n = threadIdx.x & 15, blk = (threadIdx.x & 63) >> 4;
    float* B = ln + (blk * 16) * ld + blk * 16;
    const bool in = blk < C / 16;
    float l[16] = {}, x[16] = {};
    if (in)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 v = *(const f32x4*)(B + n * ld + 4 * m);
#pragma unroll
            for (int e = 0; e < 4; ++e) l[4 * m + e] = v[e];
        }
    substitute<0>(l, x, n);
    if (in)
#pragma unroll
        for (int i = 0; i < 16; ++i) B[i * ld + n] = x[i];
}

// x <- (I + L)^-1 x for 16 columns, or (I + L)^-T x (from the last block row up); ln as invert_blocks leaves it
template <int C> DEV void solve_down(f32x4 (&x)[C / 16], const float* ln, int ld, int n, int g) {
#pragma unroll
    for (int rt = 0; rt < C / 16; ++rt) {
        f32x4 acc = x[rt];
#pragma unroll
        for (int m = 0; m < rt; ++m) acc = mma32(*(const f32x4*)(ln + (rt * 16 + n) * ld + m * 16 + 4 * g), x[m], acc);
        x[rt] = mma32(*(const f32x4*)(ln + (rt * 16 + n) * ld + rt * 16 + 4 * g), acc, f32x4{});
    }
}
template <int C> DEV void solve_up(f32x4 (&z)[C / 16], const float* ln, int ld, int n, int g) {
#pragma unroll
    for (int rt = C / 16 - 1; rt >= 0; --rt) {
        f32x4 acc = z[rt], a;
#pragma unroll
        for (int m = rt + 1; m < C / 16; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = ln[(m * 16 + 4 * g + e) * ld + rt * 16 + n];
            acc = mma32(a, z[m], acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = ln[(rt * 16 + 4 * g + e) * ld + rt * 16 + n];
        z[rt] = mma32(a, acc, f32x4{});
    }
}

// whether a chunk's rows times their factors (the write strengths: the last step's is in no other step's equation) are all
// finite, for the whole wave
template <int RT> DEV bool all_finite(const f32x4 (&x)[RT], const float* factor, int g) {
    float s = 0.0f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const f32x4 f = *(const f32x4*)(factor + rt * 16 + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += x[rt][e] * f[e] * 0.0f;              // 0, or NaN
    }
    return __builtin_amdgcn_ballot_w64(s != s) == 0;
}

// the kernel's first argument read again where it lies, so that the single steps' share of it takes no registers before
typedef const __attribute__((address_space(4))) InetDelta SameDelta;
DEV SameDelta& same_delta() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    keep_same(p);
    return *(SameDelta*)p;
}

// one step's gates: what the memory is kept by (0: emptied) and the write strength
struct StepGate {
    float keep, beta;
    DEV StepGate(SameDelta& d, int b, int h, int t) {
        const float g = gate_load(d.g, b * d.g_s[0] + t * d.g_s[1] + h * d.g_s[2], d.gate_dtype);
        beta = gate_load(d.beta, b * d.beta_s[0] + t * d.beta_s[1] + h * d.beta_s[2], d.gate_dtype);
        keep = (d.reset && d.reset[b * d.reset_s[0] + t * d.reset_s[1]]) || (double)g < DECAY_MIN ? 0.0f : expf(g);
    }
};

// a step's key or query at the lane's rows of the state. (Single steps compute their places anew each time: what they hold
// in registers the chunks' products have to do without.)
template <typename T, int KT> DEV void step_row(const T* p, int K, int g, f32x4 (&x)[KT]) {
    uint32_t row = 4 * g;
    keep(row);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t r = row + kt * 16 + e;
            const float v = (float)p[r < (uint32_t)K ? r : 0u];
            x[kt][e] = r < (uint32_t)K ? v : 0.0f;
        }
}
// a column's sum over its rows, in four lanes
template <int KT> DEV float column_sum(const f32x4 (&a)[KT], const f32x4 (&b)[KT]) {
    float s = 0.0f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += a[kt][e] * b[kt][e];
    s += __shfl_xor(s, 16);
    return s + __shfl_xor(s, 32);
}

// a chunk of up to C steps from t0 on, one by one, for a wave's 16 columns: the state after it; give(step, error, output) in a
// lane a column (OUT: outputs wanted). k, q, v: the head's rows; col: the lane's column of v (in: there is one).
template <int C, bool OUT, typename T, int KT, typename F>
DEV void steps_forward(SameDelta& d, int b, int h, int t0, const T* k, const T* q, const T* v, int64_t v_s, int col,
                       bool in, f32x4 (&S)[KT], int g, F&& give) {
#pragma nounroll
    for (int t = 0; t < C && t0 + t < d.T; ++t) {
        keep_same(b), keep_same(h), keep_same(k), keep_same(q), keep_same(v);
        uint32_t c = in ? col : 0;
        keep(c);
        const StepGate gate(d, b, h, t0 + t);
        f32x4 r[KT];
        step_row(k + (t0 + t) * d.k_s[1], d.K, g, r);
        const float value = in ? (float)v[(t0 + t) * v_s + c] : 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[kt][e] = gate.keep != 0.0f ? gate.keep * S[kt][e] : 0.0f;
        const float err = value - column_sum(r, S), w = gate.beta * err;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) S[kt] += r[kt] * w;
        float out = 0.0f;
        if (OUT) {
            step_row(q + (t0 + t) * d.q_s[1], d.K, g, r);
            out = d.scale * column_sum(r, S);
        }
        if (g == 0) give(t, err, out);
    }
}
// the same backwards: S from the gradient of the state after the chunk to that before it, give(step, Z). u: the head's rows of dO
template <int C, typename T, int KT, typename F>
DEV void steps_backward(SameDelta& d, int b, int h, int t0, const T* k, const T* q, const T* u, int64_t u_s, int col,
                        bool in, f32x4 (&S)[KT], int g, F&& give) {
#pragma nounroll
    for (int t = (d.T - t0 < C ? d.T - t0 : C) - 1; t >= 0; --t) {
        keep_same(b), keep_same(h), keep_same(k), keep_same(q), keep_same(u);
        uint32_t c = in ? col : 0;
        keep(c);
        const StepGate gate(d, b, h, t0 + t);
        f32x4 r[KT];
        const float out = in ? d.scale * (float)u[(t0 + t) * u_s + c] : 0.0f;
        step_row(q + (t0 + t) * d.q_s[1], d.K, g, r);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) S[kt] += r[kt] * out;
        step_row(k + (t0 + t) * d.k_s[1], d.K, g, r);
        const float z = column_sum(r, S), w = -gate.beta * z;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float s = S[kt][e] + r[kt][e] * w;
                S[kt][e] = gate.keep != 0.0f ? gate.keep * s : 0.0f;
            }
        if (g == 0) give(t, z);
    }
}

// both triangles of a chunk, from K and Q in LDS, and the diagonal blocks' inverses; ends with a barrier
template <int C, int KP, int NP, int NO, bool ROWS_BETA>
DEV void triangles(const Planes<NP>& Kr, const Planes<NP>& Qr, const Planes<NO>& P, const Gates<C>& gt, float* ln,
                   int ld, float scale, int w, int n, int g) {
    if (w < C / 16) triangle_l<C, KP, NP, ROWS_BETA>(Kr, gt, ln, ld, w, n, g);
    else if (C == 32) triangle_p<C, KP, NP, NO>(Kr, Qr, P, gt, scale, w - 2, n, g);
    __syncthreads();
    if (w == 0) invert_blocks<C>(ln, ld);
    if (C == 64) triangle_p<C, KP, NP, NO>(Kr, Qr, P, gt, scale, w, n, g);
    __syncthreads();
}

}  // namespace pol
