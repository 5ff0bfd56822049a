// Block norms (include/inet_policy.h): the norm after a block, its gate and residual scale, the residual sum, and the
// norm before the next block, in one pass over the rows, forward and backward.
//
// Per row, with f^ = f / rms(f) and z = y / rms(y):
//     h = f^ w_post,  y = x + s gate h,  n = z w_pre
//     dz = dn w_pre,  dy' = dy + (dz - z mean(dz z)) / rms(y),  dx = dy',  dgate = dy' s h,  ds += dy' gate h
//     df^ = dy' gate s w_post,  dw_post += dy' gate s f^,  df = (df^ - f^ mean(df^ f^)) / rms(f),  dw_pre += dn z
// Memory bounds it: each row is read once into registers (the backward pass computes y again from x and f rather than
// read it, so y stays unrounded) and every sum over a row goes across its lanes in 32 bits. LP lanes take a row, NJ groups
// of 8 values each, 16 bytes at a time wherever rows start. 131072 x 512, bfloat16, full gate: forward 113 us for 0.67 GB, 5.9
// TB/s, backward 262 us for 1.2 GB, 4.6 TB/s (a copy makes 4.8); 5001 x 999, float32, a gate a row: 20 and 40 us. Rows off the
// 16-byte grid cost up to half more (62660 x 1071, float16: forward 179 us, backward 489).
// The sums over rows for the weights stay in each workgroup's registers through all its rows, then go to the workspace
// as one partial row a workgroup; a second kernel adds those in a fixed order, so results do not vary from run to run.
#include "policy_dev.h"
#include "../../../include/inet_policy.h"

namespace pol {

constexpr int NORM_WG = 256;

// the sum over a row's LP lanes (LP <= 64), or over the workgroup (LP = 256; s: four words of LDS of its own): along the
// rows of 16 lanes by rotations, across them by swaps of rows and halves
template <int CTRL> DEV float lane_turn(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int LP> DEV float lane_sum(float x) {
    x += lane_turn<0x128>(x);
    x += lane_turn<0x124>(x);
    x += lane_turn<0x122>(x);
    x += lane_turn<0x121>(x);
    if constexpr (LP >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, x);
        const auto v = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const unsigned even = v[0], odd = v[1];
        x = __builtin_bit_cast(float, even) + __builtin_bit_cast(float, odd);
    }
    if constexpr (LP >= 64) {
        const unsigned u = __builtin_bit_cast(unsigned, x);
        const auto v = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const unsigned low = v[0], high = v[1];
        x = __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
    }
    return x;
}
// two sums at once; over a workgroup's four waves through one of two places in LDS in turn, so that one barrier a call
// is enough (a place is written again only after the other's barrier, by when all have read it)
template <int LP> struct RowSums {
    float (*s)[8];
    int turn = 0;
    DEV void sum(float& a, float& b) {
        a = lane_sum<LP>(a);
        b = lane_sum<LP>(b);
        if constexpr (LP == 256) {
            float* t = s[turn];
            turn ^= 1;
            const int w = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) {
                t[w] = a;
                t[4 + w] = b;
            }
            __syncthreads();
            a = (t[0] + t[1]) + (t[2] + t[3]);
            b = (t[4] + t[5]) + (t[6] + t[7]);
        }
    }
    DEV float sum(float a) {
        float b = 0.0f;
        sum(a, b);
        return a;
    }
};

// eight values wherever they start (WHOLE: on 16 bytes): one 16-byte access (two for float32) either way
template <typename T, bool WHOLE> struct Eight {
    typedef T Value __attribute__((ext_vector_type(8)));
    typedef T Place __attribute__((ext_vector_type(8), aligned(WHOLE ? 16 : sizeof(T))));
};

// Group j of a lane: values `base` .. base + 7 of the row, those from `skip` on its own. VEC: rows start on 16 bytes and hold
// whole groups; else the last group of a row ends with the row and shares its first values with the group before, so that it
// is one access too (a row of fewer than eight values is read one by one).
template <int LP, bool VEC> struct Group {
    int base, skip;
    bool in;
    DEV Group(int c, int j, int D) {
        const int at = (j * LP + c) * 8;
        in = at < D;
        base = VEC || at + 8 <= D || D < 8 ? at : D - 8;
        skip = VEC ? 0 : at - base;
    }
};

// a row on its way from memory: the lane's NJ groups of eight, LP groups apart
template <typename T, int LP, int NJ, bool VEC> struct Row {
    typedef typename Eight<T, VEC>::Value V8;
    V8 v[NJ];
    DEV void load(const T* __restrict__ p, int c, int D) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const Group<LP, VEC> q(c, j, D);
            v[j] = V8{};
            if (VEC || D >= 8) {
                if (q.in) v[j] = *(const typename Eight<T, VEC>::Place*)(p + q.base);
            } else if (q.in) {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (e < D) v[j][e] = p[e];
            }
        }
    }
    DEV float at(int j, int e) const { return (float)v[j][e]; }
    DEV float own(const Group<LP, VEC>& q, int j, int e) const { return VEC || e >= q.skip ? (float)v[j][e] : 0.0f; }
};

template <typename T, int LP, bool VEC> DEV void row_store(T* __restrict__ p, int c, int j, int D, const float (&x)[8]) {
    const Group<LP, VEC> q(c, j, D);
    if (!q.in) return;
    if (VEC || (q.skip == 0 && D >= 8)) {
        typename Eight<T, VEC>::Value v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)x[e];
        *(typename Eight<T, VEC>::Place*)(p + q.base) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e >= q.skip && q.base + e < D) p[q.base + e] = (T)x[e];
    }
}

// weights: 1 where there are none
template <int LP, int NJ, bool VEC> struct Weights {
    Row<float, LP, NJ, VEC> r;
    DEV void load(const float* p, int c, int D) {
        if (p) r.load(p, c, D);
        else
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) r.v[j][e] = 1.0f;
    }
    DEV float at(int j, int e) const { return r.v[j][e]; }
};

template <typename T, int LP, int NJ, bool VEC>
__global__ __launch_bounds__(NORM_WG) void norm_forward_kernel(InetNorm a) {
    constexpr int RW = NORM_WG / LP;
    __shared__ float s_sum[2][8];
    RowSums<LP> sums{s_sum};
    const int c = threadIdx.x % LP;
    const int64_t row = (int64_t)blockIdx.x * RW + threadIdx.x / LP;
    const bool live = row < a.N;
    const int D = live ? a.D : 0;
    const float inv = 1.0f / (float)a.D;
    Row<T, LP, NJ, VEC> x, f, gt;
    x.load((const T*)a.x + row * a.x_s, c, D);
    float y[NJ][8];
    if (a.f) {
        f.load((const T*)a.f + row * a.f_s, c, D);
        if (a.gate_kind == 2) gt.load((const T*)a.gate + row * a.gate_s, c, D);
        const float row_gate = a.gate_kind == 1 && live ? (float)((const T*)a.gate)[row * a.gate_s] : 1.0f;
        Weights<LP, NJ, VEC> w, s;
        w.load(a.post_weight, c, a.D);
        s.load(a.scale, c, a.D);
        float rf = 1.0f;
        if (a.post_weight) {
            float sf = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = f.own(Group<LP, VEC>(c, j, D), j, e);
                    sf += v * v;
                }
            rf = rsqrtf(sums.sum(sf) * inv + a.eps);
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[j][e] = x.own(Group<LP, VEC>(c, j, D), j, e) + f.own(Group<LP, VEC>(c, j, D), j, e) * rf * w.at(j, e) * s.at(j, e) * (a.gate_kind == 2 ? gt.at(j, e) : row_gate);
            row_store<T, LP, VEC>((T*)a.y + row * (int64_t)a.D, c, j, D, y[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] = x.own(Group<LP, VEC>(c, j, D), j, e);
    }
    if (a.pre_weight) {
        Weights<LP, NJ, VEC> w;
        w.load(a.pre_weight, c, a.D);
        float sy = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) sy += y[j][e] * y[j][e];
        const float ry = rsqrtf(sums.sum(sy) * inv + a.eps);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] *= ry * w.at(j, e);
            row_store<T, LP, VEC>((T*)a.n + row * (int64_t)a.D, c, j, D, y[j]);
        }
    }
}

template <typename T, int LP, int NJ, bool VEC>
__global__ __launch_bounds__(NORM_WG) void norm_backward_kernel(InetNorm a, InetNormGrad d) {
    constexpr int RW = NORM_WG / LP;
    __shared__ float s_sum[2][8];
    RowSums<LP> sums{s_sum};
    __shared__ float s_w[RW > 1 ? RW * LP * 8 : 1];
    const int c = threadIdx.x % LP, sub = threadIdx.x / LP;
    const float inv = 1.0f / (float)a.D;
    float ds[NJ][8] = {}, dpost[NJ][8] = {}, dpre[NJ][8] = {};
    const int64_t per = (a.N + (int64_t)gridDim.x * RW - 1) / ((int64_t)gridDim.x * RW);
    const bool pre = a.pre_weight && d.d_n;
    Row<T, LP, NJ, VEC> x, f, gt, dy, dn;
    float row_gate = 1.0f;
    auto fetch = [&](int64_t row) {                  // the next row's values, while the one before is computed with
        const int D = row < a.N ? a.D : 0;
        x.load((const T*)a.x + row * a.x_s, c, D);
        dy.load((const T*)d.d_y + row * (int64_t)a.D, c, d.d_y ? D : 0);
        if (a.f) {
            f.load((const T*)a.f + row * a.f_s, c, D);
            if (a.gate_kind == 2) gt.load((const T*)a.gate + row * a.gate_s, c, D);
            else if (a.gate_kind == 1 && D) row_gate = (float)((const T*)a.gate)[row * a.gate_s];
        }
        if (pre) dn.load((const T*)d.d_n + row * (int64_t)a.D, c, D);
    };
    fetch((int64_t)blockIdx.x * RW + sub);
    for (int64_t it = 0; it < per; ++it) {
        const int64_t row = (it * gridDim.x + blockIdx.x) * RW + sub;
        const bool live = row < a.N;
        const int D = live ? a.D : 0;
        float y[NJ][8], h[NJ][8], g[NJ][8], dv[NJ][8], z[NJ][8];
        float sf = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const Group<LP, VEC> q(c, j, a.D);
                y[j][e] = x.own(q, j, e);
                dv[j][e] = dy.own(q, j, e);
                h[j][e] = a.f ? f.own(q, j, e) : 0.0f;
                g[j][e] = a.gate_kind == 2 ? gt.at(j, e) : row_gate;
                z[j][e] = pre ? dn.own(q, j, e) : 0.0f;
                sf += h[j][e] * h[j][e];
            }
        if (it + 1 < per) fetch(row + (int64_t)gridDim.x * RW);
        Weights<LP, NJ, VEC> w, s, wp;
        float rf = 1.0f;
        if (a.f) {
            w.load(a.post_weight, c, a.D);
            s.load(a.scale, c, a.D);
            // (a row past the last is zeros: with eps 0 its reciprocal would be infinite, and NaN in the weights' sums)
            if (a.post_weight) {
                const float sum = sums.sum(sf);
                rf = live ? rsqrtf(sum * inv + a.eps) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[j][e] *= rf;                   // f^
                    y[j][e] += g[j][e] * s.at(j, e) * w.at(j, e) * h[j][e];
                }
        }
        if (pre) {
            wp.load(a.pre_weight, c, a.D);
            float sy = 0.0f, sz = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sy += y[j][e] * y[j][e];
                    sz += z[j][e] * wp.at(j, e) * y[j][e];
                }
            sums.sum(sy, sz);
            const float ry = live ? rsqrtf(sy * inv + a.eps) : 0.0f;
            sz *= inv * ry;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[j][e] *= ry;                   // z of the formulas
                    dpre[j][e] += z[j][e] * y[j][e];
                    dv[j][e] += ry * (z[j][e] * wp.at(j, e) - y[j][e] * sz);
                }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) row_store<T, LP, VEC>((T*)d.d_x + row * (int64_t)a.D, c, j, D, dv[j]);
        if (a.f) {
            float sd = 0.0f, sg = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                float dg[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float t = dv[j][e] * g[j][e], sw = s.at(j, e) * w.at(j, e);
                    ds[j][e] += t * h[j][e] * w.at(j, e);
                    dpost[j][e] += t * s.at(j, e) * h[j][e];
                    dg[e] = dv[j][e] * sw * h[j][e];
                    sg += dg[e];
                    dv[j][e] = t * sw;
                    sd += dv[j][e] * h[j][e];
                }
                if (a.gate_kind == 2) row_store<T, LP, VEC>((T*)d.d_gate + row * (int64_t)a.D, c, j, D, dg);
            }
            sums.sum(sg, sd);
            if (a.gate_kind == 1 && live && c == 0) ((T*)d.d_gate)[row] = (T)sg;
            sd = a.post_weight ? sd * inv : 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) dv[j][e] = rf * (dv[j][e] - h[j][e] * sd);
                row_store<T, LP, VEC>((T*)d.d_f + row * (int64_t)a.D, c, j, D, dv[j]);
            }
        }
    }
    // the workgroup's sums for the weights, its row groups' added in order: [workgroup][3][D]
    float* out = d.work + (int64_t)blockIdx.x * 3 * a.D;
    auto give = [&](float (&x)[NJ][8], int m) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (RW > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 8; ++e) s_w[(sub * 8 + e) * LP + c] = x[j][e];
                __syncthreads();
                if (sub == 0)
                    for (int r = 1; r < RW; ++r)
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[j][e] += s_w[(r * 8 + e) * LP + c];
            }
            if (sub == 0)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const Group<LP, VEC> q(c, j, a.D);
                    if (q.in && e >= q.skip && q.base + e < a.D) out[m * a.D + q.base + e] = x[j][e];
                }
        }
    };
    if (a.f) {
        give(ds, 0);
        give(dpost, 1);
    }
    if (a.pre_weight) give(dpre, 2);
}

// the workgroups' partial rows added up, 64 columns a workgroup of 16 waves, the waves' shares in order
__global__ __launch_bounds__(1024) void norm_weights_kernel(const float* __restrict__ work, int blocks, int D, float* ds,
                                                            float* dpost, float* dpre) {
    __shared__ float s[16][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, m = blockIdx.y;
    float* out = m == 0 ? ds : m == 1 ? dpost : dpre;
    const int col = blockIdx.x * 64 + lane;
    if (!out) return;
    const int from = blocks * w / 16, to = blocks * (w + 1) / 16;
    float x[8] = {};
    if (col < D) {
        const float* p = work + (int64_t)m * D + col;
        int b = from;
        for (; b + 8 <= to; b += 8)
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] += p[(int64_t)(b + u) * 3 * D];
        for (; b < to; ++b) x[0] += p[(int64_t)b * 3 * D];
    }
    s[w][lane] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    __syncthreads();
    if (w == 0 && col < D) {
        float y = 0.0f;
#pragma unroll
        for (int u = 0; u < 16; ++u) y += s[u][lane];
        out[col] = y;
    }
}

// workgroups of the backward pass: two a compute unit where each then has eight groups of rows or more, else one (a
// workgroup's partial rows are as long as the data's). us at 256, 512 and 1024 workgroups: 131072 x 512 bfloat16 322, 249
// and 258; 20000 x 512 42, 33 and 36; 4000 x 4000 74, 84 and 99; 5001 x 999 float32 45, 52 and 65
static int blocks_for(int64_t N, int rows) {
    const int64_t need = (N + rows - 1) / rows, want = need >= 8 * 512 ? 512 : 256;
    return (int)(need < want ? need : want);
}

template <typename T, int LP, int NJ, bool VEC> static int launch_forward(const InetNorm& a, hipStream_t st) {
    constexpr int RW = NORM_WG / LP;
    const int64_t grid = (a.N + RW - 1) / RW;
    if (grid > GRID_MAX) return INET_POLICY_EUNSUPPORTED;
    hipLaunchKernelGGL((norm_forward_kernel<T, LP, NJ, VEC>), dim3((unsigned)grid), dim3(NORM_WG), 0, st, a);
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

template <typename T, int LP, int NJ, bool VEC>
static int launch(const InetNorm& a, const InetNormGrad* d, hipStream_t st) {
    constexpr int RW = NORM_WG / LP;
    if (!d) return launch_forward<T, LP, NJ, VEC>(a, st);
    const int blocks = blocks_for(a.N, RW);
    hipLaunchKernelGGL((norm_backward_kernel<T, LP, NJ, VEC>), dim3(blocks), dim3(NORM_WG), 0, st, a, *d);
    if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH;
    hipLaunchKernelGGL(norm_weights_kernel, dim3((a.D + 63) / 64, 3), dim3(1024), 0, st, d->work, blocks, a.D,
                       a.f ? d->d_scale : nullptr, a.f ? d->d_post_weight : nullptr,
                       a.pre_weight ? d->d_pre_weight : nullptr);
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

// lanes a row and groups a lane: as few lanes as hold the row with one group each (N D = 2^25, bfloat16, full gate, training,
// us: D = 128 by 16 lanes 202, 32 lanes 292, 64 lanes 473; D = 256 by 32 lanes 195, 16 x 2 groups 203, 64 lanes 290), then two
// groups of a wave (D = 1024: 200, a workgroup a row 285), then, where rows are whole 16-bit groups on 16 bytes, three groups
// (1032: 254, a workgroup a row 296; 1304: 250, 262; 1536: 214, 237) and forward four (forward alone at 1600 61, 67, 1904 60, 69,
// 2048 59, 64; backward 182, 161, 188, 149, 134, 138), else a workgroup a row, whose waves hold few registers (odd rows at D = 1071
// 353, three groups 365; float32, N D = 2^24: 1536 192, 211; 2048 192, 292)
template <typename T, bool VEC> static int sizes(const InetNorm& a, const InetNormGrad* d, hipStream_t st) {
    if (a.D <= 128) return launch<T, 16, 1, VEC>(a, d, st);
    if (a.D <= 256) return launch<T, 32, 1, VEC>(a, d, st);
    if (a.D <= 512) return launch<T, 64, 1, VEC>(a, d, st);
    if (a.D <= 1024) return launch<T, 64, 2, VEC>(a, d, st);
    if constexpr (VEC && sizeof(T) == 2) {
        if (a.D <= 1536) return launch<T, 64, 3, VEC>(a, d, st);
        if (a.D <= 2048 && !d) return launch_forward<T, 64, 4, VEC>(a, st);
    }
    if (a.D <= 2048) return launch<T, 256, 1, VEC>(a, d, st);
    if (a.D <= 4096) return launch<T, 256, 2, VEC>(a, d, st);
    return launch<T, 256, 4, VEC>(a, d, st);
}

static int run(const InetNorm& a, const InetNormGrad* d, hipStream_t st) {
    const int e = a.dtype == INET_POLICY_F32 ? 4 : 2;
    bool vec = a.D % 8 == 0;
    auto rows = [&](const void* p, int64_t s) { vec = vec && (uintptr_t)p % 16 == 0 && s * e % 16 == 0; };
    rows(a.x, a.x_s);
    if (a.f) rows(a.f, a.f_s);
    if (a.gate_kind == 2) rows(a.gate, a.gate_s);
    for (const void* p : {(const void*)a.scale, (const void*)a.post_weight, (const void*)a.pre_weight, (const void*)a.y,
                          (const void*)a.n})
        rows(p, 0);
    if (d)
        for (const void* p : {d->d_y, d->d_n, (const void*)d->d_x, (const void*)d->d_f}) rows(p, 0);
    if (d && a.gate_kind == 2) rows(d->d_gate, 0);
    if (a.dtype == INET_POLICY_F32) return vec ? sizes<float, true>(a, d, st) : sizes<float, false>(a, d, st);
    if (a.dtype == INET_POLICY_BF16) return vec ? sizes<__bf16, true>(a, d, st) : sizes<__bf16, false>(a, d, st);
    return vec ? sizes<_Float16, true>(a, d, st) : sizes<_Float16, false>(a, d, st);
}

static int check(const InetNorm* a) {
    if (!a || a->N < 0 || a->D < 1 || a->dtype < 0 || a->dtype > 2 || a->gate_kind < 0 || a->gate_kind > 2 ||
        !(a->eps >= 0.0f))
        return INET_POLICY_EINVAL;
    if (a->D > INET_POLICY_MAX_WIDTH || a->N > (int64_t)1 << 24) return INET_POLICY_EUNSUPPORTED;
    if (a->N == 0) return INET_POLICY_OK;
    if (!a->x || (a->gate_kind && !a->gate) || (!a->f && (a->gate_kind || a->scale || a->post_weight)) ||
        (!a->f && !a->pre_weight))
        return INET_POLICY_EINVAL;
    return INET_POLICY_OK;
}

}  // namespace pol

extern "C" {

int64_t inet_policy_norm_work(int64_t N, int32_t D) {
    if (N < 0 || D < 1 || D > INET_POLICY_MAX_WIDTH) return -1;
    return (int64_t)pol::blocks_for(N, 1) * 3 * D * (int64_t)sizeof(float);
}

int32_t inet_policy_norm_forward(const InetNorm* a, void* stream) {
    if (int rc = pol::check(a)) return rc;
    if (a->N == 0) return INET_POLICY_OK;
    if ((a->f && !a->y) || (a->pre_weight && !a->n)) return INET_POLICY_EINVAL;
    return pol::run(*a, nullptr, (hipStream_t)stream);
}

int32_t inet_policy_norm_backward(const InetNorm* a, const InetNormGrad* d, void* stream) {
    if (int rc = pol::check(a)) return rc;
    if (!d || (a->N && !d->work)) return INET_POLICY_EINVAL;
    if (a->N && (!d->d_x || (a->f && !d->d_f) || (a->gate_kind && !d->d_gate))) return INET_POLICY_EINVAL;
    if ((d->d_scale && !a->scale) || (d->d_post_weight && !a->post_weight) || (d->d_pre_weight && !a->pre_weight))
        return INET_POLICY_EINVAL;
    if (a->N == 0) {                             // (no rows: the second kernel alone, over no partial rows, writes zeros)
        hipLaunchKernelGGL(pol::norm_weights_kernel, dim3((a->D + 63) / 64, 3), dim3(1024), 0,
                           (hipStream_t)stream, d->work, 0, a->D, d->d_scale, d->d_post_weight, d->d_pre_weight);
        return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
    }
    return pol::run(*a, d, (hipStream_t)stream);
}

}  // extern "C"
