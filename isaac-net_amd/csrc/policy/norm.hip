// Block norms (include/inet_policy.h): the norm after a block, its gate and residual scale, the residual sum, and the
// norm before the next block, in one pass over the rows, forward and backward.
//
// Per row, with f^ = f / rms(f) and z = y / rms(y):
//     h = f^ w_post,  y = x + s gate h,  n = z w_pre
//     dz = dn w_pre,  dy' = dy + (dz - z mean(dz z)) / rms(y),  dx = dy',  dgate = dy' s h,  ds += dy' gate h
//     df^ = dy' gate s w_post,  dw_post += dy' gate s f^,  df = (df^ - f^ mean(df^ f^)) / rms(f),  dw_pre += dn z
// Memory bounds it: each row is read once into registers (the backward pass computes y again from x and f rather than
// read it, so y stays unrounded) and every sum over a row goes across its lanes in 32 bits. LP lanes take a row,
// NJ groups of 8 values each; with rows that do not start on 16 bytes a lane takes single values LP apart instead.
// The sums over rows for the weights stay in each workgroup's registers through all its rows, then go to the workspace
// as one partial row a workgroup; a second kernel adds those in a fixed order, so results do not vary from run to run.
#include "policy_dev.h"
#include "../../../include/inet_policy.h"

namespace pol {

constexpr int NORM_WG = 256;
constexpr int NORM_BLOCKS = 1024;            // workgroups of the backward pass, at most

// the sum over a row's LP lanes (LP <= 64), or over the workgroup (LP = 256; s: four words of LDS of its own)
template <int LP> DEV float row_sum(float x, float* s) {
#pragma unroll
    for (int o = 1; o < (LP < 64 ? LP : 64); o <<= 1) x += __shfl_xor(x, o);
    if constexpr (LP == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
        __syncthreads();
        x = s[0] + s[1] + s[2] + s[3];
    }
    return x;
}

// group j of a lane's values of a row: eight in sequence, or eight LP apart
template <typename T, int LP, bool VEC> DEV void row_load(const T* __restrict__ p, int c, int j, int D, float (&x)[8]) {
    if constexpr (VEC) {
        const int at = (j * LP + c) * 8;
        if (at < D) load8(p + at, 8, true, x);
        else
            for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    } else {
        for (int e = 0; e < 8; ++e) {
            const int at = (j * 8 + e) * LP + c;
            x[e] = at < D ? (float)p[at] : 0.0f;
        }
    }
}

template <typename T, int LP, bool VEC> DEV void row_store(T* __restrict__ p, int c, int j, int D, const float (&x)[8]) {
    if constexpr (VEC) {
        const int at = (j * LP + c) * 8;
        if (at < D) {
            if constexpr (sizeof(T) == 4) {
                *(f32x4*)(p + at) = f32x4{x[0], x[1], x[2], x[3]};
                *(f32x4*)(p + at + 4) = f32x4{x[4], x[5], x[6], x[7]};
            } else {
                typedef T V8 __attribute__((ext_vector_type(8)));
                V8 v;
                for (int e = 0; e < 8; ++e) v[e] = (T)x[e];
                *(V8*)(p + at) = v;
            }
        }
    } else {
        for (int e = 0; e < 8; ++e) {
            const int at = (j * 8 + e) * LP + c;
            if (at < D) p[at] = (T)x[e];
        }
    }
}

// weights: 1 where there are none
template <int LP, bool VEC> DEV void weight_load(const float* p, int c, int j, int D, float (&x)[8]) {
    if (p) row_load<float, LP, VEC>(p, c, j, D, x);
    else
        for (int e = 0; e < 8; ++e) x[e] = 1.0f;
}

template <typename T, int LP, int NJ, bool VEC>
__global__ __launch_bounds__(NORM_WG) void norm_forward_kernel(InetNorm a) {
    constexpr int RW = NORM_WG / LP;
    __shared__ float s_sum[4];
    const int c = threadIdx.x % LP;
    const int64_t row = (int64_t)blockIdx.x * RW + threadIdx.x / LP;
    const bool live = row < a.N;
    const int D = live ? a.D : 0;
    const float inv = 1.0f / (float)a.D;
    float y[NJ][8], f[NJ][8];
    float sf = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        row_load<T, LP, VEC>((const T*)a.x + row * a.x_s, c, j, D, y[j]);
        if (a.f) {
            row_load<T, LP, VEC>((const T*)a.f + row * a.f_s, c, j, D, f[j]);
            for (int e = 0; e < 8; ++e) sf += f[j][e] * f[j][e];
        }
    }
    if (a.f) {
        const float rf = a.post_weight ? rsqrtf(row_sum<LP>(sf, s_sum) * inv + a.eps) : 1.0f;
        const float row_gate = a.gate_kind == 1 && live ? (float)((const T*)a.gate)[row * a.gate_s] : 1.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float w[8], s[8], gt[8];
            weight_load<LP, VEC>(a.post_weight, c, j, D, w);
            weight_load<LP, VEC>(a.scale, c, j, D, s);
            if (a.gate_kind == 2) row_load<T, LP, VEC>((const T*)a.gate + row * a.gate_s, c, j, D, gt);
            for (int e = 0; e < 8; ++e) {
                const float h = f[j][e] * rf * w[e] * s[e];
                y[j][e] += h * (a.gate_kind == 2 ? gt[e] : row_gate);
            }
            row_store<T, LP, VEC>((T*)a.y + row * (int64_t)a.D, c, j, D, y[j]);
        }
    }
    if (a.pre_weight) {
        float sy = 0.0f;
        for (int j = 0; j < NJ; ++j)
            for (int e = 0; e < 8; ++e) sy += y[j][e] * y[j][e];
        const float ry = rsqrtf(row_sum<LP>(sy, s_sum) * inv + a.eps);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float w[8];
            weight_load<LP, VEC>(a.pre_weight, c, j, D, w);
            for (int e = 0; e < 8; ++e) y[j][e] *= ry * w[e];
            row_store<T, LP, VEC>((T*)a.n + row * (int64_t)a.D, c, j, D, y[j]);
        }
    }
}

template <typename T, int LP, int NJ, bool VEC>
__global__ __launch_bounds__(NORM_WG) void norm_backward_kernel(InetNorm a, InetNormGrad d) {
    constexpr int RW = NORM_WG / LP;
    __shared__ float s_sum[4];
    __shared__ float s_w[RW > 1 ? RW * LP * 8 : 1];
    const int c = threadIdx.x % LP, sub = threadIdx.x / LP;
    const float inv = 1.0f / (float)a.D;
    float ds[NJ][8] = {}, dpost[NJ][8] = {}, dpre[NJ][8] = {};
    const int64_t per = (a.N + (int64_t)gridDim.x * RW - 1) / ((int64_t)gridDim.x * RW);
    for (int64_t it = 0; it < per; ++it) {
        const int64_t row = (it * gridDim.x + blockIdx.x) * RW + sub;
        const bool live = row < a.N;
        const int D = live ? a.D : 0;
        float y[NJ][8], f[NJ][8] = {}, dy[NJ][8];
        float sf = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            row_load<T, LP, VEC>((const T*)a.x + row * a.x_s, c, j, D, y[j]);
            if (d.d_y) row_load<T, LP, VEC>((const T*)d.d_y + row * (int64_t)a.D, c, j, D, dy[j]);
            else
                for (int e = 0; e < 8; ++e) dy[j][e] = 0.0f;
            if (a.f) {
                row_load<T, LP, VEC>((const T*)a.f + row * a.f_s, c, j, D, f[j]);
                for (int e = 0; e < 8; ++e) sf += f[j][e] * f[j][e];
            }
        }
        const float rf = a.f && a.post_weight ? rsqrtf(row_sum<LP>(sf, s_sum) * inv + a.eps) : 1.0f;
        const float row_gate = a.gate_kind == 1 && live ? (float)((const T*)a.gate)[row * a.gate_s] : 1.0f;
        float gt[NJ][8];
        if (a.f)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                float w[8], s[8];
                weight_load<LP, VEC>(a.post_weight, c, j, D, w);
                weight_load<LP, VEC>(a.scale, c, j, D, s);
                if (a.gate_kind == 2) row_load<T, LP, VEC>((const T*)a.gate + row * a.gate_s, c, j, D, gt[j]);
                else
                    for (int e = 0; e < 8; ++e) gt[j][e] = row_gate;
                for (int e = 0; e < 8; ++e) {
                    f[j][e] *= rf;
                    y[j][e] += gt[j][e] * s[e] * w[e] * f[j][e];
                }
            }
        if (a.pre_weight && d.d_n) {
            float sy = 0.0f, sz = 0.0f, dz[NJ][8];
            for (int j = 0; j < NJ; ++j)
                for (int e = 0; e < 8; ++e) sy += y[j][e] * y[j][e];
            const float ry = rsqrtf(row_sum<LP>(sy, s_sum) * inv + a.eps);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                float w[8];
                row_load<T, LP, VEC>((const T*)d.d_n + row * (int64_t)a.D, c, j, D, dz[j]);
                weight_load<LP, VEC>(a.pre_weight, c, j, D, w);
                for (int e = 0; e < 8; ++e) {
                    y[j][e] *= ry;
                    dpre[j][e] += dz[j][e] * y[j][e];
                    dz[j][e] *= w[e];
                    sz += dz[j][e] * y[j][e];
                }
            }
            sz = row_sum<LP>(sz, s_sum) * inv;
            for (int j = 0; j < NJ; ++j)
                for (int e = 0; e < 8; ++e) dy[j][e] += ry * (dz[j][e] - y[j][e] * sz);
        }
        for (int j = 0; j < NJ; ++j)
            row_store<T, LP, VEC>((T*)d.d_x + row * (int64_t)a.D, c, j, D, dy[j]);
        if (a.f) {
            float sd = 0.0f, sg = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                float w[8], s[8], dg[8];
                weight_load<LP, VEC>(a.post_weight, c, j, D, w);
                weight_load<LP, VEC>(a.scale, c, j, D, s);
                for (int e = 0; e < 8; ++e) {
                    const float t = dy[j][e] * gt[j][e], h = f[j][e] * w[e];
                    ds[j][e] += t * h;
                    dpost[j][e] += t * s[e] * f[j][e];
                    dg[e] = dy[j][e] * s[e] * h;
                    sg += dg[e];
                    dy[j][e] = t * s[e] * w[e];
                    sd += dy[j][e] * f[j][e];
                }
                if (a.gate_kind == 2) row_store<T, LP, VEC>((T*)d.d_gate + row * (int64_t)a.D, c, j, D, dg);
            }
            if (a.gate_kind == 1) {
                sg = row_sum<LP>(sg, s_sum);
                if (live && c == 0) ((T*)d.d_gate)[row] = (T)sg;
            }
            sd = a.post_weight ? row_sum<LP>(sd, s_sum) * inv : 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                for (int e = 0; e < 8; ++e) dy[j][e] = rf * (dy[j][e] - f[j][e] * sd);
                row_store<T, LP, VEC>((T*)d.d_f + row * (int64_t)a.D, c, j, D, dy[j]);
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
                for (int e = 0; e < 8; ++e) s_w[(sub * 8 + e) * LP + c] = x[j][e];
                __syncthreads();
                if (sub == 0)
                    for (int r = 1; r < RW; ++r)
                        for (int e = 0; e < 8; ++e) x[j][e] += s_w[(r * 8 + e) * LP + c];
            }
            if (sub == 0)
                for (int e = 0; e < 8; ++e) {
                    const int at = VEC ? (j * LP + c) * 8 + e : (j * 8 + e) * LP + c;
                    if (at < a.D) out[m * a.D + at] = x[j][e];
                }
        }
    };
    if (a.f) {
        give(ds, 0);
        give(dpost, 1);
    }
    if (a.pre_weight) give(dpre, 2);
}

// the workgroups' partial rows added up, 64 columns a workgroup, its waves' shares in order
__global__ __launch_bounds__(NORM_WG) void norm_weights_kernel(const float* __restrict__ work, int blocks, int D,
                                                               float* ds, float* dpost, float* dpre) {
    __shared__ float s[4][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, m = blockIdx.y;
    float* out = m == 0 ? ds : m == 1 ? dpost : dpre;
    const int col = blockIdx.x * 64 + lane;
    if (!out) return;
    const int from = blocks * w / 4, to = blocks * (w + 1) / 4;
    float x[4] = {};
    if (col < D) {
        const float* p = work + (int64_t)m * D + col;
        int b = from;
        for (; b + 4 <= to; b += 4)
            for (int u = 0; u < 4; ++u) x[u] += p[(int64_t)(b + u) * 3 * D];
        for (; b < to; ++b) x[0] += p[(int64_t)b * 3 * D];
    }
    s[w][lane] = (x[0] + x[1]) + (x[2] + x[3]);
    __syncthreads();
    if (w == 0 && col < D) out[col] = (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]);
}

static int blocks_for(int64_t N, int rows) {
    const int64_t need = (N + rows - 1) / rows;
    return (int)(need < NORM_BLOCKS ? need : NORM_BLOCKS);
}

template <typename T, int LP, int NJ, bool VEC>
static int launch(const InetNorm& a, const InetNormGrad* d, hipStream_t st) {
    constexpr int RW = NORM_WG / LP;
    if (!d) {
        hipLaunchKernelGGL((norm_forward_kernel<T, LP, NJ, VEC>), dim3((unsigned)((a.N + RW - 1) / RW)), dim3(NORM_WG),
                           0, st, a);
        return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
    }
    const int blocks = blocks_for(a.N, RW);
    hipLaunchKernelGGL((norm_backward_kernel<T, LP, NJ, VEC>), dim3(blocks), dim3(NORM_WG), 0, st, a, *d);
    if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH;
    hipLaunchKernelGGL(norm_weights_kernel, dim3((a.D + 63) / 64, 3), dim3(NORM_WG), 0, st, d->work, blocks, a.D,
                       a.f ? d->d_scale : nullptr, a.f ? d->d_post_weight : nullptr,
                       a.pre_weight ? d->d_pre_weight : nullptr);
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

// lanes a row and groups a lane: as few lanes as hold the row with one group each, then more groups, and the whole
// workgroup from 2048 values on
template <typename T, bool VEC> static int sizes(const InetNorm& a, const InetNormGrad* d, hipStream_t st) {
    if (a.D <= 128) return launch<T, 16, 1, VEC>(a, d, st);
    if (a.D <= 256) return launch<T, 32, 1, VEC>(a, d, st);
    if (a.D <= 512) return launch<T, 64, 1, VEC>(a, d, st);
    if (a.D <= 1024) return launch<T, 64, 2, VEC>(a, d, st);
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
    if (!a || a->N < 0 || a->D < 1 || a->dtype < 0 || a->dtype > 2 || a->gate_kind < 0 || a->gate_kind > 2)
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
        hipLaunchKernelGGL(pol::norm_weights_kernel, dim3((a->D + 63) / 64, 3), dim3(pol::NORM_WG), 0,
                           (hipStream_t)stream, d->work, 0, a->D, d->d_scale, d->d_post_weight, d->d_pre_weight);
        return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
    }
    return pol::run(*a, d, (hipStream_t)stream);
}

}  // extern "C"
