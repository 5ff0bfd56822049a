// The gated feed-forward (include/inet_policy.h): y = act(x Wg^T) * (x Wu^T), forward and backward, on the 16-bit matrix
// instructions with sums in 32 bits.
//
// Forward: a workgroup computes a 128 x 128 tile of both projections from one pass over its rows of x, and the
// activation and the product in registers; neither projection goes to memory. Backward: the same tile again from x (the
// two projections would cost a write and a read of 2 N F values, more than the products at the widths measured), then
// da = dy u act'(a) and du = dy act(a), rounded to the type, as they are and transposed; then
//     dx = [da du] [Wg; Wu]        a product over 2 F,        dWg = da^T x,  dWu = du^T x     products over N
// all with both operands' rows along the sum (W and x transposed once). The products over N are split where the tiles of
// dW are fewer than the chip's compute units; the parts are added in order, so results do not vary from run to run.
#include <type_traits>

#include "policy_dev.h"
#include "../../../include/inet_policy.h"

namespace pol {

constexpr int FFN_WG = 256, BM = 128, BN = 128, BK = 64, LDK = BK + 8;

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

template <typename T> DEV f32x4 mfma16(typename Vec8<T>::type a, typename Vec8<T>::type b, f32x4 c) {
    if constexpr (std::is_same<T, __bf16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// rows r0 .. r0 + 127 of p (row stride st, rows valid rows), columns k0 .. k0 + 63 of `cols` (a multiple of 8), one
// 16-byte load a thread and pass; outside: 0
template <typename T> struct Tile {
    typename Vec8<T>::type v[4];
    DEV void load(const T* __restrict__ p, int64_t st, int64_t r0, int64_t rows, int64_t k0, int64_t cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = threadIdx.x + i * FFN_WG;
            const int64_t r = r0 + at / 8, k = k0 + at % 8 * 8;
            if (r < rows && k < cols) v[i] = *(const typename Vec8<T>::type*)(p + r * st + k);
            else v[i] = typename Vec8<T>::type{};
        }
    }
    DEV void put(T* s) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = threadIdx.x + i * FFN_WG;
            *(typename Vec8<T>::type*)(s + at / 8 * LDK + at % 8 * 8) = v[i];
        }
    }
};

// acc[m] (64 x 64 a wave) of A [rows][k] against NB matrices B_m [cols][k], both along k
template <typename T, int NB>
DEV void product(const T* __restrict__ A, int64_t as, int64_t r0, int64_t rows, const T* const (&B)[NB],
                 const int64_t (&bs)[NB], int64_t c0, int64_t cols, int64_t k_from, int64_t k_to, T* lds,
                 f32x4 (&acc)[NB][4][4]) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wr = (w >> 1) * 64, wc = (w & 1) * 64;
    Tile<T> ta, tb[NB];
    ta.load(A, as, r0, rows, k_from, k_to);
#pragma unroll
    for (int m = 0; m < NB; ++m) tb[m].load(B[m], bs[m], c0, cols, k_from, k_to);
    for (int64_t k = k_from; k < k_to; k += BK) {
        __syncthreads();
        ta.put(lds);
#pragma unroll
        for (int m = 0; m < NB; ++m) tb[m].put(lds + (1 + m) * BM * LDK);
        __syncthreads();
        if (k + BK < k_to) {
            ta.load(A, as, r0, rows, k + BK, k_to);
#pragma unroll
            for (int m = 0; m < NB; ++m) tb[m].load(B[m], bs[m], c0, cols, k + BK, k_to);
        }
#pragma unroll
        for (int kk = 0; kk < BK; kk += 32) {
            typename Vec8<T>::type a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a[i] = *(const typename Vec8<T>::type*)(lds + (wr + i * 16 + n) * LDK + kk + 8 * g);
#pragma unroll
            for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const auto b = *(const typename Vec8<T>::type*)(lds + (1 + m) * BM * LDK +
                                                                   (wc + j * 16 + n) * LDK + kk + 8 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i][j] = mfma16<T>(a[i], b, acc[m][i][j]);
                }
        }
    }
}

// act(a) and its derivative
DEV void activation(int act, float a, float& h, float& dh) {
    if (act == INET_POLICY_SILU) {
        const float s = 1.0f / (1.0f + __expf(-a));
        h = a * s;
        dh = s * (1.0f + a * (1.0f - s));
    } else if (act == INET_POLICY_GELU) {
        // 0.5 (1 + tanh u) = 1 / (1 + e^{-2 u})
        const float a2 = a * a, u = 0.7978845608028654f * a * (1.0f + 0.044715f * a2);
        const float s = 1.0f / (1.0f + __expf(-2.0f * u));
        h = a * s;
        dh = s + a * s * (1.0f - s) * 2.0f * 0.7978845608028654f * (1.0f + 0.134145f * a2);
    } else {
        h = a > 0.0f ? a : 0.0f;
        dh = a > 0.0f ? 1.0f : 0.0f;
    }
}

struct FfnShape {
    int64_t N, x_s, wg_s, wu_s, y_s;
    int D, D8, F, F8, act;
    int64_t N8;
};

template <typename T, bool BACK>
__global__ __launch_bounds__(FFN_WG) void ffn_gates_kernel(FfnShape p, const T* __restrict__ x,
                                                           const T* __restrict__ wg, const T* __restrict__ wu,
                                                           T* __restrict__ y, const T* __restrict__ dy, int64_t dy_s,
                                                           T* __restrict__ da, T* __restrict__ dat) {
    __shared__ alignas(16) T lds[3 * BM * LDK];
    const int64_t r0 = (int64_t)blockIdx.y * BM;
    const int c0 = blockIdx.x * BN;
    f32x4 acc[2][4][4] = {};
    const T* const B[2] = {wg, wu};
    const int64_t bs[2] = {p.wg_s, p.wu_s};
    product<T, 2>(x, p.x_s, r0, p.N, B, bs, c0, p.F, 0, p.D8, lds, acc);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wr = (w >> 1) * 64, wc = (w & 1) * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = c0 + wc + j * 16 + n;
            float a_out[4], u_out[4];
            for (int e = 0; e < 4; ++e) {
                const int64_t row = r0 + wr + i * 16 + 4 * g + e;
                const bool in = row < p.N && col < p.F;
                float h, dh;
                activation(p.act, acc[0][i][j][e], h, dh);
                if (!BACK) {
                    if (in) y[row * p.y_s + col] = (T)(h * acc[1][i][j][e]);
                } else {
                    const float d = in ? (float)dy[row * dy_s + col] : 0.0f;
                    a_out[e] = d * acc[1][i][j][e] * dh;
                    u_out[e] = d * h;
                    if (row < p.N && col < p.F8) {
                        da[row * 2 * p.F8 + col] = (T)a_out[e];
                        da[row * 2 * p.F8 + p.F8 + col] = (T)u_out[e];
                    }
                }
            }
            if (BACK && col < p.F) {
                const int64_t row = r0 + wr + i * 16 + 4 * g;
                for (int e = 0; e < 4; ++e)
                    if (row + e < p.N8) {
                        dat[(int64_t)col * p.N8 + row + e] = (T)a_out[e];
                        dat[(int64_t)(p.F + col) * p.N8 + row + e] = (T)u_out[e];
                    }
            }
        }
}

// C [rows][cols] = A [rows][k] B [cols][k]^T; blockIdx.z: a share of k, each to its own C in 32 bits
template <typename T, typename O>
__global__ __launch_bounds__(FFN_WG) void ffn_product_kernel(const T* __restrict__ A, int64_t as, int64_t rows,
                                                             const T* __restrict__ B, int64_t b_s, int64_t cols,
                                                             int64_t K, int64_t share, O* __restrict__ C, int64_t cs) {
    __shared__ alignas(16) T lds[2 * BM * LDK];
    const int64_t r0 = (int64_t)blockIdx.y * BM, c0 = (int64_t)blockIdx.x * BN;
    f32x4 acc[1][4][4] = {};
    const T* const Bm[1] = {B};
    const int64_t bs[1] = {b_s}, from = blockIdx.z * share, to = from + share < K ? from + share : K;
    product<T, 1>(A, as, r0, rows, Bm, bs, c0, cols, from, to, lds, acc);
    C += blockIdx.z * rows * cs;
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wr = (w >> 1) * 64, wc = (w & 1) * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            for (int e = 0; e < 4; ++e) {
                const int64_t row = r0 + wr + i * 16 + 4 * g + e, col = c0 + wc + j * 16 + n;
                if (row < rows && col < cols) C[row * cs + col] = (O)acc[0][i][j][e];
            }
}

// out [cols][rows8] = in [rows][cols] transposed, zeros in rows .. rows8 - 1; 64 x 64 tiles
template <typename T>
__global__ __launch_bounds__(256) void ffn_transpose_kernel(const T* __restrict__ in, int64_t in_s, int64_t rows,
                                                            int64_t cols, T* __restrict__ out, int64_t out_s,
                                                            int64_t rows8) {
    __shared__ T s[64][66];
    const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int64_t r = r0 + i / 64, c = c0 + i % 64;
        s[i / 64][i % 64] = r < rows && c < cols ? in[r * in_s + c] : (T)0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int64_t c = c0 + i / 64, r = r0 + i % 64;
        if (c < cols && r < rows8) out[c * out_s + r] = s[i % 64][i / 64];
    }
}

// rows padded to a multiple of eight with zeros
template <typename T>
__global__ __launch_bounds__(256) void ffn_pad_kernel(const T* __restrict__ in, int64_t in_s, int64_t rows, int D,
                                                      T* __restrict__ out, int D8) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * D8) return;
    const int64_t r = i / D8;
    const int c = (int)(i % D8);
    out[i] = c < D ? in[r * in_s + c] : (T)0.0f;
}

// the shares of a product over N added up in order: out [n]
template <typename T>
__global__ __launch_bounds__(256) void ffn_add_kernel(const float* __restrict__ parts, int count, int64_t n,
                                                      T* __restrict__ out, int64_t stride) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float x = 0.0f;
    for (int s = 0; s < count; ++s) x += parts[s * stride + i];
    out[i] = (T)x;
}

static int64_t up8(int64_t x) { return (x + 7) & ~(int64_t)7; }
static int64_t tiles(int64_t x) { return (x + BM - 1) / BM; }
static unsigned blocks256(int64_t n) { return (unsigned)((n + 255) / 256); }

// shares of a product over N: enough workgroups for the chip's 256 compute units twice over, no share under 512 rows
static int shares(int64_t N, int D, int F) {
    const int64_t t = tiles(F) * tiles(D) * 2, want = (512 + t - 1) / t, most = (N + 511) / 512;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s);
}

// the workspace's parts, in bytes from its start
struct Work {
    int64_t x, wg, wu, da, dat, xt, wt, parts, bytes;
    Work(int64_t N, int64_t D, int64_t F, bool back) {
        const int64_t D8 = up8(D), F8 = up8(F), N8 = up8(N);
        int64_t at = 0;
        auto take = [&](int64_t n) {
            const int64_t p = at;
            at += (n + 255) & ~(int64_t)255;
            return p;
        };
        const bool pad = D8 != D;
        x = take(pad ? N * D8 * 2 : 0);
        wg = take(pad ? F * D8 * 2 : 0);
        wu = take(pad ? F * D8 * 2 : 0);
        da = take(back ? N * 2 * F8 * 2 : 0);
        dat = take(back ? 2 * F * N8 * 2 : 0);
        xt = take(back ? D * N8 * 2 : 0);
        wt = take(back ? D * 2 * F8 * 2 : 0);
        parts = take(back ? (int64_t)shares(N, (int)D, (int)F) * 2 * F * D * 4 : 0);
        bytes = at;
    }
};

#define LAUNCHED                                                        \
    do {                                                                \
        if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH; \
    } while (0)

template <typename T> static int run(const InetFfn& a, const InetFfnGrad* d, hipStream_t st) {
    const Work at(a.N, a.D, a.F, d != nullptr);
    char* work = (char*)a.work;
    FfnShape p{a.N, a.x_s, a.w_gate_s, a.w_up_s, a.y_s, a.D, (int)up8(a.D), a.F, (int)up8(a.F), a.act, up8(a.N)};
    const T *x = (const T*)a.x, *wg = (const T*)a.w_gate, *wu = (const T*)a.w_up;
    if (p.D8 != p.D) {
        struct { const T* in; int64_t s, rows; T* out; } pads[3] = {{x, a.x_s, a.N, (T*)(work + at.x)},
                                                                    {wg, a.w_gate_s, a.F, (T*)(work + at.wg)},
                                                                    {wu, a.w_up_s, a.F, (T*)(work + at.wu)}};
        for (auto& q : pads) {
            hipLaunchKernelGGL(ffn_pad_kernel<T>, dim3(blocks256(q.rows * p.D8)), dim3(256), 0, st, q.in, q.s, q.rows,
                               p.D, q.out, p.D8);
            LAUNCHED;
        }
        x = pads[0].out, wg = pads[1].out, wu = pads[2].out;
        p.x_s = p.wg_s = p.wu_s = p.D8;
    }
    const dim3 grid((unsigned)tiles(a.F), (unsigned)tiles(a.N));
    if (!d) {
        hipLaunchKernelGGL((ffn_gates_kernel<T, false>), grid, dim3(FFN_WG), 0, st, p, x, wg, wu, (T*)a.y,
                           (const T*)nullptr, (int64_t)0, (T*)nullptr, (T*)nullptr);
        LAUNCHED;
        return INET_POLICY_OK;
    }
    T *da = (T*)(work + at.da), *dat = (T*)(work + at.dat), *xt = (T*)(work + at.xt), *wt = (T*)(work + at.wt);
    hipLaunchKernelGGL((ffn_gates_kernel<T, true>), grid, dim3(FFN_WG), 0, st, p, x, wg, wu, (T*)nullptr,
                       (const T*)d->d_y, d->d_y_s, da, dat);
    LAUNCHED;
    if (d->d_x) {
        for (int m = 0; m < 2; ++m) {
            hipLaunchKernelGGL(ffn_transpose_kernel<T>, dim3((a.F + 63) / 64, (a.D + 63) / 64), dim3(256), 0, st,
                               m ? wu : wg, m ? p.wu_s : p.wg_s, (int64_t)a.F, (int64_t)a.D, wt + m * p.F8,
                               (int64_t)2 * p.F8, (int64_t)p.F8);
            LAUNCHED;
        }
        hipLaunchKernelGGL((ffn_product_kernel<T, T>), dim3((unsigned)tiles(a.D), (unsigned)tiles(a.N)), dim3(FFN_WG),
                           0, st, da, (int64_t)2 * p.F8, a.N, wt, (int64_t)2 * p.F8, (int64_t)a.D, (int64_t)2 * p.F8,
                           (int64_t)2 * p.F8, (T*)d->d_x, (int64_t)a.D);
        LAUNCHED;
    }
    if (d->d_w_gate || d->d_w_up) {
        hipLaunchKernelGGL(ffn_transpose_kernel<T>, dim3((unsigned)((a.N + 63) / 64), (a.D + 63) / 64), dim3(256), 0,
                           st, x, p.x_s, a.N, (int64_t)a.D, xt, p.N8, p.N8);
        LAUNCHED;
        const int s = shares(a.N, a.D, a.F);
        const int64_t share = ((p.N8 + s - 1) / s + BK - 1) / BK * BK;
        float* parts = (float*)(work + at.parts);
        hipLaunchKernelGGL((ffn_product_kernel<T, float>), dim3((unsigned)tiles(a.D), (unsigned)tiles(2 * (int64_t)a.F), s),
                           dim3(FFN_WG), 0, st, dat, p.N8, (int64_t)2 * a.F, xt, p.N8, (int64_t)a.D, p.N8, share, parts,
                           (int64_t)a.D);
        LAUNCHED;
        // (the shares of both matrices lie one after the other: [share][2 F][D])
        const int64_t one = (int64_t)a.F * a.D;
        for (int m = 0; m < 2; ++m) {
            T* out = (T*)(m ? d->d_w_up : d->d_w_gate);
            if (!out) continue;
            hipLaunchKernelGGL(ffn_add_kernel<T>, dim3(blocks256(one)), dim3(256), 0, st, parts + m * one, s, one, out,
                               2 * one);
            LAUNCHED;
        }
    }
    return INET_POLICY_OK;
}

static int check(const InetFfn* a) {
    if (!a || a->N < 0 || a->D < 1 || a->F < 1 || a->act < 0 || a->act > 2 || a->dtype < 0 || a->dtype > 2)
        return INET_POLICY_EINVAL;
    if (a->dtype == INET_POLICY_F32 || a->D > 1 << 20 || a->F > 1 << 20) return INET_POLICY_EUNSUPPORTED;
    if (tiles(a->N) > 65535) return INET_POLICY_EUNSUPPORTED;
    if (a->N == 0) return INET_POLICY_OK;
    if (!a->x || !a->w_gate || !a->w_up) return INET_POLICY_EINVAL;
    if (a->D % 8 == 0) {                      // rows are read 16 bytes at a time; other widths are padded first
        const void* p[3] = {a->x, a->w_gate, a->w_up};
        const int64_t s[3] = {a->x_s, a->w_gate_s, a->w_up_s};
        for (int i = 0; i < 3; ++i)
            if ((uintptr_t)p[i] % 16 || s[i] % 8) return INET_POLICY_EINVAL;
    }
    if (!a->work && Work(a->N, a->D, a->F, false).bytes) return INET_POLICY_EINVAL;
    return INET_POLICY_OK;
}

template <typename T> static int zero_weights(const InetFfn& a, const InetFfnGrad& d, hipStream_t st) {
    const int64_t one = (int64_t)a.F * a.D;
    for (void* out : {d.d_w_gate, d.d_w_up})
        if (out) {
            hipLaunchKernelGGL(ffn_add_kernel<T>, dim3(blocks256(one)), dim3(256), 0, st, (const float*)nullptr, 0, one,
                               (T*)out, one);
            LAUNCHED;
        }
    return INET_POLICY_OK;
}

}  // namespace pol

extern "C" {

int64_t inet_policy_ffn_work(int64_t N, int32_t D, int32_t F, int32_t backward) {
    if (N < 0 || D < 1 || F < 1) return -1;
    return pol::Work(N, D, F, backward != 0).bytes;
}

int32_t inet_policy_ffn_forward(const InetFfn* a, void* stream) {
    if (int rc = pol::check(a)) return rc;
    if (a->N == 0) return INET_POLICY_OK;
    if (!a->y) return INET_POLICY_EINVAL;
    return a->dtype == INET_POLICY_BF16 ? pol::run<__bf16>(*a, nullptr, (hipStream_t)stream)
                                        : pol::run<_Float16>(*a, nullptr, (hipStream_t)stream);
}

int32_t inet_policy_ffn_backward(const InetFfn* a, const InetFfnGrad* d, void* stream) {
    if (int rc = pol::check(a)) return rc;
    if (!d) return INET_POLICY_EINVAL;
    if (a->N == 0)                            // (no rows: the weights' gradients are zero)
        return a->dtype == INET_POLICY_BF16 ? pol::zero_weights<__bf16>(*a, *d, (hipStream_t)stream)
                                            : pol::zero_weights<_Float16>(*a, *d, (hipStream_t)stream);
    if (!d->d_y || !a->work) return INET_POLICY_EINVAL;
    return a->dtype == INET_POLICY_BF16 ? pol::run<__bf16>(*a, d, (hipStream_t)stream)
                                        : pol::run<_Float16>(*a, d, (hipStream_t)stream);
}

}  // extern "C"
