// The gated feed-forward (include/inet_policy.h): y = act(x Wg^T) * (x Wu^T), forward and backward, on the 16-bit matrix
// instructions with sums in 32 bits.
//
// Forward: a workgroup computes a tile of both projections from one pass over its rows of x, and the activation and the
// product in registers; neither projection goes to memory. Backward: the same tile again from x, then da = dy u act'(a)
// and du = dy act(a), rounded to the type (half the bytes and the matrix instructions' rate for the two products that follow,
// for one rounding more in their sums; float16's range: Range below); then
//     dx = [da du] [Wg; Wu]        a product over 2 F,        dWg = da^T x,  dWu = du^T x     products over N.
// All are one product (Product): tiles of 64 along the sum go to LDS, the next one on its way from memory while the present
// one is computed with, and a matrix whose rows lie across the sum (W for dx, x and da for dW) is transposed by the LDS
// reads.
// The products over N are split where the tiles of dW are fewer than the chip's compute units; the parts are added in
// order, so results do not vary from run to run.
#include <type_traits>

#include "policy_dev.h"
#include "../../../include/inet_policy.h"

namespace pol {

constexpr int BK = 64;                       // along the sum, a step

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

template <typename T> DEV f32x4 mfma16(typename Vec8<T>::type a, typename Vec8<T>::type b, f32x4 c) {
    if constexpr (std::is_same<T, __bf16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 16 bytes of zeros, where a tile reaches past its matrix
__device__ __attribute__((aligned(16))) const uint32_t zero16[4] = {0, 0, 0, 0};

// 64 lanes' 16 bytes each from memory to LDS, lane after lane from `to` on (the same in all lanes)
DEV void load_lds(const void* from, void* to) {
    typedef __attribute__((address_space(1))) const uint32_t* Mem;
    typedef __attribute__((address_space(3))) uint32_t* Lds;
    __builtin_amdgcn_global_load_lds((Mem)from, (Lds)to, 16, 0, 0);
}

// A matrix of a product: element (i, k) for index i of the result and k of the sum.
// ALONG: rows along the sum, p[i * st + k], i < rows. TWO: a second matrix p2 of the same shape, where the tile's second
// half of indexes comes from.
// else across: p[k * st + i], i < rows (rows a multiple of eight).
template <typename T, bool ALONG> struct Operand {
    const T *p, *p2;
    int64_t st, st2, rows;
};

// A tile of R indexes x 64 of the sum on its way to LDS. The lanes' places in memory are 32-bit offsets from a place that
// moves along the sum; indexes past the matrix read its last (their results are not stored), what is past the sum is zero.
// DIRECT (ALONG alone): memory to LDS without registers, row i's group c of eight at place c ^ (i % 8) of the row's eight,
// so that a read's lanes fall on distinct banks. Else through registers, to rows with a gap: ALONG 64 + 8 by index, across
// R + 16 by the sum, and a read's places are one address and constants.
template <typename T, bool ALONG, int R, int THREADS, bool TWO, bool DIRECT> struct Tile {
    static constexpr int LOADS = R * 8 / THREADS, LD = DIRECT ? 64 : ALONG ? 72 : R + 16,
                         SIZE = (ALONG ? R : BK) * LD;
    typedef typename Vec8<T>::type V8;
    const char *base, *base2;
    uint32_t off[LOADS];
    int64_t step;
    V8 v[DIRECT ? 1 : LOADS];
    // load j of this thread: its row of the tile and its group of eight in the row
    static DEV int row_at(int j) { return (j * THREADS + (int)threadIdx.x) / (ALONG ? 8 : R / 8); }
    static DEV int group_at(int j) {
        const int at = (j * THREADS + (int)threadIdx.x) % (ALONG ? 8 : R / 8);
        return DIRECT ? at ^ (row_at(j) & 7) : at;
    }
    static constexpr bool second(int j) { return TWO && j >= LOADS / 2; }     // (half the loads are half the rows)
    DEV void start(const Operand<T, ALONG>& m, int64_t r0, int64_t k0) {
        base = (const char*)(ALONG ? m.p + r0 * m.st + k0 : m.p + k0 * m.st + r0);
        base2 = TWO ? (const char*)(m.p2 + r0 * m.st2 + k0) : nullptr;
        step = BK * (ALONG ? 1 : m.st) * (int64_t)sizeof(T);
        const int64_t last = m.rows - 1 - r0;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int r = row_at(j), c = group_at(j) * 8;
            if constexpr (ALONG) {
                int64_t i = second(j) ? r - R / 2 : r;
                i = i < last ? i : last;
                off[j] = (uint32_t)((i * (second(j) ? m.st2 : m.st) + c) * (int64_t)sizeof(T));
            } else {
                off[j] = (uint32_t)((r * m.st + (c < last - 7 ? c : last - 7)) * (int64_t)sizeof(T));
            }
        }
    }
    DEV void next() {
        base += step;
        if (TWO) base2 += step;
    }
    // the tile of the next 64, `left` of them inside the sum: straight to LDS
    DEV void fetch(int64_t left, T* lds) {
        const int w = threadIdx.x >> 6;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const char* from = (second(j) ? base2 : base) + off[j];
            if (left < BK && group_at(j) * 8 >= left) from = (const char*)zero16;
            load_lds(from, lds + (j * (THREADS / 64) + w) * 512);
        }
        next();
    }
    // or into registers, and put() when the buffer is free
    DEV void load(int64_t left) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            v[j] = V8{};
            if ((ALONG ? group_at(j) * 8 : row_at(j)) < left) v[j] = *(const V8*)((second(j) ? base2 : base) + off[j]);
        }
        next();
    }
    DEV void put(T* lds) const {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) *(V8*)(lds + row_at(j) * LD + group_at(j) * 8) = v[j];
    }
    // indexes i0 + n, 8 g .. 8 g + 7 of the 32 from kk on
    static DEV V8 frag(const T* lds, int i0, int kk, int n, int g) {
        if constexpr (DIRECT) {
            const int r = i0 + n, c = (kk >> 3) + g;
            return *(const V8*)(lds + r * 64 + ((c ^ (r & 7)) << 3));
        } else if constexpr (ALONG) {
            return *(const V8*)(lds + (i0 + n) * LD + kk + 8 * g);
        } else {
            const __bf16* p = (const __bf16*)lds + (kk + 8 * g + (n >> 2)) * LD + i0 + (n & 3) * 4;
            return __builtin_bit_cast(V8, __builtin_shufflevector(read_tr(p), read_tr(p + 4 * LD), 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// acc[c][r] += tiles of the product of `rows` (BM indexes) and `cols` (BN), over k_from .. k_to - 1; WR x WC waves. A lane
// holds four columns (16 c + 4 g + e of the wave's) of one row (16 r + n). The columns come in two halves where HALVES:
// the wave's first CT / 2 tiles from the first half of the tile's columns, the others from the second.
template <typename T, int BM_, int BN_, int WR_, int WC_, bool ROWS_ALONG, bool COLS_ALONG, bool HALVES> struct Product {
    static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_, THREADS = 64 * WR * WC, RT = BM / WR / 16,
                         CT = BN / WC / 16;
    // straight to LDS where no read of LDS transposes: the compiler has those wait for all of memory
    static constexpr bool DIRECT = ROWS_ALONG && COLS_ALONG;
    typedef Tile<T, ROWS_ALONG, BM, THREADS, false, DIRECT> TR;
    typedef Tile<T, COLS_ALONG, BN, THREADS, HALVES, DIRECT> TC;
    static constexpr int BUF = TR::SIZE + TC::SIZE, LDS = 2 * BUF * (int)sizeof(T);
    // the first column of the wave's tile c
    static DEV int col(int wc, int c) {
        return HALVES ? (c < CT / 2 ? 0 : BN / 2) + wc * (BN / 2 / WC) + (c % (CT / 2)) * 16 : wc * (BN / WC) + c * 16;
    }
    // (rows2 and cols2: a second pair, added where rows2.p is there)
    static DEV void run(const Operand<T, ROWS_ALONG>& rows1, const Operand<T, COLS_ALONG>& cols1,
                        const Operand<T, ROWS_ALONG>& rows2, const Operand<T, COLS_ALONG>& cols2, int64_t r0, int64_t c0,
                        int64_t k_from, int64_t k_to, T* lds, f32x4 (&acc)[CT][RT]) {
        const int pairs = rows2.p ? 2 : 1;
#pragma nounroll
        for (int m = 0; m < pairs; ++m) one(m ? rows2 : rows1, m ? cols2 : cols1, r0, c0, k_from, k_to, lds, acc);
    }
    static DEV void one(const Operand<T, ROWS_ALONG>& rows, const Operand<T, COLS_ALONG>& cols, int64_t r0, int64_t c0,
                        int64_t k_from, int64_t k_to, T* lds, f32x4 (&acc)[CT][RT]) {
        if (k_from >= k_to) return;
        TR tr;
        TC tc;
        tr.start(rows, r0, k_from);
        tc.start(cols, c0, k_from);
        __syncthreads();                     // (a product before this one has been computed with its buffers)
        if constexpr (DIRECT) {
            tr.fetch(k_to - k_from, lds);
            tc.fetch(k_to - k_from, lds + TR::SIZE);
        } else {
            tr.load(k_to - k_from);
            tc.load(k_to - k_from);
        }
        int cur = 0;
        for (int64_t k = k_from; k < k_to; k += BK, cur ^= 1) {
            if constexpr (DIRECT) {
                // this step's tiles have arrived, and nobody reads the other buffer any more
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (k + BK < k_to) {
                    tr.fetch(k_to - k - BK, lds + (cur ^ 1) * BUF);
                    tc.fetch(k_to - k - BK, lds + (cur ^ 1) * BUF + TR::SIZE);
                }
            } else {
                tr.put(lds + cur * BUF);
                tc.put(lds + cur * BUF + TR::SIZE);
                __syncthreads();
                if (k + BK < k_to) {
                    tr.load(k_to - k - BK);
                    tc.load(k_to - k - BK);
                }
            }
            step(lds + cur * BUF, acc);
        }
    }
    // one tile along the sum
    static DEV void step(const T* lr, f32x4 (&acc)[CT][RT]) {
        const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wr = w / WC, wc = w % WC;
        const T* lc = lr + TR::SIZE;
#pragma unroll
        for (int kk = 0; kk < BK; kk += 32) {
            typename Vec8<T>::type b[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) b[r] = TR::frag(lr, wr * (BM / WR) + r * 16, kk, n, g);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const auto x = TC::frag(lc, col(wc, c), kk, n, g);
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[c][r] = mfma16<T>(x, b[r], acc[c][r]);
            }
        }
    }
};

// The tiles (and shares of the sum) in an order in which the workgroups that run together on one of the eight dies, each
// with an L2 of its own, share what they read: die d takes a stretch of the sequence of all shares, of each share's row
// tiles, and of each row tile's column tiles.
DEV void tile_order(int64_t at, int64_t total, int64_t row_tiles, int col_tiles, int64_t& r, int& c, int& share) {
    const int64_t die = at % 8, per = total / 8, rest = total % 8;
    const int64_t mine = die * per + (die < rest ? die : rest) + at / 8, tile = mine / col_tiles;
    c = (int)(mine % col_tiles);
    r = tile % row_tiles;
    share = (int)(tile / row_tiles);
}

// four values of a row from column col on, of `cols`
template <bool WHOLE, typename O> DEV void put_row4(O* p, int col, int cols, bool vec, f32x4 x) {
    if (WHOLE || (vec && col + 4 <= cols)) {
        typedef O V4 __attribute__((ext_vector_type(4)));
        V4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (O)x[e];
        *(V4*)(p + col) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < cols) p[col + e] = (O)x[e];
    }
}

// 1 / (1 + e^-x) (the reciprocal to one unit in the last place; x of any size: e^-x may be infinite, the result then 0)
DEV float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// act(a) and its derivative; gelu's 0.5 (1 + tanh u) is logistic(2 u)
template <int ACT> DEV void activation(float a, float& h, float& dh) {
    if constexpr (ACT == INET_POLICY_SILU) {
        const float s = logistic(a);
        h = a * s;
        dh = s + h * (1.0f - s);
    } else if constexpr (ACT == INET_POLICY_GELU) {
        // (a2 bounded: from |a| of 10^4 on s is 0 or 1 to the last bit, and past 2^64 a * a would be infinite, dh NaN)
        const float a2 = fminf(a * a, 1e8f), s = logistic(1.5957691216057308f * a * (1.0f + 0.044715f * a2));
        h = a * s;
        dh = s + h * (1.0f - s) * (1.5957691216057308f + 0.21406440f * a2);
    } else {
        h = a <= 0.0f ? 0.0f : a;              // (NaN stays)
        dh = a > 0.0f ? 1.0f : 0.0f;
    }
}

// da and du in float16 keep to its range: each workgroup leaves the largest of its finite values, and where the largest of all
// is past 65504, or so small (below 2^-4) that the usual ones would lose bits below 2^-14, the tiles are computed once more,
// scaled by the power of two that takes it to 2^14 .. 2^15; the products' results are scaled back. Bfloat16 has the range of 32
// bits. 16383 x 504 x 1352: 4.8 us for the launch that finds nothing to do, 89 for the tiles again.
struct Range {
    static constexpr int TOPS = 1024;        // more than a launch's workgroups: 256 that go on, or four times the fewer than 256
                                             // tiles of the next size
    static bool __device__ in(float top) { return top == 0.0f || (top >= 0.0625f && top <= 65504.0f); }
    static float __device__ scale(float top) {
        const int e = 14 - ilogbf(top);
        return ldexpf(1.0f, e < -120 ? -120 : e > 120 ? 120 : e);
    }
};

// the largest of a workgroup's values, in all lanes (s: a word a wave)
template <int THREADS> DEV float workgroup_max(float x, float* s) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) x = fmaxf(x, s[w]);
    return x;
}

struct FfnShape {
    int64_t N, y_s;
    int D8, F, F8;
    bool vec_y;                              // y (or dy) by four values at a time
};

// y, or (BACK) da and du side by side in da [N][2 F8]. A workgroup takes tile after tile: the next one's first step is on
// its way, and dy has come during the last step, while the results are stored. The matrix instructions bound it, then what
// the activation and the stores leave of their time: 131072 x 512 x 2048, bfloat16, silu: y 641 us, 857 TFLOP/s (the library's
// product of these sizes alone 716, 8192^3 1302); da and du 1021 us with 1.6 GB of dy, da and du beside the same products.
template <typename T, typename P, int ACT, bool BACK>
__global__ __launch_bounds__(P::THREADS, P::THREADS == 512 ? 2 : 1)
void ffn_gates_kernel(FfnShape p, Operand<T, true> x, Operand<T, true> w, T* __restrict__ y, const T* __restrict__ dy,
                      int64_t dy_s, T* __restrict__ da, float* __restrict__ tops, bool again) {
    extern __shared__ char lds_raw[];
    constexpr int COLS = P::BN / 2, RT = P::RT, CT = P::CT;
    constexpr bool RANGED = BACK && std::is_same<T, _Float16>::value;
    T* const lds = (T*)lds_raw;
    float top = 0.0f, scale = 1.0f;
    if constexpr (RANGED)
        if (again) {
            for (unsigned i = threadIdx.x; i < gridDim.x; i += P::THREADS) top = fmaxf(top, tops[i]);
            top = workgroup_max<P::THREADS>(top, (float*)lds_raw);
            const bool in = Range::in(top);
            if (!in) scale = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, Range::scale(top))));
            if (blockIdx.x == 0 && threadIdx.x == 0) tops[Range::TOPS] = 1.0f / scale;
            if (in) return;
            __syncthreads();
        }
    const int64_t row_tiles = (p.N + P::BM - 1) / P::BM;
    const int col_tiles = (p.F + COLS - 1) / COLS, steps = (p.D8 + BK - 1) / BK;
    const int64_t total = row_tiles * col_tiles;
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wr = wv / P::WC, wc = wv % P::WC;
    typename P::TR tr;
    typename P::TC tc;
    int64_t rt;
    int ct, all, buf = 0;
    auto begin = [&](int64_t at) {
        tile_order(at, total, row_tiles, col_tiles, rt, ct, all);
        tr.start(x, rt * P::BM, 0);
        tc.start(w, (int64_t)ct * COLS, 0);
        tr.fetch(p.D8, lds + buf * P::BUF);
        tc.fetch(p.D8, lds + buf * P::BUF + P::TR::SIZE);
    };
    begin(blockIdx.x);
    for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
        const int64_t r0 = rt * P::BM, c0 = (int64_t)ct * COLS;
        const int rows = (int)(p.N - r0 < P::BM ? p.N - r0 : P::BM), cols = (int)(p.F - c0), cols8 = (int)(p.F8 - c0);
        f32x4 acc[CT][RT] = {};
        for (int k = 0; k < steps; ++k, buf ^= 1) {
            // this step's tiles have arrived, and nobody reads the other buffer any more
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (k + 1 < steps) {
                tr.fetch(p.D8 - (k + 1) * BK, lds + (buf ^ 1) * P::BUF);
                tc.fetch(p.D8 - (k + 1) * BK, lds + (buf ^ 1) * P::BUF + P::TR::SIZE);
            }
            P::step(lds + buf * P::BUF, acc);
        }
        if (at + gridDim.x < total) begin(at + gridDim.x);
    // WHOLE: the tile inside the matrices, four values at a time; offsets from the tile's corner
    auto finish = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        T* const out = BACK ? da + r0 * 2 * p.F8 + c0 : y + r0 * p.y_s + c0;
        const T* const in = BACK ? dy + r0 * dy_s + c0 : nullptr;
#pragma unroll
        for (int r = 0; r < P::RT; ++r) {
            const int row = wr * (P::BM / P::WR) + r * 16 + n;
            if (!WHOLE && row >= rows) continue;
            f32x4 d[P::CT / 2];
            if constexpr (BACK)
#pragma unroll
                for (int c = 0; c < P::CT / 2; ++c) {
                    const int col = P::col(wc, c) + 4 * g;
                    float v[4] = {};
                    if (WHOLE || col < cols) load4(in + (int64_t)row * dy_s + col, cols - col, WHOLE || p.vec_y, v);
                    d[c] = f32x4{v[0], v[1], v[2], v[3]};
                }
#pragma unroll
            for (int c = 0; c < P::CT / 2; ++c) {
                const int col = P::col(wc, c) + 4 * g;
                const f32x4 a = acc[c][r], u = acc[c + P::CT / 2][r];
                f32x4 h, dh;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x, y2;
                    activation<ACT>(a[e], x, y2);
                    h[e] = x;
                    dh[e] = y2;
                }
                if constexpr (!BACK) {
                    put_row4<WHOLE>(out + row * p.y_s, col, cols, p.vec_y, h * u);
                } else if (WHOLE || col < cols8) {
                    f32x4 x1 = d[c] * u * dh, x2 = d[c] * h;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!WHOLE && col + e >= cols) x1[e] = x2[e] = 0.0f;
                    if constexpr (RANGED) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float m = fmaxf(fabsf(x1[e]), fabsf(x2[e]));
                            top = m < INFINITY ? fmaxf(top, m) : top;
                        }
                        x1 *= scale;
                        x2 *= scale;
                    }
                    put_row4<WHOLE>(out + (int64_t)row * 2 * p.F8, col, cols8, true, x1);
                    put_row4<WHOLE>(out + (int64_t)row * 2 * p.F8 + p.F8, col, cols8, true, x2);
                }
            }
        }
    };
    if (rows == P::BM && COLS <= cols && p.vec_y) finish(std::true_type{});
    else finish(std::false_type{});
    }
    if constexpr (RANGED)
        if (!again) {
            top = workgroup_max<P::THREADS>(top, (float*)lds_raw);
            if (threadIdx.x == 0) tops[blockIdx.x] = top;
        }
}

// C [rows][cols] = a b (+ a2 b2 where there are such), or shares of the sum each to a C of its own. At the sizes above: dx
// 679 us, 810 TFLOP/s (the library's product 925); both dW 606 us, 907 TFLOP/s (559). An operand across the sum goes through
// registers and is transposed by LDS reads, which is what keeps it from the rate of 8192^3.
template <typename T, typename P, bool RA, bool CA, typename O>
__global__ __launch_bounds__(P::THREADS, P::THREADS == 512 ? 2 : 1)
void ffn_product_kernel(Operand<T, RA> a, Operand<T, CA> b, Operand<T, RA> a2, Operand<T, CA> b2, int64_t K,
                        int64_t share, O* __restrict__ C, int64_t rows, int64_t cols, bool vec,
                        const float* __restrict__ unscale) {
    extern __shared__ char lds_raw[];
    int64_t rt;
    int ct, part;
    tile_order(blockIdx.x, gridDim.x, (rows + P::BM - 1) / P::BM, (int)((cols + P::BN - 1) / P::BN), rt, ct, part);
    const int64_t r0 = rt * P::BM, c0 = (int64_t)ct * P::BN;
    const int64_t from = part * share, to = from + share < K ? from + share : K;
    f32x4 acc[P::CT][P::RT] = {};
    P::run(a, b, a2, b2, r0, c0, from, to, (T*)lds_raw, acc);
    if constexpr (std::is_same<O, _Float16>::value) {
        const float f = *unscale;
#pragma unroll
        for (int c = 0; c < P::CT; ++c)
#pragma unroll
            for (int r = 0; r < P::RT; ++r) acc[c][r] *= f;
    }
    C += part * rows * cols;
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wr = wv / P::WC, wc = wv % P::WC;
    auto finish = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        O* const out = C + r0 * cols + c0;
        const int left = (int)(cols - c0 < P::BN ? cols - c0 : P::BN);
#pragma unroll
        for (int r = 0; r < P::RT; ++r) {
            const int row = wr * (P::BM / P::WR) + r * 16 + n;
            if (!WHOLE && r0 + row >= rows) continue;
#pragma unroll
            for (int c = 0; c < P::CT; ++c) {
                const int col = P::col(wc, c) + 4 * g;
                if (WHOLE || col < left) put_row4<WHOLE>(out + row * cols, col, left, vec, acc[c][r]);
            }
        }
    };
    if (r0 + P::BM <= rows && c0 + P::BN <= cols && vec) finish(std::true_type{});
    else finish(std::false_type{});
}

// rows padded to a multiple of eight with zeros (a copy; odd widths alone)
template <typename T>
__global__ __launch_bounds__(256) void ffn_pad_kernel(const T* __restrict__ in, int64_t in_s, int64_t rows, int D,
                                                      T* __restrict__ out, int D8) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * D8; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / D8;
        const int c = (int)(i % D8);
        out[i] = c < D ? in[r * in_s + c] : (T)0.0f;
    }
}

// the shares of a product over N added up in order: out [rows][D] of parts [count][.][cols]. Memory bounds it: 17 us for both
// weights at 131072 x 512 x 2048 (8 shares, 72 MB, from the L2s in part)
template <typename T>
__global__ __launch_bounds__(256) void ffn_add_kernel(const float* __restrict__ parts, int count, int64_t stride,
                                                      int64_t rows, int D, int cols, T* __restrict__ out,
                                                      const float* __restrict__ unscale) {
    const float f = unscale ? *unscale : 1.0f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * D; i += (int64_t)gridDim.x * 256) {
        const float* p = parts + i / D * cols + i % D;
        float x = 0.0f;
        for (int s = 0; s < count; ++s) x += p[s * stride];
        out[i] = (T)(x * f);
    }
}

static int64_t up8(int64_t x) { return (x + 7) & ~(int64_t)7; }
static int64_t tiles(int64_t x, int t) { return (x + t - 1) / t; }

// The tile of a product by how many of the largest it has: 256 x 256 (eight waves, a compute unit's LDS to itself) where
// they fill the chip's 256 compute units, else 128 x 128, else 64 x 64. Forward, us by tiles of 64, 128 and 256: 512 x 256 x 1024
// 5, 7, 12; 1500 x 512 x 2048 16, 15, 20; 2048 x 512 x 2048 19, 16, 20; 4096 x 512 x 2048 34, 27, 23; 8192 x 256 x 1024 21, 19,
// 16; 65536 x 512 x 2048 549, 460, 332.
static int size_for(int64_t rows, int64_t cols) {
    return tiles(rows, 256) * tiles(cols, 256) >= 256 ? 2 : tiles(rows, 128) * tiles(cols, 128) >= 256 ? 1 : 0;
}
template <typename F> static int by_size(int size, F&& f) {
    return size == 2 ? f(std::integral_constant<int, 2>{}) : size == 1 ? f(std::integral_constant<int, 1>{})
                                                                      : f(std::integral_constant<int, 0>{});
}
template <typename T, int SIZE, bool RA, bool CA, bool HALVES>
using Sized = typename std::conditional<SIZE == 2, Product<T, 256, 256, 2, 4, RA, CA, HALVES>,
              typename std::conditional<SIZE == 1, Product<T, 128, 128, 2, 2, RA, CA, HALVES>,
                                        Product<T, 64, 64, 2, 2, RA, CA, HALVES>>::type>::type;

// the weights' gradients: the tile, and shares of the sum over N, at least 512 rows each, until the chip is full, of the smaller
// tile twice over. us of dx and dW with the adding up, by tiles of 128 and 256: 65536 x 512 x 2048 735, 629; 65536 x 512 x 1024
// 383, 360; 65536 x 256 x 1024 213, 207; 4096 x 256 x 1024 50, 61; 4096 x 512 x 1024 59, 64. By 256 and 512 workgroups: 65536 x
// 512 x 2048 of 128 1031, 735, of 256 629, 637. By 256, 512 and 1024 rows a share at least: 4096 x 512 x 1024 60, 59, 90.
static int dw_size(int64_t D8, int64_t F8) { return tiles(2 * F8, 256) * tiles(D8, 256) >= 16 ? 2 : 1; }
static int shares(int64_t N, int64_t D8, int64_t F8) {
    const int size = dw_size(D8, F8), b = size == 2 ? 256 : 128;
    const int64_t t = tiles(2 * F8, b) * tiles(D8, b), want = ((size == 2 ? 256 : 512) + t - 1) / t, most = tiles(N, 512);
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s);
}

// the workspace's parts, in bytes from its start
struct Work {
    int64_t x, wg, wu, da, parts, tops, bytes;
    Work(int64_t N, int64_t D, int64_t F, bool back) {
        const int64_t D8 = up8(D), F8 = up8(F);
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
        parts = take(back ? (int64_t)shares(N, D8, F8) * 2 * F8 * D8 * 4 : 0);
        tops = take(back ? (Range::TOPS + 1) * 4 : 0);
        bytes = at;
    }
};

#define LAUNCHED                                                        \
    do {                                                                \
        if (hipGetLastError() != hipSuccess) return INET_POLICY_ELAUNCH; \
    } while (0)

static bool allow_lds(const void* kernel, int bytes) {
    return bytes <= 64 * 1024 ||
           hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
}

template <typename T, int ACT, bool BACK>
static int gates(const FfnShape& p, const Operand<T, true>& x, const Operand<T, true>& w, T* y, const T* dy, int64_t dy_s,
                 T* da, float* tops, hipStream_t st) {
    return by_size(size_for(p.N, 2 * (int64_t)p.F), [&](auto size) {
        typedef Sized<T, decltype(size)::value, true, true, true> P;
        auto k = ffn_gates_kernel<T, P, ACT, BACK>;
        if (!allow_lds((const void*)k, P::LDS)) return INET_POLICY_ELAUNCH;
        const int64_t all = tiles(p.N, P::BM) * tiles(p.F, P::BN / 2), grid = P::THREADS == 512 && all > 256 ? 256 : all;
        const bool ranged = BACK && std::is_same<T, _Float16>::value;
        for (int again = 0; again <= (ranged ? 1 : 0); ++again) {
            hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(P::THREADS), P::LDS, st, p, x, w, y, dy, dy_s, da, tops, again != 0);
            LAUNCHED;
        }
        return INET_POLICY_OK;
    });
}
template <typename T, bool BACK, typename... A> static int gates_for(int act, const A&... a) {
    return act == INET_POLICY_SILU ? gates<T, INET_POLICY_SILU, BACK>(a...)
           : act == INET_POLICY_GELU ? gates<T, INET_POLICY_GELU, BACK>(a...) : gates<T, INET_POLICY_RELU, BACK>(a...);
}

template <typename T, bool RA, bool CA, typename O>
static int product(int size, const Operand<T, RA>& a, const Operand<T, CA>& b, const Operand<T, RA>& a2,
                   const Operand<T, CA>& b2, int64_t K, int count, int64_t share, O* C,
                   int64_t rows, int64_t cols, bool vec, const float* unscale, hipStream_t st) {
    return by_size(size, [&](auto sz) {
        typedef Sized<T, decltype(sz)::value, RA, CA, false> P;
        auto k = ffn_product_kernel<T, P, RA, CA, O>;
        if (!allow_lds((const void*)k, P::LDS)) return INET_POLICY_ELAUNCH;
        const int64_t grid = tiles(rows, P::BM) * tiles(cols, P::BN);
        hipLaunchKernelGGL(k, dim3((unsigned)(grid * count)), dim3(P::THREADS), P::LDS, st, a, b, a2, b2, K, share, C, rows,
                           cols, vec, unscale);
        LAUNCHED;
        return INET_POLICY_OK;
    });
}

template <typename T> static int run(const InetFfn& a, const InetFfnGrad* d, hipStream_t st) {
    const Work at(a.N, a.D, a.F, d != nullptr);
    char* work = (char*)a.work;
    const int D8 = (int)up8(a.D), F8 = (int)up8(a.F);
    Operand<T, true> x{(const T*)a.x, nullptr, a.x_s, 0, a.N};
    Operand<T, true> w{(const T*)a.w_gate, (const T*)a.w_up, a.w_gate_s, a.w_up_s, a.F};
    if (D8 != a.D) {
        struct { const T* in; int64_t s, rows; T* out; } pads[3] = {{x.p, a.x_s, a.N, (T*)(work + at.x)},
                                                                    {w.p, a.w_gate_s, a.F, (T*)(work + at.wg)},
                                                                    {w.p2, a.w_up_s, a.F, (T*)(work + at.wu)}};
        for (auto& q : pads) {
            hipLaunchKernelGGL(ffn_pad_kernel<T>, dim3(blocks256(q.rows * D8)), dim3(256), 0, st, q.in, q.s, q.rows,
                               a.D, q.out, D8);
            LAUNCHED;
        }
        x.p = pads[0].out, w.p = pads[1].out, w.p2 = pads[2].out;
        x.st = w.st = w.st2 = D8;
    }
    auto by4 = [](const void* p, int64_t s) { return (uintptr_t)p % 8 == 0 && s % 4 == 0; };
    FfnShape p{a.N, a.y_s, D8, a.F, F8, d ? by4(d->d_y, d->d_y_s) : by4(a.y, a.y_s)};
    if (!d) return gates_for<T, false>(a.act, p, x, w, (T*)a.y, (const T*)nullptr, 0, (T*)nullptr, (float*)nullptr, st);
    T* da = (T*)(work + at.da);
    float* tops = (float*)(work + at.tops);
    const float* unscale = std::is_same<T, _Float16>::value ? tops + Range::TOPS : nullptr;
    if (int rc = gates_for<T, true>(a.act, p, x, w, (T*)nullptr, (const T*)d->d_y, d->d_y_s, da, tops, st)) return rc;
    if (d->d_x) {
        const Operand<T, true> dg{da, nullptr, 2 * F8, 0, a.N}, du{da + F8, nullptr, 2 * F8, 0, a.N};
        const Operand<T, false> wg{w.p, nullptr, w.st, 0, D8}, wu{w.p2, nullptr, w.st2, 0, D8};
        if (int rc = product<T, true, false, T>(size_for(a.N, D8), dg, wg, du, wu, a.F, 1, F8, (T*)d->d_x, a.N, a.D,
                                                by4(d->d_x, a.D), unscale, st))
            return rc;
    }
    if (d->d_w_gate || d->d_w_up) {
        const Operand<T, false> dat{da, nullptr, 2 * F8, 0, 2 * F8}, xt{x.p, nullptr, x.st, 0, D8}, no{};
        const int s = shares(a.N, D8, F8);
        const int64_t share = (tiles(a.N, s) + BK - 1) / BK * BK, one = (int64_t)2 * F8 * D8;
        float* parts = (float*)(work + at.parts);
        if (int rc = product<T, false, false, float>(dw_size(D8, F8), dat, xt, no, no, a.N, s, share, parts, 2 * F8, D8, true,
                                                      nullptr, st))
            return rc;
        for (int m = 0; m < 2; ++m) {
            T* out = (T*)(m ? d->d_w_up : d->d_w_gate);
            if (!out) continue;
            hipLaunchKernelGGL(ffn_add_kernel<T>, dim3(blocks256((int64_t)a.F * a.D)), dim3(256), 0, st,
                               parts + (int64_t)m * F8 * D8, s, one, (int64_t)a.F, a.D, D8, out, unscale);
            LAUNCHED;
        }
    }
    return INET_POLICY_OK;
}

static int check(const InetFfn* a, bool back) {
    if (!a || a->N < 0 || a->D < 1 || a->F < 1 || a->act < 0 || a->act > 2 || a->dtype < 0 || a->dtype > 2)
        return INET_POLICY_EINVAL;
    if (a->dtype == INET_POLICY_F32 || a->D > 1 << 20 || a->F > 1 << 20) return INET_POLICY_EUNSUPPORTED;
    for (int64_t s : {a->x_s, a->w_gate_s, a->w_up_s})       // (a tile's offsets are 32-bit)
        if (s < 0 || s > (int64_t)1 << 22) return INET_POLICY_EUNSUPPORTED;
    if (a->N > (int64_t)1 << 23) return INET_POLICY_EUNSUPPORTED;
    if (tiles(a->N, 64) * tiles(a->F, 32) > GRID_MAX || tiles(a->N, 64) * tiles(a->D, 64) > GRID_MAX)
        return INET_POLICY_EUNSUPPORTED;     // (workgroups a launch)
    if (back) {                              // (and of the weights' gradients, of 512 lanes for tiles of 256)
        const int64_t D8 = up8(a->D), F8 = up8(a->F), big = dw_size(D8, F8) == 2 ? 2 : 1;
        if (tiles(2 * F8, 128 * big) * tiles(D8, 128 * big) * shares(a->N, D8, F8) > GRID_MAX / big)
            return INET_POLICY_EUNSUPPORTED;
    }
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
            hipLaunchKernelGGL(ffn_add_kernel<T>, dim3(blocks256(one)), dim3(256), 0, st, (const float*)nullptr, 0,
                               (int64_t)0, (int64_t)a.F, a.D, a.D, (T*)out, (const float*)nullptr);
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
    if (int rc = pol::check(a, false)) return rc;
    if (a->N == 0) return INET_POLICY_OK;
    if (!a->y) return INET_POLICY_EINVAL;
    return a->dtype == INET_POLICY_BF16 ? pol::run<__bf16>(*a, nullptr, (hipStream_t)stream)
                                        : pol::run<_Float16>(*a, nullptr, (hipStream_t)stream);
}

int32_t inet_policy_ffn_backward(const InetFfn* a, const InetFfnGrad* d, void* stream) {
    if (int rc = pol::check(a, true)) return rc;
    if (!d) return INET_POLICY_EINVAL;
    if (a->N == 0)                            // (no rows: the weights' gradients are zero)
        return a->dtype == INET_POLICY_BF16 ? pol::zero_weights<__bf16>(*a, *d, (hipStream_t)stream)
                                            : pol::zero_weights<_Float16>(*a, *d, (hipStream_t)stream);
    if (!d->d_y || !a->work) return INET_POLICY_EINVAL;
    return a->dtype == INET_POLICY_BF16 ? pol::run<__bf16>(*a, d, (hipStream_t)stream)
                                        : pol::run<_Float16>(*a, d, (hipStream_t)stream);
}

}  // extern "C"
