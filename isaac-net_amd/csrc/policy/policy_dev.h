// Device helpers of the policy operators: element types, bfloat16 planes and the matrix instructions' fragments.
//
// Products of 32-bit precision on the bfloat16 matrix instructions. A value is held as a sum of planes, each the
// bfloat16 nearest to what the planes before it leave over: one plane is a bfloat16 value itself, two hold a float16
// value, three hold a float32 value to its last bit (3 x 8 significand bits). A product of two such sums keeps the
// plane products whose orders add up to at most ORD: ORD = 2 drops what is below 2^-24 of the product, ORD = 1 what is
// below 2^-16. The 32-bit matrix instruction has a sixteenth of the bfloat16 one's rate, six plane products (3 x 3
// planes, ORD = 2) a sixth, and a bfloat16 operand against three planes a third.
//
// Fragments of v_mfma_f32_16x16x32_bf16 (lane l, n = l % 16, g = l / 16): A holds row n, B column n, each at the
// contraction indexes 8 g .. 8 g + 7; the result holds column n at rows 4 g .. 4 g + 3. Two results stacked (rows 0..15
// and 16..31) are a B fragment of a 32-long contraction in the order perm(): index 16 t + 4 g + i at place
// 8 g + 4 t + i. Matrices that meet such a fragment are kept in that order, so a state or a row of values goes from one
// product into the next without leaving its registers.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#define DEV __device__ __forceinline__

namespace pol {

// workgroups of 256 lanes a launch: a grid has fewer than 2^32 lanes
constexpr int64_t GRID_MAX = (1 << 24) - 1;
// for `items` elements, a lane each; a kernel so launched strides over what is past the grid
inline unsigned blocks256(int64_t items) {
    const int64_t n = (items + 255) / 256;
    return (unsigned)(n < GRID_MAX ? n : GRID_MAX);
}

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int planes = 3, ord = 2; };
template <> struct Elem<__bf16> { static constexpr int planes = 1, ord = 1; };
template <> struct Elem<_Float16> { static constexpr int planes = 2, ord = 1; };

// eight consecutive elements, the first n of them inside the row (the others read as 0); vec: the row starts are
// aligned to 16 bytes and rows hold whole groups of eight
template <typename T> DEV void load8(const T* __restrict__ p, int n, bool vec, float (&x)[8]) {
    if (vec && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
        } else {
            typedef T V8 __attribute__((ext_vector_type(8)));
            const V8 a = *(const V8*)p;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < n ? (float)p[i] : 0.0f;
    }
}

// the same for four (vec: aligned to four elements)
template <typename T> DEV void load4(const T* __restrict__ p, int n, bool vec, float (&x)[4]) {
    if (vec && n >= 4) {
        typedef T V4 __attribute__((ext_vector_type(4)));
        const V4 a = *(const V4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)a[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < n ? (float)p[i] : 0.0f;
    }
}

template <int N> struct Frag { bf16x8 p[N]; };

// two values to bfloat16 in one instruction, and what they leave over
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
DEV uint32_t round2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
DEV float low_of(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
DEV float high_of(uint32_t u) { return __builtin_bit_cast(float, u & 0xffff0000u); }

// values to planes, two at a time: plane i of values 2 j, 2 j + 1 in out[i][j]
template <int N, int PAIRS> DEV void split_pairs(const float (&x)[2 * PAIRS], uint32_t (&out)[N][PAIRS]) {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
        float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t h = round2(a, b);
            out[i][j] = h;
            if (i + 1 < N) {
                a -= low_of(h);
                b -= high_of(h);
            }
        }
    }
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int N> DEV Frag<N> split8(const float (&x)[8]) {
    uint32_t u[N][4];
    split_pairs<N, 4>(x, u);
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) f.p[i] = __builtin_bit_cast(bf16x8, (u32x4{u[i][0], u[i][1], u[i][2], u[i][3]}));
    return f;
}

// two stacked 16 x 16 results as a B fragment
template <int N> DEV Frag<N> split_tiles(f32x4 lo, f32x4 hi) {
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return split8<N>(x);
}

// c + A B over a 32-long contraction; the small plane products first
template <int ORD, int NA, int NB> DEV f32x4 mma(const Frag<NA>& a, const Frag<NB>& b, f32x4 c) {
#pragma unroll
    for (int s = ORD; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[s - i], c, 0, 0, 0);
    return c;
}

// the same for several A against one B, plane product by plane product, so that no instruction waits for the one before it
template <int ORD, int NA, int NB, int R> DEV void mma_rows(const Frag<NA> (&a)[R], const Frag<NB>& b, f32x4 (&c)[R]) {
#pragma unroll
    for (int s = ORD; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    c[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[r].p[i], b.p[s - i], c[r], 0, 0, 0);
}

// c + A B over a 16-long contraction in 32 bits: a = A's row n at columns 4 g .. 4 g + 3, b a 16 x 16 result
DEV f32x4 mma32(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
}

// place of contraction index c in the order of two stacked results
DEV int perm(int c) { return (c & ~31) | ((c & 12) << 1) | ((c & 16) >> 2) | (c & 3); }

// four rows x 16 columns of 16-bit values in LDS, transposed: lanes 0..15 of a group point to four values each (lane n:
// row n / 4, columns 4 (n % 4) ..), and lane n receives column n
DEV bf16x4 read_tr(const __bf16* p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* Lds;
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p);
    return __builtin_bit_cast(bf16x4, v);
}

// a matrix of N planes in LDS, rows of ld elements (ld / 8 odd: 16 lanes' 16-byte reads fall on distinct banks)
template <int N> struct Planes {
    __bf16* p;
    int ld, plane;
    DEV Frag<N> frag(int row, int k8) const {            // eight elements from place k8 of a row
        Frag<N> f;
#pragma unroll
        for (int i = 0; i < N; ++i) f.p[i] = *(const bf16x8*)(p + i * plane + row * ld + k8);
        return f;
    }
    // the A fragment of the transpose: row 16 ct + n of it, contraction over rows 32 rp .. 32 rp + 31 in the order of two
    // stacked results. The matrix's columns are in the order perm().
    DEV Frag<N> tr_frag(int ct, int rp, int n, int g) const {
        Frag<N> f;
        const __bf16* at = p + (32 * rp + 4 * g + (n >> 2)) * ld + 32 * (ct >> 1) + (n & 3) * 8 + (ct & 1) * 4;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bf16x4 lo = read_tr(at + i * plane), hi = read_tr(at + i * plane + 16 * ld);
            f.p[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
    // rows 16 rt .. and columns 16 ct .. (columns in the order perm()) as a result's tile: lane column n, rows 4 g + e
    DEV f32x4 tr_tile(int ct, int rt, int n, int g) const {
        f32x4 x = {};
        const __bf16* at = p + (16 * rt + 4 * g + (n >> 2)) * ld + 32 * (ct >> 1) + (n & 3) * 8 + (ct & 1) * 4;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            const bf16x4 v = read_tr(at + i * plane);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += (float)v[e];
        }
        return x;
    }
    DEV void put1(int row, int place, float x) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const __bf16 h = (__bf16)x;
            p[i * plane + row * ld + place] = h;
            x -= (float)h;
        }
    }
    DEV void put4(int row, int place, float a, float b, float c, float d) const {
        const float x[4] = {a, b, c, d};
        uint32_t u[N][2];
        split_pairs<N, 2>(x, u);
#pragma unroll
        for (int i = 0; i < N; ++i) *(u32x2*)(p + i * plane + row * ld + place) = u32x2{u[i][0], u[i][1]};
    }
};

// inclusive sum over the wave's lanes
template <int CTRL, int ROWS> DEV int lane_shift(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, true);
}
template <int CTRL, int ROWS> DEV double lane_shift(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)lane_shift<CTRL, ROWS>((int)(uint32_t)u), hi = (uint32_t)lane_shift<CTRL, ROWS>((int)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <typename T> DEV T lane_scan(T x) {
    x += lane_shift<0x111, 0xf>(x);          // one, two, four, eight lanes along a row of 16
    x += lane_shift<0x112, 0xf>(x);
    x += lane_shift<0x114, 0xf>(x);
    x += lane_shift<0x118, 0xf>(x);
    x += lane_shift<0x142, 0xa>(x);          // rows 1 and 3 gain the last lane of the row before
    x += lane_shift<0x143, 0xc>(x);          // rows 2 and 3 that of row 1
    return x;
}

template <typename T> DEV void store4(T* p, int n, bool vec, const float (&x)[4]) {
    if (vec && n >= 4) {
        typedef T V4 __attribute__((ext_vector_type(4)));
        V4 v;
        for (int i = 0; i < 4; ++i) v[i] = (T)x[i];
        *(V4*)p = v;
    } else {
        for (int i = 0; i < 4; ++i) if (i < n) p[i] = (T)x[i];
    }
}

}  // namespace pol
