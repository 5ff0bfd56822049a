// One control step of the gated delta rule (a rollout), the state updated in place, and the delta rule's C ABI.
//
// What bounds it is the state: 8 K V bytes a head, read and written once, against 6 K V operations. A wave takes one
// head's block of columns into its registers: LP lanes across the columns, VW each (one 16-byte load), 64 / LP rows at
// a time, RL such loads a lane; the sums over the rows are taken in the lane and then across the row groups.
// 131072 robots x 2 heads of 64 x 64: 1598 us for 8.73 GB, 5.5 TB/s; 512 robots x 2 heads of 32 x 32: 5.1 us, a launch and one
// round trip to memory.
#include "delta.h"
#include "delta_launch.h"

namespace pol {

template <typename T, int LP, int VW, int RL>
__global__ __launch_bounds__(256) void delta_step_kernel(InetDelta d, int blocks) {
    constexpr int RG = 64 / LP;                                  // rows a load
    typedef float Vec __attribute__((ext_vector_type(VW)));
    __shared__ float s_k[4][RL * RG], s_q[4][RL * RG];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane % LP, r0 = lane / LP;
    const int64_t unit = (int64_t)blockIdx.x * 4 + w, heads = (int64_t)d.B * d.H;
    const int64_t bh = unit / blocks;
    const bool live = bh < heads;
    const int b = live ? (int)(bh / d.H) : 0, h = live ? (int)(bh % d.H) : 0, hk = h / (d.H / d.Hk);
    const int col = ((int)(unit % blocks) * LP + c) * VW;
    const bool in = live && col < d.V;
    float* S = d.state_out + (bh * d.K) * d.V + col;
    Vec x[RL];
#pragma unroll
    for (int i = 0; i < RL; ++i) {
        const int row = i * RG + r0;
        x[i] = in && row < d.K ? *(const Vec*)(S + (int64_t)row * d.V) : Vec{};
    }
    if (live)
        for (int i = lane; i < RL * RG; i += 64) {
            s_k[w][i] = i < d.K ? (float)((const T*)d.k)[b * d.k_s[0] + hk * d.k_s[2] + i] : 0.0f;
            s_q[w][i] = i < d.K ? (float)((const T*)d.q)[b * d.q_s[0] + hk * d.q_s[2] + i] : 0.0f;
        }
    float keep = 1.0f, beta = 0.0f;
    Vec v = {};
    if (live) {
        const float g = gate_load(d.g, b * d.g_s[0] + h * d.g_s[2], d.gate_dtype);
        beta = gate_load(d.beta, b * d.beta_s[0] + h * d.beta_s[2], d.gate_dtype);
        keep = (d.reset && d.reset[b * d.reset_s[0]]) || (double)g < DECAY_MIN ? 0.0f : expf(g);
    }
    if (in)
        for (int e = 0; e < VW; ++e) v[e] = (float)((const T*)d.v)[b * d.v_s[0] + h * d.v_s[2] + col + e];
    __syncthreads();
    Vec read = {};
#pragma unroll
    for (int i = 0; i < RL; ++i) {
        const float kk = s_k[w][i * RG + r0];
        for (int e = 0; e < VW; ++e) {
            x[i][e] = keep != 0.0f ? keep * x[i][e] : 0.0f;      // (an emptied state is empty whatever it held)
            read[e] += kk * x[i][e];
        }
    }
#pragma unroll
    for (int o = LP; o < 64; o <<= 1)
        for (int e = 0; e < VW; ++e) read[e] += __shfl_xor(read[e], o);
    Vec out = {};
    for (int e = 0; e < VW; ++e) v[e] = beta * (v[e] - read[e]);
#pragma unroll
    for (int i = 0; i < RL; ++i) {
        const int row = i * RG + r0;
        const float kk = s_k[w][row], qq = s_q[w][row];
        for (int e = 0; e < VW; ++e) {
            x[i][e] += kk * v[e];
            out[e] += qq * x[i][e];
        }
        if (in && row < d.K) *(Vec*)(S + (int64_t)row * d.V) = x[i];
    }
#pragma unroll
    for (int o = LP; o < 64; o <<= 1)
        for (int e = 0; e < VW; ++e) out[e] += __shfl_xor(out[e], o);
    if (in && r0 == 0)
        for (int e = 0; e < VW; ++e) ((T*)d.o)[bh * d.V + col + e] = (T)(d.scale * out[e]);
}

template <typename T, int LP, int VW, int RL> static int launch(const InetDelta& d, hipStream_t st) {
    const int blocks = (d.V + LP * VW - 1) / (LP * VW);
    const int64_t grid = ((int64_t)d.B * d.H * blocks + 3) / 4;
    if (grid > GRID_MAX) return INET_POLICY_EUNSUPPORTED;
    auto k = delta_step_kernel<T, LP, VW, RL>;
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(256), 0, st, d, blocks);
    return hipGetLastError() == hipSuccess ? INET_POLICY_OK : INET_POLICY_ELAUNCH;
}

// rows a lane: the smallest build that holds K
template <typename T, int LP, int VW> static int rows(const InetDelta& d, hipStream_t st) {
    constexpr int RG = 64 / LP;
    const int need = (d.K + RG - 1) / RG;
    if constexpr (128 / RG > 16)
        if (need > 16) return launch<T, LP, VW, 32>(d, st);
    if constexpr (128 / RG > 8)
        if (need > 8) return launch<T, LP, VW, 16>(d, st);
    if (need > 4) return launch<T, LP, VW, 8>(d, st);
    return launch<T, LP, VW, 4>(d, st);
}

template <typename T> static int widths(const InetDelta& d, hipStream_t st) {
    // columns a lane: four where rows start on 16 bytes, else one; lanes across: the narrowest that takes all columns,
    // up to 16 (more rows a load, so a head of 128 columns is two waves' and keeps half the registers). us by 4, 8 and 16 lanes
    // of four and 16 of one, 4 heads of 64 rows: V = 16, 32768 robots 206, 220, 327, 216; V = 32, 512 robots 9, 8, 9, 10, 32768
    // robots 415, 419, 408, 427; V = 64 811, 839, 810, 844; V = 128 1691, 1678, 1606, 1795
    if (d.V % 4 || (uintptr_t)d.state_out % 16) return rows<T, 16, 1>(d, st);
    if (d.V <= 16) return rows<T, 4, 4>(d, st);
    return d.V <= 32 ? rows<T, 8, 4>(d, st) : rows<T, 16, 4>(d, st);
}

int delta_step(const InetDelta& d, hipStream_t st) {
    if (d.dtype == INET_POLICY_F32) return widths<float>(d, st);
    if (d.dtype == INET_POLICY_BF16) return widths<__bf16>(d, st);
    return widths<_Float16>(d, st);
}

// ------------------------------------------------------------------------------------------------ C ABI
static int elem_size(int dtype) { return dtype == INET_POLICY_F32 ? 4 : 2; }

static int check(const InetDelta* a) {
    if (!a || a->B < 0 || a->T < 0 || a->Hk < 1 || a->H < 1 || a->K < 1 || a->V < 1) return INET_POLICY_EINVAL;
    if (a->H % a->Hk || a->dtype < 0 || a->dtype > 2 || a->gate_dtype < 0 || a->gate_dtype > 2)
        return INET_POLICY_EINVAL;
    if (a->K > INET_POLICY_MAX_HEAD || a->V > INET_POLICY_MAX_HEAD) return INET_POLICY_EUNSUPPORTED;
    if ((int64_t)a->B * a->H > GRID_MAX) return INET_POLICY_EUNSUPPORTED;
    return INET_POLICY_OK;
}

// The way through a window. The matrices of a chunk and what they make grow with C, and with them the LDS a workgroup holds:
// by chunks of 32 three share a compute unit, by 64 two. 2048 robots of 4 heads of 64 x 64, bfloat16, training, us at 32 and
// 64 steps a chunk: 24 steps 275 and 875, 64 steps 740 and 1045, 200 steps 2534 and 3258.
// A window of a few robots is delta_split.hip's, which takes all its chunks at once but for the state's own chain (`groups`
// workgroups). From five chunks on and up to 96 groups: one pass and split by 32, us, training, bfloat16, 64 x 64:
//     T        16 groups      64 groups      96 groups      128 groups     256 groups
//     100       64,  63        71,  72        73,  77        72,  79
//     400      152, 110       165, 136       179, 156       185, 179       226, 268
//     1000     365, 203       391, 248       410, 317       442, 377       547, 596
//     2000     700, 320       773, 496       828, 604       873, 728      1055, 1132
// and at T = 1000 of other sizes and types:
//     forward alone   155,  82       160, 100       165, 113       165, 124       165, 211
//     128 x 128       459, 272       495, 380       550, 476       594, 559       769, 917
//     32 x 32         308, 210       331, 212       339, 218       347, 219       382, 328
//     float32         425, 215       471, 312       507, 413       553, 496       711, 821
//     its 128 x 128   588, 324       678, 550       758, 702       834, 853      1127, 1441
//     float16         419, 204       452, 270       473, 341       509, 425       630, 687
// (the two sides meet between 100 and 250 groups, the earlier the larger the heads; the rule keeps below the first). There the
// chain's length counts, and chunks of 64 halve it: at T = 2000, 16, 64 and 96 groups, 271, 480 and 624 us for the 320, 496 and
// 604 by 32, of 128 x 128 409, 745 and 965 for 480, 747 and 939, but of 32 x 32 218, 317 and 389 for 222, 297 and 344; up to
// T = 600 they gain nothing. Bfloat16 alone takes 64: float16's second plane makes them no faster (64 groups, T = 1000: 299
// by 32, 331 by 64), and float32's third does not fit the LDS.
static int64_t groups_of(const InetDelta* a) { return (int64_t)a->B * a->H * ((a->V + 63) / 64); }
static bool split(const InetDelta* a) {
    const int64_t chunks = ((int64_t)a->T + a->chunk - 1) / a->chunk;
    return chunks >= 5 && groups_of(a) <= 96;
}
static int chunk_of(const InetDelta* a) {
    return a->dtype == INET_POLICY_BF16 && a->T > 512 && groups_of(a) <= 96 ? 64 : 32;
}

static int check_window(const InetDelta* a) {
    if (int rc = check(a)) return rc;
    if (a->chunk != chunk_of(a)) return INET_POLICY_EINVAL;
    if ((int64_t)a->H * a->V > 1 << 22) return INET_POLICY_EUNSUPPORTED;      // (a chunk's offsets are 32-bit)
    const int64_t chunks = ((int64_t)a->T + a->chunk - 1) / a->chunk;
    if ((int64_t)a->B * a->H * chunks > GRID_MAX) return INET_POLICY_EUNSUPPORTED;
    return INET_POLICY_OK;
}

// whether the inputs' rows start on 16 bytes and hold whole groups of eight
static bool aligned(const InetDelta* a) {
    const int e = elem_size(a->dtype);
    auto rows = [&](const void* p, const int64_t* s) {
        return (uintptr_t)p % 16 == 0 && s[0] * e % 16 == 0 && s[1] * e % 16 == 0 && s[2] * e % 16 == 0;
    };
    return a->K % 8 == 0 && a->V % 8 == 0 && rows(a->k, a->k_s) && rows(a->q, a->q_s) && rows(a->v, a->v_s);
}

}  // namespace pol

extern "C" {

int32_t inet_policy_delta_chunk(const InetDelta* a) { return pol::check(a) ? 0 : pol::chunk_of(a); }

int64_t inet_policy_delta_work(const InetDelta* a, int32_t backward) {
    if (pol::check_window(a)) return -1;
    return a->B && pol::split(a) ? (int64_t)pol::delta_split_bytes(*a, backward != 0) : 0;
}

int32_t inet_policy_delta_forward(const InetDelta* a, void* stream) {
    if (int rc = pol::check_window(a)) return rc;
    if (a->B == 0) return INET_POLICY_OK;
    if (!a->state_out || a->state == a->state_out) return INET_POLICY_EINVAL;
    if (a->T > 0 && (!a->q || !a->k || !a->v || !a->g || !a->beta || !a->o)) return INET_POLICY_EINVAL;
    if (a->T > a->chunk && !a->err != !a->chunk_state) return INET_POLICY_EINVAL;
    if (pol::split(a) != (a->work != nullptr) || (a->work && (!a->err || (uintptr_t)a->work % 16)))
        return INET_POLICY_EINVAL;
    return pol::delta_forward(*a, pol::aligned(a) && (uintptr_t)a->o % 16 == 0, (hipStream_t)stream);
}

int32_t inet_policy_delta_backward(const InetDelta* a, const InetDeltaGrad* d, void* stream) {
    if (int rc = pol::check_window(a)) return rc;
    if (!d) return INET_POLICY_EINVAL;
    if (a->B == 0 || (a->T == 0 && !d->d_state)) return INET_POLICY_OK;
    if (a->T > 0 && (!a->q || !a->k || !a->v || !a->g || !a->beta || !a->err || !d->d_q || !d->d_k || !d->d_v || !d->d_g ||
                     !d->d_beta))
        return INET_POLICY_EINVAL;
    if (a->T > a->chunk && (!a->chunk_state || !d->chunk_grad || !d->err_grad)) return INET_POLICY_EINVAL;
    if (pol::split(a) != (a->work != nullptr) || (uintptr_t)a->work % 16) return INET_POLICY_EINVAL;
    if (a->H != a->Hk && a->T > 0 && !d->head_grad) return INET_POLICY_EINVAL;
    bool vec = pol::aligned(a);
    for (const void* p : {(const void*)a->err, (const void*)a->chunk_state, (const void*)d->err_grad, d->d_o,
                          (const void*)d->chunk_grad, (const void*)d->d_q, (const void*)d->d_k, (const void*)d->d_v,
                          (const void*)d->head_grad, (const void*)a->state, (const void*)d->d_state_out})
        vec = vec && (uintptr_t)p % 16 == 0;
    return pol::delta_backward(*a, *d, vec, (hipStream_t)stream);
}

int32_t inet_policy_delta_step(const InetDelta* a, void* stream) {
    if (int rc = pol::check(a)) return rc;
    if (a->T != 1) return INET_POLICY_EINVAL;
    if (a->B == 0) return INET_POLICY_OK;
    if (!a->q || !a->k || !a->v || !a->g || !a->beta || !a->o || !a->state_out) return INET_POLICY_EINVAL;
    return pol::delta_step(*a, (hipStream_t)stream);
}

}  // extern "C"
