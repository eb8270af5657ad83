// Per-head RMS norm of queries and keys, rotation by one or several position
// axes and KV append, in one pass over a step's new rows (gfx950).
//
// Per head row x of D elements, with the pairs (i, i + half) of the first
// 2 * half dims and the position of axis a(i) of the row's token:
//     y    = x / sqrt(mean(x^2) + eps) * w             (only with a weight w)
//     phi  = position[a(i)][t] * inv_freq[i]
//     out  = (y1 cos phi - y2 sin phi, y2 cos phi + y1 sin phi)
// Everything between the load and the one rounding at the store is fp32; the
// angle is reduced to a fraction of a turn in fp64 (positions of 2^31 times a
// frequency of one keep 1e-7 of a turn; an fp32 product loses 0.01 rad from
// position 1e5 on).
//
// Bound by HBM: each row is read once and written once (k and v rows only to
// the pool unless k_out asks for them).  A group of LPR lanes holds a head row,
// two 16-byte units per lane: units l and half / W + l, so that both elements
// of a pair are in one lane, or two neighbouring units of the unrotated tail.
// The sum of squares is a DPP reduction over the group.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"

namespace llkv {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 128;   // head_dim up to 256
constexpr int kMostAngles = 512; // of a work-group's tokens

struct NormRopeArgs {
    void* qo;
    void* ko;          // may be null: k rows go to the pool only
    const void* q;     // may be null
    const void* k;
    const void* v;
    void* kp;
    void* vp;
    int64_t qs, ks, vs, qos, kos;   // elements between tokens
    const int64_t* slots;
    const int* pos;    // [axes][T]
    const float* freq;
    const float* qw;   // null: no norm
    const float* kw;
    float eps;
    int T, Hq, Hkv, D, half, axes;
    uint32_t axis[kMaxPairs / 16];   // 2 bits per pair
};

// cos and sin of position * frequency; the angle's turns are split off in fp64.
__device__ inline void angle(int pos, float freq, float& c, float& s) {
    constexpr double kInv2Pi = 0.15915494309189533577;
    const double turns = (double)pos * ((double)freq * kInv2Pi);
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
}

__device__ inline void rotate_pair(float c, float s, float& x1, float& x2) {
    const float a = x1 * c - x2 * s;
    x2 = x2 * c + x1 * s;
    x1 = a;
}

// The 2-bit axis of pair i (a chain of selects: an indexed kernel argument
// would be copied to scratch memory).
__device__ inline uint32_t axis_word(const NormRopeArgs& a, int word) {
    uint32_t w = a.axis[0];
#pragma unroll
    for (int j = 1; j < kMaxPairs / 16; ++j) w = word == j ? a.axis[j] : w;
    return w;
}

// W consecutive floats from a 16-byte aligned address.
template <int W>
__device__ inline void load_floats(const float* p, float* f) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(p + i);
        f[i] = x.x;
        f[i + 1] = x.y;
        f[i + 2] = x.z;
        f[i + 3] = x.w;
    }
}

// Where row r of token t (q rows, then k rows, then v rows) is read and written.
template <typename T>
struct Row {
    const T* src;
    T* dst;    // null: not written
    T* dst2;   // the pool row of a k row that is also written to ko; null otherwise
    const float* w;
    bool rotated;
};

template <typename T>
__device__ inline Row<T> row_of(const NormRopeArgs& a, int t, int r, int64_t slot) {
    Row<T> o;
    o.dst2 = nullptr;
    if (r < a.Hq) {
        o.src = reinterpret_cast<const T*>(a.q) + t * a.qs + (int64_t)r * a.D;
        o.dst = reinterpret_cast<T*>(a.qo) + t * a.qos + (int64_t)r * a.D;
        o.w = a.qw;
        o.rotated = true;
        return o;
    }
    const bool isk = r < a.Hq + a.Hkv;
    const int h = r - a.Hq - (isk ? 0 : a.Hkv);
    const int64_t row = (slot * a.Hkv + h) * a.D;
    o.src = isk ? reinterpret_cast<const T*>(a.k) + t * a.ks + (int64_t)h * a.D
                : reinterpret_cast<const T*>(a.v) + t * a.vs + (int64_t)h * a.D;
    o.dst = slot < 0 ? nullptr : reinterpret_cast<T*>(isk ? a.kp : a.vp) + row;
    if (isk && a.ko) {
        o.dst2 = o.dst;
        o.dst = reinterpret_cast<T*>(a.ko) + t * a.kos + (int64_t)h * a.D;
    }
    o.w = isk ? a.kw : nullptr;
    o.rotated = isk;
    return o;
}

// 16-byte units.  Grid (groups of tpw tokens, slices of a group's rows): a work-group
// takes rows [slice, slice + per) of its tokens' tpw * R head rows, 256 / LPR at a
// time, and the tokens' tpw * half angles from LDS, which its threads compute once
// while their first rows are on the way.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a, int tpw, int per) {
    constexpr int W = Chunk<T>::VEC;
    constexpr int RPI = 256 / LPR;   // rows at a time
    constexpr int NI = 2;            // of them in flight
    __shared__ alignas(16) float cs[2][kMostAngles];   // cosines, sines [token][pair]
    const int tid = threadIdx.x, l = tid % LPR;
    const int R = a.Hq + 2 * a.Hkv, NU = a.D / W, hu = a.half / W;
    const int t0 = blockIdx.x * tpw, tokens = min(tpw, a.T - t0);
    const int r0 = blockIdx.y * per, r1 = min(r0 + per, tokens * R);
    const bool rot = l < hu;
    const int ua = rot ? l : 2 * hu + 2 * (l - hu);
    const int ub = rot ? hu + l : ua + 1;
    const bool va = ua < NU, vb = ub < NU;
    uint4 xa[NI], xb[NI];
    Row<T> row[NI];
    int tok[NI];
    auto load = [&](int r) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int x = r + i * RPI + tid / LPR;
            tok[i] = x < r1 ? x / R : 0;
            xa[i] = xb[i] = make_uint4(0, 0, 0, 0);
            row[i].dst = row[i].dst2 = nullptr;
            row[i].w = nullptr;
            row[i].rotated = false;
            if (x < r1) {
                const int t = t0 + tok[i];
                row[i] = row_of<T>(a, t, x - tok[i] * R, a.slots[t]);
                if (va) xa[i] = *reinterpret_cast<const uint4*>(row[i].src + ua * W);
                if (vb) xb[i] = *reinterpret_cast<const uint4*>(row[i].src + ub * W);
            }
        }
    };
    // The angles' positions and frequencies before the rows (loads return in order).
    constexpr int NA = kMostAngles / 256;
    int pos[NA];
    float freq[NA];
#pragma unroll
    for (int j = 0; j < NA; ++j) {
        const int x = tid + 256 * j;
        pos[j] = 0;
        freq[j] = 0.0f;
        if (x < tokens * a.half) {
            const int k = x / a.half, i = x - k * a.half;
            const int axis = (int)(axis_word(a, i / 16) >> (2 * (i % 16)) & 3u);
            pos[j] = a.pos[(int64_t)axis * a.T + t0 + k];
            freq[j] = a.freq[i];
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    load(r0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NA; ++j) {
        const int x = tid + 256 * j;
        if (x < tokens * a.half) angle(pos[j], freq[j], cs[0][x], cs[1][x]);
    }
    __syncthreads();
    for (int r = r0; r < r1; r += NI * RPI) {
        if (r > r0) load(r);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            if (row[i].dst == nullptr && row[i].dst2 == nullptr) continue;
            if (row[i].rotated) {
                float f[2 * W];
                Chunk<T>::unpack(xa[i], f);
                Chunk<T>::unpack(xb[i], f + W);
                if (row[i].w != nullptr) {
                    float ss = 0.0f;
#pragma unroll
                    for (int e = 0; e < 2 * W; ++e) ss = fmaf(f[e], f[e], ss);
                    ss = group_sum<LPR>(ss);   // lanes of one group share a row and its branch
                    const float n = 1.0f / sqrtf(ss / (float)a.D + a.eps);
                    float wa[W], wb[W];
                    load_floats<W>(row[i].w + (va ? ua : 0) * W, wa);
                    load_floats<W>(row[i].w + (vb ? ub : 0) * W, wb);
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        f[e] *= n * wa[e];
                        f[W + e] *= n * wb[e];
                    }
                }
                if (rot) {
                    float c[W], s[W];
                    load_floats<W>(&cs[0][tok[i] * a.half + l * W], c);
                    load_floats<W>(&cs[1][tok[i] * a.half + l * W], s);
#pragma unroll
                    for (int e = 0; e < W; ++e) rotate_pair(c[e], s[e], f[e], f[W + e]);
                }
                xa[i] = Chunk<T>::pack(f);
                xb[i] = Chunk<T>::pack(f + W);
            }
            if (row[i].dst != nullptr) {
                if (va) *reinterpret_cast<uint4*>(row[i].dst + ua * W) = xa[i];
                if (vb) *reinterpret_cast<uint4*>(row[i].dst + ub * W) = xb[i];
            }
            if (row[i].dst2 != nullptr) {
                if (va) *reinterpret_cast<uint4*>(row[i].dst2 + ua * W) = xa[i];
                if (vb) *reinterpret_cast<uint4*>(row[i].dst2 + ub * W) = xb[i];
            }
        }
    }
}

// Any head_dim up to 256, any even rotary_dim, any alignment: one wave per
// head row, lane l holding pairs l, l + 64 and dims 2 * half + l, .. + 64 j.
template <typename T>
__global__ __launch_bounds__(256) void norm_rope_generic_kernel(NormRopeArgs a) {
    const int lane = threadIdx.x & 63;
    const int R = a.Hq + 2 * a.Hkv;
    const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = wave / R;
    if (t >= a.T) return;
    const Row<T> row = row_of<T>(a, t, wave - t * R, a.slots[t]);
    if (row.dst == nullptr && row.dst2 == nullptr) return;
    float f[8];   // pair halves (0, 1), (2, 3), then the tail
    int dim[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = lane + 64 * j;
        dim[2 * j] = i < a.half ? i : -1;
        dim[2 * j + 1] = i < a.half ? a.half + i : -1;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int d = 2 * a.half + lane + 64 * j;
        dim[4 + j] = d < a.D ? d : -1;
    }
    if (!row.rotated) {   // a v row: moved bit for bit
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (dim[j] >= 0) row.dst[dim[j]] = row.src[dim[j]];
        return;
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        f[j] = 0.0f;
        if (dim[j] >= 0) f[j] = Elem<T>::to_f32(row.src[dim[j]]);
        ss = fmaf(f[j], f[j], ss);
    }
    if (row.w != nullptr) {
        const float n = 1.0f / sqrtf(wave_sum(ss) / (float)a.D + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (dim[j] >= 0) f[j] *= n * row.w[dim[j]];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = lane + 64 * j;
        if (i >= a.half) continue;
        float c, s;
        const uint32_t axis = (axis_word(a, i / 16) >> (2 * (i % 16))) & 3u;
        angle(a.pos[(int64_t)axis * a.T + t], a.freq[i], c, s);
        rotate_pair(c, s, f[2 * j], f[2 * j + 1]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (dim[j] < 0) continue;
        if (row.dst != nullptr) row.dst[dim[j]] = Elem<T>::from_f32(f[j]);
        if (row.dst2 != nullptr) row.dst2[dim[j]] = Elem<T>::from_f32(f[j]);
    }
}

// Few tokens: one per group, its rows spread over work-groups.  Many: up to four (512
// angles) per work-group, which then compute two angles a thread (28/4/128 bf16 with
// three axes, 5001 tokens: 40 us with every wave computing its own).
template <typename T, int LPR>
void launch_units(const NormRopeArgs& a, hipStream_t st) {
    constexpr int RPI = 256 / LPR;
    const int R = a.Hq + 2 * a.Hkv;
    const int most = std::max(1, std::min(4, a.half > 0 ? kMostAngles / a.half : 4));
    const int tpw = (int)std::max<int64_t>(1, std::min<int64_t>(most, a.T / (4ll * device_cus())));
    const int per = tpw > 1 ? tpw * R : std::min(R, 2 * RPI);
    norm_rope_kernel<T, LPR><<<dim3((a.T + tpw - 1) / tpw, (tpw * R + per - 1) / per), 256, 0, st>>>(a, tpw, per);
}

template <typename T>
int launch(const NormRopeArgs& a, bool vec, hipStream_t st) {
    if (vec) {
        const int lanes = (a.D / Chunk<T>::VEC + 1) / 2;   // at most 32
        if (lanes <= 4) launch_units<T, 4>(a, st);
        else if (lanes <= 8) launch_units<T, 8>(a, st);
        else if (lanes <= 16) launch_units<T, 16>(a, st);
        else launch_units<T, 32>(a, st);
    } else {
        const int64_t waves = (int64_t)a.T * (a.Hq + 2 * a.Hkv);
        norm_rope_generic_kernel<T><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a);
    }
    return check_launch("llkv_qk_norm_rope_append");
}

}  // namespace
}  // namespace llkv

using namespace llkv;

extern "C" int llkv_qk_norm_rope_append(void* q_out, void* k_out, const void* q, const void* k, const void* v,
                                        int64_t q_out_stride, int64_t k_out_stride, int64_t q_stride,
                                        int64_t k_stride, int64_t v_stride, void* k_pool, void* v_pool,
                                        const int64_t* slot_mapping, const int* positions, int num_axes,
                                        const uint8_t* pair_axis, const float* inv_freq, const float* q_weight,
                                        const float* k_weight, float eps, int num_tokens, int num_q_heads,
                                        int num_kv_heads, int head_dim, int rotary_dim, int dtype, void* stream) {
    const char* fn = "llkv_qk_norm_rope_append";
    if (num_tokens == 0) return LLKV_OK;
    if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || (q && num_q_heads <= 0))
        return set_error(LLKV_ERR_INVALID, "%s: bad shape arguments", fn);
    if (head_dim > 256) return set_error(LLKV_ERR_UNSUPPORTED, "%s: head_dim too large (%d > 256)", fn, head_dim);
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
        return set_error(LLKV_ERR_INVALID, "%s: rotary_dim %d must be even and in [0, %d]", fn, rotary_dim, head_dim);
    const size_t es = dtype_bytes(dtype);
    if (es == 0) return set_error(LLKV_ERR_INVALID, "%s: unsupported dtype %d", fn, dtype);
    if (!k || !v || !k_pool || !v_pool || !slot_mapping || (q && !q_out) ||
        (rotary_dim > 0 && (!positions || !inv_freq)))
        return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    if (rotary_dim > 0 && (num_axes < 1 || num_axes > kMaxAxes))
        return set_error(LLKV_ERR_INVALID, "%s: num_axes %d must be in [1, %d]", fn, num_axes, kMaxAxes);
    if (rotary_dim > 0 && num_axes > 1 && !pair_axis)
        return set_error(LLKV_ERR_INVALID, "%s: %d axes need pair_axis", fn, num_axes);
    if (!(eps >= 0.0f)) return set_error(LLKV_ERR_INVALID, "%s: eps must not be negative", fn);
    const int hq = q ? num_q_heads : 0;
    const int64_t qrow = (int64_t)hq * head_dim, krow = (int64_t)num_kv_heads * head_dim;
    if (q_stride < 0 || k_stride < 0 || v_stride < 0 || (q && q_out_stride < qrow && num_tokens > 1) ||
        (k_out && k_out_stride < krow && num_tokens > 1))
        return set_error(LLKV_ERR_INVALID, "%s: bad strides", fn);
    if ((int64_t)num_tokens * (hq + 2ll * num_kv_heads) > (1ll << 31) - 256)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: 2^31 or more head rows in one call", fn);
    NormRopeArgs a = {};
    a.qo = q_out;
    a.ko = k_out;
    a.q = q;
    a.k = k;
    a.v = v;
    a.kp = k_pool;
    a.vp = v_pool;
    a.qs = q_stride;
    a.ks = k_stride;
    a.vs = v_stride;
    a.qos = q_out_stride;
    a.kos = k_out_stride;
    a.slots = slot_mapping;
    a.pos = positions;
    a.freq = inv_freq;
    a.qw = q_weight;
    a.kw = k_weight;
    a.eps = eps;
    a.T = num_tokens;
    a.Hq = hq;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.half = rotary_dim / 2;
    a.axes = num_axes;
    if (num_axes > 1) {
        for (int i = 0; i < a.half; ++i) {
            if (pair_axis[i] >= num_axes)
                return set_error(LLKV_ERR_INVALID, "%s: pair_axis[%d] = %d is no axis of %d", fn, i, pair_axis[i],
                                 num_axes);
            a.axis[i / 16] |= (uint32_t)pair_axis[i] << (2 * (i % 16));
        }
    }
    const int W = (int)(16 / es);
    auto aligned = [&](const void* p, int64_t stride) { return !p || (((uintptr_t)p | (uintptr_t)(stride * es)) & 15) == 0; };
    const bool vec = a.half % W == 0 && head_dim % W == 0 && aligned(q, q_stride) && aligned(k, k_stride) &&
                     aligned(v, v_stride) && aligned(q ? q_out : nullptr, q_out_stride) && aligned(k_out, k_out_stride) &&
                     aligned(k_pool, 0) && aligned(v_pool, 0) && aligned(q_weight, 0) && aligned(k_weight, 0);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == LLKV_DTYPE_F32) return launch<float>(a, vec, st);
    if (dtype == LLKV_DTYPE_F16) return launch<_Float16>(a, vec, st);
    return launch<bf16_t>(a, vec, st);
}
