// Cutting a paged cache down to the keys that attention uses (gfx950):
// selection by accumulated weight and the move of the chosen rows.
//
// llkv_evict_select, per (sequence, kv head) of L keys: all of them when
// L <= budget; otherwise the first `sinks`, the last `recent`, and of the
// others those with the largest totals, ties going to the lower position, up to
// `budget`.  The threshold is found digit by digit from the top (a radix
// select over the order-preserving integer image of the totals); the positions
// come out in rising order by a prefix sum.
//
// llkv_compact moves rows of K and V from positions keep[i] to positions
// start + i, for every head on its own or for all heads alike: to other pages,
// as one parallel copy, or within the same pages (an accepted branch of drafted
// tokens), where a row may only be overwritten once it has been read.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"

namespace llkv {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;

struct SelectArgs {
    const float* mass;
    const int* lens;
    int* keep;        // [N][Hkv][budget]
    int* counts;      // [N]
    float* mass_out;
    int64_t mass_bs, mass_hs, out_bs, out_hs;
    int width;        // of mass_out's rows
    int budget, sinks, recent, max_len, Hkv;
};

// Unsigned image of a total: larger totals are larger integers, the two zeros
// are equal, NaN is below everything, and 0xFFFFFFFF is above every total.
__device__ inline uint32_t rank_of(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ inline uint32_t rank_at(const SelectArgs& a, const float* mass, int j, int L) {
    if (j < a.sinks || j >= L - a.recent) return 0xFFFFFFFFu;
    return rank_of(mass[j]);
}

// Grid (Hkv, N).
__global__ __launch_bounds__(kSelThreads) void select_kernel(SelectArgs a) {
    __shared__ int hist[256];
    __shared__ int s_digit, s_left;
    __shared__ int s_above[kSelWaves], s_equal[kSelWaves];
    const int kvh = blockIdx.x, n = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int len = a.lens[n], L = len < 0 ? 0 : (len > a.max_len ? a.max_len : len);
    const int count = min(L, a.budget);
    const float* mass = a.mass + n * a.mass_bs + kvh * a.mass_hs;
    float* out = a.mass_out + n * a.out_bs + kvh * a.out_hs;
    int* keep = a.keep + ((int64_t)n * a.Hkv + kvh) * a.budget;
    if (kvh == 0 && tid == 0) a.counts[n] = count;
    for (int i = count + tid; i < a.budget; i += kSelThreads) keep[i] = -1;
    for (int i = count + tid; i < a.width; i += kSelThreads) out[i] = 0.0f;
    if (L <= a.budget) {   // uniform
        for (int i = tid; i < count; i += kSelThreads) {
            keep[i] = i;
            out[i] = mass[i];
        }
        return;
    }
    // The count-th largest rank: `prefix` holds its digits so far, `left` how many of the
    // ranks with that prefix are kept.
    uint32_t prefix = 0;
    int left = count;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < L; j += kSelThreads) {
            const uint32_t r = rank_at(a, mass, j, L);
            if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[(r >> shift) & 255], 1);
        }
        __syncthreads();
        if (wv == 0) {
            // lane l holds digits 255 - 4 l .. 252 - 4 l, the largest first
            int h[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h[e] = hist[255 - 4 * lane - e];
                sum += h[e];
            }
            int incl = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int t = __shfl_up(incl, off, 64);
                if (lane >= off) incl += t;
            }
            int before = incl - sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (before < left && before + h[e] >= left) {
                    s_digit = 255 - 4 * lane - e;
                    s_left = left - before;
                }
                before += h[e];
            }
        }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        left = s_left;
        __syncthreads();
    }
    // Kept: ranks above `prefix`, and the first `left` equal to it.
    int above = 0, equal = 0;   // of the rounds before
    for (int j0 = 0; j0 < L; j0 += kSelThreads) {
        const int j = j0 + tid;
        const uint32_t r = j < L ? rank_at(a, mass, j, L) : 0u;
        const bool gt = j < L && r > prefix, eq = j < L && r == prefix;
        const uint64_t bg = __builtin_amdgcn_ballot_w64(gt), be = __builtin_amdgcn_ballot_w64(eq);
        const uint64_t lower = (1ull << lane) - 1;
        if (lane == 0) {
            s_above[wv] = __builtin_popcountll(bg);
            s_equal[wv] = __builtin_popcountll(be);
        }
        __syncthreads();
        int ga = above, ea = equal, gsum = 0, esum = 0;
        for (int i = 0; i < kSelWaves; ++i) {
            if (i < wv) {
                ga += s_above[i];
                ea += s_equal[i];
            }
            gsum += s_above[i];
            esum += s_equal[i];
        }
        ga += __builtin_popcountll(bg & lower);
        ea += __builtin_popcountll(be & lower);
        if (gt || (eq && ea < left)) {
            const int i = ga + min(ea, left);
            keep[i] = j;
            out[i] = mass[j];
        }
        above += gsum;
        equal += esum;
        __syncthreads();
    }
}

struct CompactArgs {
    char* k;
    char* v;
    const int* src;      // block tables
    const int* dst;
    const int* keep;     // [N][H][M]
    const int* counts;   // [N]
    const int* start;    // [N] or null (0)
    int src_blocks, dst_blocks, bs, N, H, M, Hkv;
    int units;           // of U bytes per moved row part (a head's row, or all heads')
    int64_t row_bytes;   // Hkv * D * esize
    int64_t part_bytes;  // of a part: row_bytes / H
};

// Byte offset of head part h of position pos, or -1 where the table has no page.
__device__ inline int64_t part_at(const CompactArgs& a, const int* table, int blocks, int n, int h, int pos) {
    if (pos < 0 || pos / a.bs >= blocks) return -1;
    const int64_t page = table[(int64_t)n * blocks + pos / a.bs];
    if (page < 0) return -1;
    return (page * a.bs + pos % a.bs) * a.row_bytes + h * a.part_bytes;
}

// Source and destination pages are different: a flat copy, one unit of K and of
// V per lane.  Grid-stride over (sequence, kept position, head, unit).
template <typename U>
__global__ __launch_bounds__(256) void compact_copy_kernel(CompactArgs a) {
    const int64_t total = (int64_t)a.N * a.M * a.H * a.units;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < total; x += (int64_t)gridDim.x * 256) {
        const int64_t part = x / a.units;
        const int u = (int)(x - part * a.units);
        const int64_t row = part / a.H;
        const int h = (int)(part - row * a.H);
        const int n = (int)(row / a.M), i = (int)(row - (int64_t)n * a.M);
        if (i >= a.counts[n]) continue;
        const int64_t s = part_at(a, a.src, a.src_blocks, n, h, a.keep[((int64_t)n * a.H + h) * a.M + i]);
        const int64_t d = part_at(a, a.dst, a.dst_blocks, n, h, (a.start ? a.start[n] : 0) + i);
        if (s < 0 || d < 0) continue;
        const int64_t off = (int64_t)u * sizeof(U);
        const U kk = *reinterpret_cast<const U*>(a.k + s + off), vv = *reinterpret_cast<const U*>(a.v + s + off);
        *reinterpret_cast<U*>(a.k + d + off) = kk;
        *reinterpret_cast<U*>(a.v + d + off) = vv;
    }
}

// The same pages: rows move to lower positions (or stay) in rising order, so a
// work-group that reads kLoads * kRows rows, waits for all of them and only then
// writes them overwrites nothing that is still to be read: row i + 1's source
// lies above row i's destination, and the next round's sources above this
// round's destinations.  A work-group owns kUnits units of every row of one
// (sequence, head part) in K or in V, which no other work-group touches.
// Grid (units / kUnits, H, 2 N).
constexpr int kUnits = 8;
constexpr int kRows = 256 / kUnits;
constexpr int kLoads = 4;

template <typename U>
__global__ __launch_bounds__(256) void compact_inplace_kernel(CompactArgs a) {
    const int n = blockIdx.z >> 1, h = blockIdx.y;
    char* pool = blockIdx.z & 1 ? a.v : a.k;
    const int u = blockIdx.x * kUnits + threadIdx.x % kUnits;
    const int r = threadIdx.x / kUnits;
    const int64_t off = (int64_t)u * sizeof(U);
    const int count = min(a.counts[n], a.M), start = a.start ? a.start[n] : 0;
    const int* keep = a.keep + ((int64_t)n * a.H + h) * a.M;
    for (int i0 = 0; i0 < count; i0 += kLoads * kRows) {
        U x[kLoads];
        int64_t to[kLoads];
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
            const int i = i0 + e * kRows + r;
            to[e] = -1;
            if (i < count && u < a.units) {
                const int from = keep[i];
                const int64_t s = part_at(a, a.src, a.src_blocks, n, h, from);
                if (s >= 0 && from != start + i) {   // (a row that stays is not touched)
                    to[e] = part_at(a, a.src, a.src_blocks, n, h, start + i);
                    x[e] = *reinterpret_cast<const U*>(pool + s + off);
                }
            }
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0x3F70);   // vmcnt(0): this wave's rows have arrived
        __builtin_amdgcn_s_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
        for (int e = 0; e < kLoads; ++e)
            if (to[e] >= 0) *reinterpret_cast<U*>(pool + to[e] + off) = x[e];
    }
}

int unit_bytes(int64_t part_bytes, const void* k, const void* v) {
    const uintptr_t m = (uintptr_t)k | (uintptr_t)v | (uintptr_t)part_bytes;
    return (m & 15) == 0 ? 16 : (m & 7) == 0 ? 8 : (m & 3) == 0 ? 4 : 2;
}

template <typename U>
void launch_compact(CompactArgs a, bool in_place, hipStream_t st) {
    a.units = (int)(a.part_bytes / sizeof(U));
    if (!in_place) {
        const int64_t total = (int64_t)a.N * a.M * a.H * a.units;
        const unsigned grid = (unsigned)std::min<int64_t>((total + 255) / 256, 1 << 20);
        compact_copy_kernel<U><<<grid, 256, 0, st>>>(a);
        return;
    }
    constexpr int kMost = 32767;   // sequences per launch (a grid's extent in z)
    const int N = a.N;
    for (int n0 = 0; n0 < N; n0 += kMost) {
        CompactArgs b = a;
        b.N = std::min(N - n0, kMost);
        b.src += (int64_t)n0 * a.src_blocks;
        b.keep += (int64_t)n0 * a.H * a.M;
        b.counts += n0;
        if (b.start) b.start += n0;
        compact_inplace_kernel<U><<<dim3((a.units + kUnits - 1) / kUnits, a.H, 2 * b.N), 256, 0, st>>>(b);
    }
}

}  // namespace
}  // namespace llkv

using namespace llkv;

extern "C" int llkv_evict_select(int* keep, int* counts, float* mass_out, int64_t out_seq_stride,
                                 int64_t out_head_stride, int out_width, const float* mass, int64_t mass_seq_stride,
                                 int64_t mass_head_stride, const int* seq_lens, int num_seqs, int num_kv_heads,
                                 int max_seq_len, int budget, int sinks, int recent, void* stream) {
    const char* fn = "llkv_evict_select";
    if (num_seqs == 0) return LLKV_OK;
    if (num_seqs < 0 || num_kv_heads <= 0 || max_seq_len < 0)
        return set_error(LLKV_ERR_INVALID, "%s: bad shape arguments", fn);
    if (budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
        return set_error(LLKV_ERR_INVALID, "%s: %d sinks and %d recent keys of a budget of %d", fn, sinks, recent, budget);
    if (!keep || !counts || !mass_out || !mass || !seq_lens) return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    if (mass_head_stride < max_seq_len || (num_seqs > 1 && mass_seq_stride < (int64_t)num_kv_heads * mass_head_stride))
        return set_error(LLKV_ERR_INVALID, "%s: totals of %lld keys a head for up to %d", fn,
                         (long long)mass_head_stride, max_seq_len);
    if (out_width < std::min(budget, max_seq_len) || out_head_stride < out_width ||
        (num_seqs > 1 && out_seq_stride < (int64_t)num_kv_heads * out_head_stride))
        return set_error(LLKV_ERR_INVALID, "%s: %d kept totals do not fit rows of %d", fn, std::min(budget, max_seq_len),
                         out_width);
    if (max_seq_len > INT32_MAX - 2 * kSelThreads || num_seqs > 65535)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: too many sequences or keys", fn);
    SelectArgs a = {};
    a.mass = mass;
    a.lens = seq_lens;
    a.keep = keep;
    a.counts = counts;
    a.mass_out = mass_out;
    a.mass_bs = mass_seq_stride;
    a.mass_hs = mass_head_stride;
    a.out_bs = out_seq_stride;
    a.out_hs = out_head_stride;
    a.width = out_width;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    a.max_len = max_seq_len;
    a.Hkv = num_kv_heads;
    select_kernel<<<dim3(num_kv_heads, num_seqs), kSelThreads, 0, (hipStream_t)stream>>>(a);
    return check_launch(fn);
}

extern "C" int llkv_compact(void* k_pool, void* v_pool, const int* src_table, int src_max_blocks, const int* dst_table,
                            int dst_max_blocks, const int* keep, int keep_heads, int max_keep, const int* counts,
                            const int* dst_start, int num_seqs, int num_kv_heads, int head_dim, int block_size,
                            int dtype, void* stream) {
    const char* fn = "llkv_compact";
    if (num_seqs == 0 || max_keep == 0) return LLKV_OK;
    if (num_seqs < 0 || max_keep < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || src_max_blocks <= 0 ||
        (dst_table && dst_max_blocks <= 0))
        return set_error(LLKV_ERR_INVALID, "%s: bad shape arguments", fn);
    if (keep_heads != 1 && keep_heads != num_kv_heads)
        return set_error(LLKV_ERR_INVALID, "%s: positions for %d heads of %d (1 or all)", fn, keep_heads, num_kv_heads);
    const size_t es = dtype_bytes(dtype);
    if (es == 0) return set_error(LLKV_ERR_INVALID, "%s: unsupported dtype %d", fn, dtype);
    if (!k_pool || !v_pool || !src_table || !keep || !counts) return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    const int64_t widest = std::max(src_max_blocks, dst_table ? dst_max_blocks : 0);
    if (widest * block_size > INT32_MAX - max_keep || num_kv_heads > 65535)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: block table too large", fn);
    CompactArgs a = {};
    a.k = reinterpret_cast<char*>(k_pool);
    a.v = reinterpret_cast<char*>(v_pool);
    a.src = src_table;
    a.dst = dst_table;
    a.keep = keep;
    a.counts = counts;
    a.start = dst_start;
    a.src_blocks = src_max_blocks;
    a.dst_blocks = dst_max_blocks;
    a.bs = block_size;
    a.N = num_seqs;
    a.H = keep_heads;
    a.M = max_keep;
    a.Hkv = num_kv_heads;
    a.row_bytes = (int64_t)num_kv_heads * head_dim * es;
    a.part_bytes = a.row_bytes / keep_heads;
    hipStream_t st = (hipStream_t)stream;
    switch (unit_bytes(a.part_bytes, k_pool, v_pool)) {
        case 16: launch_compact<uint4>(a, !dst_table, st); break;
        case 8: launch_compact<uint2>(a, !dst_table, st); break;
        case 4: launch_compact<uint32_t>(a, !dst_table, st); break;
        default: launch_compact<uint16_t>(a, !dst_table, st); break;
    }
    return check_launch(fn);
}
