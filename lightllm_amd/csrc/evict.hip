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
constexpr int kBins = 2048;          // of a digit: two per thread
constexpr int kOnePass = 16;         // keys per thread of the one-launch form, at most
constexpr int kChunk = 8 * kSelThreads;   // keys per work-group of the other

// The three digits of a rank, from the top.
constexpr int kShift[3] = {21, 10, 0};

struct SelectArgs {
    const float* mass;
    const int* lens;
    int* keep;        // [N][Hkv][budget]
    int* counts;      // [N]
    float* mass_out;
    int64_t mass_bs, mass_hs, out_bs, out_hs;
    int width;        // of mass_out's rows
    int budget, sinks, recent, max_len, Hkv;
    // Keys in chunks (max_len > kOnePass * kSelThreads): per (sequence, kv head, chunk) the
    // digit histograms, 16 bits a bin, of the first and third digit and of the second, and
    // the number of keys above the threshold by the first and by the second digit.
    int chunks;
    uint32_t* hist[2];   // [units][chunks][kBins / 2]
    int* above[2];       // [units][chunks]
    int* found;          // [units][4]: (digits so far, keys left) after the first and the second digit
};

// Unsigned image of a total: larger totals are larger integers, the two zeros
// are equal, NaN is below everything, and 0xFFFFFFFF is above every total.
__device__ inline uint32_t rank_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t r = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return x != x ? 0u : r;
}

struct Unit {
    int n, kvh, L, count;
    const float* mass;
    float* out;
    int* keep;
    int64_t index;
};

__device__ inline Unit unit_of(const SelectArgs& a, int kvh, int n) {
    Unit u;
    const int len = a.lens[n];
    u.n = n;
    u.kvh = kvh;
    u.L = len < 0 ? 0 : (len > a.max_len ? a.max_len : len);
    u.count = min(u.L, a.budget);
    u.mass = a.mass + n * a.mass_bs + kvh * a.mass_hs;
    u.out = a.mass_out + n * a.out_bs + kvh * a.out_hs;
    u.index = (int64_t)n * a.Hkv + kvh;
    u.keep = a.keep + u.index * a.budget;
    return u;
}

// Ranks of the keys j0 + 1024 e + thread, 0 beyond the unit's last (with `valid` cleared).
template <int VPT>
struct Ranks {
    uint32_t r[VPT];
    uint32_t valid;

    __device__ inline void load(const SelectArgs& a, const Unit& u, int j0) {
        valid = 0;
        float x[VPT];
#pragma unroll
        for (int e = 0; e < VPT; ++e) {
            const int j = j0 + e * kSelThreads + (int)threadIdx.x;
            x[e] = u.mass[min(j, u.L - 1)];
        }
#pragma unroll
        for (int e = 0; e < VPT; ++e) {
            const int j = j0 + e * kSelThreads + (int)threadIdx.x;
            r[e] = (j < a.sinks || j >= u.L - a.recent) ? 0xFFFFFFFFu : rank_of(x[e]);
            valid |= (uint32_t)(j < u.L) << e;
        }
    }

    // Whether key e has the digits of `prefix` above digit `pass`.
    __device__ inline bool matches(int e, int pass, uint32_t prefix) const {
        return pass == 0 || (r[e] >> kShift[pass - 1]) == (prefix >> kShift[pass - 1]);
    }

    // Adds the digits `pass` of the keys whose digits above are those of `prefix`.  Totals
    // crowd in few bins of the first digit (equal ones in one bin of each): a wave whose
    // keys share a bin adds once.
    __device__ inline void histogram(int* hist, int pass, uint32_t prefix) const {
        const int shift = pass == 0 ? kShift[0] : (pass == 1 ? kShift[1] : kShift[2]);
        const int bits = pass == 2 ? 10 : 11;
#pragma unroll
        for (int e = 0; e < VPT; ++e) {
            const bool in = (valid >> e & 1u) && matches(e, pass, prefix);
            const int d = (int)(r[e] >> shift) & ((1 << bits) - 1);
            const uint64_t act = __builtin_amdgcn_ballot_w64(in);
            if (act == 0) continue;
            const int first = __builtin_ctzll(act);
            const int d0 = __builtin_amdgcn_readlane(d, first);
            if (__builtin_amdgcn_ballot_w64(in && d == d0) == act) {
                if ((int)(threadIdx.x & 63) == first) atomicAdd(&hist[d0], __builtin_popcountll(act));
            } else if (in) {
                atomicAdd(&hist[d], 1);
            }
        }
    }
};

struct SelectSmem {
    int hist[kBins];
    int wave_sum[kSelWaves];
    int digit, left;
    int gt[kOnePass * kSelWaves], eq[kOnePass * kSelWaves];
};

__device__ inline int wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int t = __shfl_up(v, off, 64);
        if (lane >= off) v += t;
    }
    return v;
}

// The digit at which the `left` largest end: thread t holds the numbers hi and lo
// of bins 2047 - 2t and 2046 - 2t.  Every thread gets the digit, how many of its
// bin are kept.
__device__ inline void find_digit(SelectSmem& s, int hi, int lo, int left, int& digit, int& keep) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int incl = wave_scan(hi + lo);
    if (lane == 63) s.wave_sum[wv] = incl;
    __syncthreads();
    int before = incl - hi - lo;
    for (int i = 0; i < wv; ++i) before += s.wave_sum[i];
    const int bin = kBins - 1 - 2 * (int)threadIdx.x;
    if (before < left && before + hi >= left) {
        s.digit = bin;
        s.left = left - before;
    } else if (before + hi < left && before + hi + lo >= left) {
        s.digit = bin - 1;
        s.left = left - before - hi;
    }
    __syncthreads();
    digit = s.digit;
    keep = s.left;
    __syncthreads();
}

// Writes the kept keys of these ranks: those above the threshold and, of the ones
// equal to it, the first `left`, ga and ea of which lie in earlier chunks.
template <int VPT>
__device__ inline void write_kept(const SelectArgs& a, const Unit& u, SelectSmem& s, const Ranks<VPT>& k, int j0,
                                  uint32_t threshold, int left, int ga, int ea) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
        const bool valid = k.valid >> e & 1u;
        const uint64_t bg = __builtin_amdgcn_ballot_w64(valid && k.r[e] > threshold);
        const uint64_t be = __builtin_amdgcn_ballot_w64(valid && k.r[e] == threshold);
        if (lane == 0) {
            s.gt[e * kSelWaves + wv] = __builtin_popcountll(bg);
            s.eq[e * kSelWaves + wv] = __builtin_popcountll(be);
        }
    }
    __syncthreads();
    if (wv < 2) {   // exclusive prefix sums in the order of the positions
        int* list = wv == 0 ? s.gt : s.eq;
        int run = wv == 0 ? ga : ea;
        for (int i0 = 0; i0 < VPT * kSelWaves; i0 += 64) {
            const int v = list[i0 + lane], incl = wave_scan(v);
            list[i0 + lane] = run + incl - v;
            run += __shfl(incl, 63, 64);
        }
    }
    __syncthreads();
    const uint64_t lower = (1ull << lane) - 1;
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
        const bool valid = k.valid >> e & 1u;
        const bool gt = valid && k.r[e] > threshold, eq = valid && k.r[e] == threshold;
        const int g = s.gt[e * kSelWaves + wv] + __builtin_popcountll(__builtin_amdgcn_ballot_w64(gt) & lower);
        const int q = s.eq[e * kSelWaves + wv] + __builtin_popcountll(__builtin_amdgcn_ballot_w64(eq) & lower);
        if (gt || (eq && q < left)) {
            const int j = j0 + e * kSelThreads + (int)threadIdx.x, i = g + min(q, left);
            u.keep[i] = j;
            u.out[i] = u.mass[j];
        }
    }
}

// What is there beside the kept keys: the rest of the rows, and units that keep all.
// Threads `first`, first + `step` .. of the unit; true when there is nothing to select.
__device__ inline bool select_rest(const SelectArgs& a, const Unit& u, int first, int step) {
    if (u.kvh == 0 && first == 0) a.counts[u.n] = u.count;
    for (int i = u.count + first; i < a.budget; i += step) u.keep[i] = -1;
    for (int i = u.count + first; i < a.width; i += step) u.out[i] = 0.0f;
    if (u.L > a.budget) return false;
    for (int i = first; i < u.count; i += step) {
        u.keep[i] = i;
        u.out[i] = u.mass[i];
    }
    return true;
}

// One launch: a work-group per (kv head, sequence), its ranks in registers.
template <int VPT>
__global__ __launch_bounds__(kSelThreads) void select_kernel(SelectArgs a) {
    __shared__ SelectSmem s;
    const Unit u = unit_of(a, blockIdx.x, blockIdx.y);
    const int tid = threadIdx.x;
    if (select_rest(a, u, tid, kSelThreads)) return;
    Ranks<VPT> k;
    k.load(a, u, 0);
    uint32_t prefix = 0;
    int left = u.count;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        s.hist[2 * tid] = s.hist[2 * tid + 1] = 0;
        __syncthreads();
        k.histogram(s.hist, pass, prefix);
        __syncthreads();
        int digit;
        find_digit(s, s.hist[kBins - 1 - 2 * tid], s.hist[kBins - 2 - 2 * tid], left, digit, left);
        prefix |= (uint32_t)digit << kShift[pass];
    }
    write_kept<VPT>(a, u, s, k, 0, prefix, left, 0, 0);
}

// The sum of a per-thread number over the work-group, in every thread.
__device__ inline int group_total(SelectSmem& s, int v) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int incl = wave_scan(v);
    if (lane == 63) s.wave_sum[wv] = incl;
    __syncthreads();
    int total = 0;
    for (int i = 0; i < kSelWaves; ++i) total += s.wave_sum[i];
    __syncthreads();
    return total;
}

// Chunks: one launch per digit and one for the output, grid (chunks, Hkv, N).
// Launch `pass` finds digit pass - 1 from all chunks' histograms (every
// work-group for itself) and leaves the histogram of its own chunk's digit
// `pass`; the last launch takes from them, too, how many of the kept keys lie in
// the chunks before its own.
__global__ __launch_bounds__(kSelThreads) void select_chunk_kernel(SelectArgs a, int pass) {
    __shared__ SelectSmem s;
    const Unit u = unit_of(a, blockIdx.y, blockIdx.z);
    const int tid = threadIdx.x, c = blockIdx.x, chunks = (u.L + kChunk - 1) / kChunk;
    if (pass == 3) select_rest(a, u, c * kSelThreads + tid, gridDim.x * kSelThreads);
    if (u.L <= a.budget || c >= chunks) return;   // uniform
    constexpr int VPT = kChunk / kSelThreads;
    Ranks<VPT> k;
    k.load(a, u, c * kChunk);
    const int64_t base = u.index * a.chunks;
    uint32_t prefix = 0;
    int left = u.count, digit = 0;
    int before_hi = 0, before_lo = 0;   // of the bins, in the chunks before this one
    if (pass > 0) {
        const int p = pass - 1;
        if (p > 0) {   // the digits above, found by the launch before
            prefix = (uint32_t)a.found[u.index * 4 + 2 * (p - 1)];
            left = a.found[u.index * 4 + 2 * (p - 1) + 1];
        }
        const uint32_t* h = a.hist[p & 1] + base * (kBins / 2) + (kBins / 2 - 1 - tid);
        int hi = 0, lo = 0;
        constexpr int kAhead = 16;
        for (int i0 = 0; i0 < chunks; i0 += kAhead) {
            uint32_t v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) v[i] = i0 + i < chunks ? h[(int64_t)(i0 + i) * (kBins / 2)] : 0u;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (i0 + i == c) {
                    before_hi = hi;
                    before_lo = lo;
                }
                lo += (int)(v[i] & 0xFFFFu);
                hi += (int)(v[i] >> 16);
            }
        }
        find_digit(s, hi, lo, left, digit, left);
        const uint32_t above = prefix;
        prefix |= (uint32_t)digit << kShift[p];
        if (pass < 3) {
            if (c == 0 && tid == 0) {
                a.found[u.index * 4 + 2 * p] = (int)prefix;
                a.found[u.index * 4 + 2 * p + 1] = left;
            }
            int n = 0;
#pragma unroll
            for (int e = 0; e < VPT; ++e)
                n += (k.valid >> e & 1u) && k.matches(e, p, above) && (k.r[e] >> kShift[p]) > (prefix >> kShift[p]);
            n = group_total(s, n);
            if (tid == 0) a.above[p][base + c] = n;
        }
    }
    if (pass < 3) {
        s.hist[2 * tid] = s.hist[2 * tid + 1] = 0;
        __syncthreads();
        k.histogram(s.hist, pass, prefix);
        __syncthreads();
        a.hist[pass & 1][(base + c) * (kBins / 2) + tid] = (uint32_t)s.hist[2 * tid] | (uint32_t)s.hist[2 * tid + 1] << 16;
        return;
    }
    const int bin = kBins - 1 - 2 * tid;   // the thread's bins: bin (hi), bin - 1 (lo)
    int ga = (bin > digit ? before_hi : 0) + (bin - 1 > digit ? before_lo : 0);
    for (int i = tid; i < c; i += kSelThreads) ga += a.above[0][base + i] + a.above[1][base + i];
    ga = group_total(s, ga);
    const int ea = group_total(s, bin == digit ? before_hi : (bin - 1 == digit ? before_lo : 0));
    write_kept<VPT>(a, u, s, k, c * kChunk, prefix, left, ga, ea);
}

// Units of a move.  (Native vectors: an array of HIP's uint4 went to LDS, addressed by
// the work-group's size, which is read from the launch packet in host memory: an
// in-place move of nine rows 17 us.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// Byte offset of head part h of position pos, or -1 where the table has no page.  No
// branch around the load, so that several of them are under way at once.
__device__ inline int64_t part_at(const CompactArgs& a, const int* table, int blocks, int n, int h, int pos) {
    const int index = max(pos, 0) / a.bs;
    const bool inside = pos >= 0 && index < blocks;
    const int64_t page = table[(int64_t)n * blocks + (inside ? index : 0)];
    const int64_t at = (page * a.bs + (max(pos, 0) - index * a.bs)) * a.row_bytes + h * a.part_bytes;
    return inside && page >= 0 ? at : -1;
}

// A load of a row that is not read again: past the caches, so that they keep what is
// written (32 x 1024 rows of 8 x 128 fp16 with its selection 72 us a call, 63 so; with
// stores past them as well 68).
template <typename U>
__device__ inline U load_once(const char* p) {
    if constexpr (sizeof(U) == 16) {
        return __builtin_nontemporal_load(reinterpret_cast<const U*>(p));
    } else {
        return *reinterpret_cast<const U*>(p);
    }
}

// Source and destination pages are different: a parallel copy.  Grid (blocks of
// kept positions, heads, N); `lanes` lanes of a work-group take a row part, in K and
// in V, and nothing more: with two rows a lane, an eighth fewer work-groups in flight
// behind the chain count -> position -> page -> row (32 x 1024 rows of 8 x 128 fp16
// 67 us, this 58).
template <typename U>
__global__ __launch_bounds__(256) void compact_copy_kernel(CompactArgs a, int lanes) {
    const int n = blockIdx.z, h = blockIdx.y;
    const int r = threadIdx.x / lanes, rows = 256 / lanes;
    const int i = blockIdx.x * rows + r;
    if (i >= min(a.counts[n], a.M)) return;
    const int64_t s = part_at(a, a.src, a.src_blocks, n, h, a.keep[((int64_t)n * a.H + h) * a.M + i]);
    const int64_t d = part_at(a, a.dst, a.dst_blocks, n, h, (a.start ? a.start[n] : 0) + i);
    if (s < 0 || d < 0) return;
    for (int u = threadIdx.x - r * lanes; u < a.units; u += lanes) {
        const int64_t off = (int64_t)u * sizeof(U);
        const U kk = load_once<U>(a.k + s + off), vv = load_once<U>(a.v + s + off);
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
constexpr int kLoads = 4;

template <typename U, int kUnits>
__global__ __launch_bounds__(256) void compact_inplace_kernel(CompactArgs a) {
    constexpr int kRows = 256 / kUnits;
    const int n = blockIdx.z >> 1, h = blockIdx.y;
    char* pool = blockIdx.z & 1 ? a.v : a.k;
    const int u = blockIdx.x * kUnits + threadIdx.x % kUnits;
    const int r = threadIdx.x / kUnits;
    const int64_t off = (int64_t)u * sizeof(U);
    const int count = min(a.counts[n], a.M), start = a.start ? a.start[n] : 0;
    const int* keep = a.keep + ((int64_t)n * a.H + h) * a.M;
    for (int i0 = 0; i0 < count; i0 += kLoads * kRows) {
        U x[kLoads];
        int from[kLoads];
        int64_t at[kLoads], to[kLoads];
#pragma unroll
        for (int e = 0; e < kLoads; ++e) from[e] = keep[min(i0 + e * kRows + r, count - 1)];
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
            const int i = i0 + e * kRows + r;
            at[e] = part_at(a, a.src, a.src_blocks, n, h, from[e]);
            to[e] = part_at(a, a.src, a.src_blocks, n, h, start + i);
            // (a row that stays is not touched)
            if (i >= count || u >= a.units || at[e] < 0 || from[e] == start + i) to[e] = -1;
        }
#pragma unroll
        for (int e = 0; e < kLoads; ++e)
            if (to[e] >= 0) x[e] = *reinterpret_cast<const U*>(pool + at[e] + off);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0x3F70);   // vmcnt(0): this wave's rows have arrived
        __builtin_amdgcn_s_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
        for (int e = 0; e < kLoads; ++e)
            if (to[e] >= 0) *reinterpret_cast<U*>(pool + to[e] + off) = x[e];
    }
}

struct SelectPlan {
    int chunks = 0;   // 0: one launch, no workspace
    size_t hist[2], above[2], found, total = 0;
};

SelectPlan select_plan(int N, int Hkv, int max_len) {
    SelectPlan p;
    if (max_len <= kOnePass * kSelThreads) return p;
    p.chunks = (int)(((int64_t)max_len + kChunk - 1) / kChunk);
    const size_t parts = (size_t)N * Hkv * p.chunks;
    for (int i = 0; i < 2; ++i) {
        p.hist[i] = p.total;
        p.total += parts * (kBins / 2) * sizeof(uint32_t);
    }
    for (int i = 0; i < 2; ++i) {
        p.above[i] = p.total;
        p.total += (parts * sizeof(int) + 15) & ~(size_t)15;
    }
    p.found = p.total;
    p.total += (size_t)N * Hkv * 4 * sizeof(int);
    return p;
}

int unit_bytes(int64_t part_bytes, const void* k, const void* v) {
    const uintptr_t m = (uintptr_t)k | (uintptr_t)v | (uintptr_t)part_bytes;
    return (m & 15) == 0 ? 16 : (m & 7) == 0 ? 8 : (m & 3) == 0 ? 4 : 2;
}

template <typename U>
void launch_compact(CompactArgs a, bool in_place, hipStream_t st) {
    a.units = (int)(a.part_bytes / sizeof(U));
    int lanes = 1;   // of a part: a power of two up to the work-group
    while (lanes < a.units && lanes < 256) lanes *= 2;
    const int per = 256 / lanes;
    constexpr int kMost = 32767;   // sequences per launch (a grid's extent in z)
    const int N = a.N;
    for (int n0 = 0; n0 < N; n0 += kMost) {
        CompactArgs b = a;
        b.N = std::min(N - n0, kMost);
        b.src += (int64_t)n0 * a.src_blocks;
        b.keep += (int64_t)n0 * a.H * a.M;
        b.counts += n0;
        if (b.start) b.start += n0;
        if (!in_place) {
            b.dst += (int64_t)n0 * a.dst_blocks;
            compact_copy_kernel<U><<<dim3((a.M + per - 1) / per, a.H, b.N), 256, 0, st>>>(b, lanes);
            continue;
        }
        // a few rows: wide parts of them in one round; many: narrow parts, for work-groups enough
        const bool few = a.M <= 256 / 64 * kLoads;
        const dim3 grid((a.units + (few ? 64 : 8) - 1) / (few ? 64 : 8), a.H, 2 * b.N);
        if (few) compact_inplace_kernel<U, 64><<<grid, 256, 0, st>>>(b);
        else compact_inplace_kernel<U, 8><<<grid, 256, 0, st>>>(b);
    }
}

}  // namespace
}  // namespace llkv

using namespace llkv;

extern "C" size_t llkv_evict_select_workspace_size(int num_seqs, int num_kv_heads, int max_seq_len) {
    if (num_seqs <= 0 || num_kv_heads <= 0 || max_seq_len < 0 || max_seq_len > INT32_MAX - kChunk) return 0;
    return select_plan(num_seqs, num_kv_heads, max_seq_len).total;
}

extern "C" int llkv_evict_select(int* keep, int* counts, float* mass_out, int64_t out_seq_stride,
                                 int64_t out_head_stride, int out_width, const float* mass, int64_t mass_seq_stride,
                                 int64_t mass_head_stride, const int* seq_lens, int num_seqs, int num_kv_heads,
                                 int max_seq_len, int budget, int sinks, int recent, void* workspace,
                                 size_t workspace_bytes, void* stream) {
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
    if (max_seq_len > INT32_MAX - kChunk || num_seqs > 65535 || num_kv_heads > 65535)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: too many sequences or keys", fn);
    const SelectPlan p = select_plan(num_seqs, num_kv_heads, max_seq_len);
    if (workspace_bytes < p.total || (p.total > 0 && !workspace))
        return set_error(LLKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, p.total);
    if (((uintptr_t)workspace & 15) != 0) return set_error(LLKV_ERR_INVALID, "%s: workspace not 16-byte aligned", fn);
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
    hipStream_t st = (hipStream_t)stream;
    const dim3 units(num_kv_heads, num_seqs);
    if (p.chunks > 0) {
        char* ws = reinterpret_cast<char*>(workspace);
        a.chunks = p.chunks;
        for (int i = 0; i < 2; ++i) {
            a.hist[i] = reinterpret_cast<uint32_t*>(ws + p.hist[i]);
            a.above[i] = reinterpret_cast<int*>(ws + p.above[i]);
        }
        a.found = reinterpret_cast<int*>(ws + p.found);
        const dim3 grid(p.chunks, num_kv_heads, num_seqs);
        for (int pass = 0; pass < 4; ++pass) select_chunk_kernel<<<grid, kSelThreads, 0, st>>>(a, pass);
    } else if (max_seq_len <= 4 * kSelThreads) {
        select_kernel<4><<<units, kSelThreads, 0, st>>>(a);
    } else if (max_seq_len <= 8 * kSelThreads) {
        select_kernel<8><<<units, kSelThreads, 0, st>>>(a);
    } else {
        select_kernel<kOnePass><<<units, kSelThreads, 0, st>>>(a);
    }
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
        case 16: launch_compact<u32x4>(a, !dst_table, st); break;
        case 8: launch_compact<u32x2>(a, !dst_table, st); break;
        case 4: launch_compact<uint32_t>(a, !dst_table, st); break;
        default: launch_compact<uint16_t>(a, !dst_table, st); break;
    }
    return check_launch(fn);
}
