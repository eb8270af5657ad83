// Attention of several new rows per sequence over its paged cache, for few rows
// (gfx950): the arguments, the schedule and the wave-level body shared by the
// drafted-tree attention and by the decode step that keeps its weights
// (tree.hip).
//
// The P new rows of a sequence times the G query heads of a kv head are the
// columns of one problem, column c being row c / G under head c % G, so that
// every byte of K and V is read once for all of them:
//     S^T [keys x columns] = K Q^T,   O^T [dims x columns] = V^T P^T.
// A unit is a block of kCols columns of one (sequence, kv head) over the
// sequence's keys in tiles of 64.  The batch's T tiles (over all units, in the
// order sequence, kv head, column block) are shared equally by the work-groups
// of one resident set, whatever the mix of lengths and tree sizes: work-group
// w of W takes tiles [floor(w T / W), floor((w + 1) T / W)).  A unit inside one
// share is written out directly.  A unit that is cut leaves one partial per
// share, a normalised fp32 row and its log2-sum-exp2 per column, which a second
// kernel joins.  A share has at most two cut units, its first and its last, so
// that two partial slots per work-group are enough.
//
// Where most sequences have as many column blocks as the widest one, B > 1, the
// work-groups form teams of B neighbours: the teams share the tiles, and each
// member of a team runs the same tiles for a block of its own, so that K and V
// come from HBM once and from the XCD's L2 for the others.
#pragma once

#include "attn_common.h"
#include "decode_mfma.h"

namespace llkv {

constexpr int kTreeTile = 64;      // keys per tile: one page per wave
constexpr int kTreeSeqs = 512;     // sequences per launch (their prefix sums are in LDS; 1024 cost head_dim 128 a work-group per CU)

// A cut unit, left by the work-group w that it begins in for the second kernel: part
// j's slot is `slot` for j = 0, else 2 * (w + j * step).  parts 0: none begins there.
struct TreeCut {
    int q0, cols, c0, kvh, slot, parts, step;
};

struct TreeArgs {
    void* out;
    const void* q;
    const void* k;
    const void* v;
    const int* bt;
    const int* cu_q;      // null: one row per sequence, which sees every key
    const int* lens;
    const int* mask;      // [rows][words]; null with cu_q
    int words;
    int max_blocks, N, Hq, Hkv, D, bs;
    int max_len;          // keys beyond are cut off (the caller's bound)
    int nwg;
    TreeCut* cuts;        // [nwg]
    int* rounds;          // [nwg]: joining rounds of each work-group's cut unit, 0 without one
    int64_t* plan;        // [N + 1] prefix sums of column blocks x tiles (kept weights alone)
    float* part_o;        // [2 * nwg][kCols][D]
    float* part_lse;      // [2 * nwg][kCols]
    // Kept weights: scaled scores [N * Hkv * G][score_stride], log2-sum-exp2 of
    // the units that were not cut [N * Hq], and the totals.
    float* scores;
    float* lse;
    int64_t score_stride;
    float* mass;
    int64_t mass_bs, mass_hs;
    float scale_log2;     // last: beside nwg and plan the compiler loaded the three as one vector through LDS
};

struct TreeSeq {
    int q0, P, L, hist;   // hist: keys before row 0's own (L when one row sees all)
};

__device__ inline TreeSeq tree_seq(const TreeArgs& a, int n) {
    TreeSeq s;
    const int l = a.lens[n];
    const int cap = min(a.max_blocks * a.bs, a.max_len);
    s.L = l < 0 ? 0 : (l > cap ? cap : l);
    if (a.cu_q == nullptr) {
        s.q0 = n;
        s.P = 1;
        s.hist = s.L;
    } else {
        s.q0 = a.cu_q[n];
        s.P = max(a.cu_q[n + 1] - s.q0, 0);
        s.hist = s.L - s.P;
    }
    return s;
}

// A sequence with rows and no keys keeps one empty tile, which writes its zeros.
__device__ inline int tree_tiles(const TreeSeq& s) { return s.P == 0 ? 0 : max(1, (s.L + kTreeTile - 1) / kTreeTile); }

template <int COLS>
__device__ inline int tree_blocks(const TreeSeq& s, int G) {
    return (int)(((int64_t)s.P * G + COLS - 1) / COLS);
}

// Column block cb of (sequence n, kv head kvh), tiles [t0, t1).
struct TreeSeg {
    TreeSeq s;
    int n, kvh, cols, c0, t0, t1, slot;
    bool direct, stream;   // written out directly; K and V by streaming loads
};

__device__ inline int64_t wave_incl_scan64(int64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t t = __shfl_up((long long)v, off, 64);
        if (lane >= off) v += t;
    }
    return v;
}

// sP[n] = column blocks x tiles of sequences [0, n), n = 0 .. N, and, where sT is
// given, sT[n] = their tiles; wave 0, ends with a barrier.  Returns the most blocks
// of a sequence to wave 0.
template <int COLS>
__device__ inline int tree_scan(const TreeArgs& a, int64_t* sP, int64_t* sT) {
    int most = 0;
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x, G = a.Hq / a.Hkv;
        int64_t run = 0, run_t = 0;
        for (int n0 = 0; n0 < a.N; n0 += 64) {
            const int n = n0 + lane;
            int64_t t = 0, v = 0;
            if (n < a.N) {
                const TreeSeq s = tree_seq(a, n);
                const int b = tree_blocks<COLS>(s, G);
                t = tree_tiles(s);
                v = b * t;
                most = max(most, b);
            }
            const int64_t incl = wave_incl_scan64(v);
            if (n < a.N) sP[n + 1] = run + incl;
            run += __shfl((long long)incl, 63, 64);
            if (sT) {
                const int64_t incl_t = wave_incl_scan64(t);
                if (n < a.N) sT[n + 1] = run_t + incl_t;
                run_t += __shfl((long long)incl_t, 63, 64);
            }
        }
        if (lane == 0) {
            sP[0] = 0;
            if (sT) sT[0] = 0;
        }
        if (sT) {
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) most = max(most, __shfl_xor(most, off, 64));
        }
    }
    __syncthreads();
    return most;
}

// The sequence whose tiles hold position p: Hkv * P[n] <= p < Hkv * P[n + 1].
__device__ inline int tree_find(const int64_t* P, int N, int Hkv, int64_t p) {
    int lo = 0, hi = N;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (Hkv * P[mid] <= p) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Position p's unit: its column block and kv head, its first position and its tiles.
struct TreeUnit {
    int n, kvh, cb, tiles;
    int64_t begin;
};

__device__ inline TreeUnit tree_unit(const TreeArgs& a, const int64_t* P, int n, int tiles, int64_t p) {
    TreeUnit u;
    u.n = n;
    u.tiles = tiles;
    const int64_t base = a.Hkv * P[n], per_head = P[n + 1] - P[n];
    u.kvh = (int)div_floor(p - base, per_head);
    const int64_t head = base + u.kvh * per_head;
    u.cb = (int)div_floor(p - head, tiles);
    u.begin = head + (int64_t)u.cb * tiles;
    return u;
}

}  // namespace llkv
