// Attention for trees of drafted tokens over the paged cache, and the decode
// step that adds its attention weights to each key's total (gfx950).  The
// schedule is in tree_attn.h.
//
// Bodies.  FewCols (fp32): a page of 16 keys at a time, K and V straight
// into the operand registers of the matrix instructions in the decode's layouts
// (decode_mfma.h), NCT tiles of 16 columns against each.  The four waves of a
// work-group take the four pages of a tile and join their softmax states
// through LDS at the end of a segment.  ManyCols (16-bit pools): tiles of K and V
// staged in a ring in LDS by direct loads, each wave with its own 16 or 32
// columns over all keys, as the prefill.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "lds_dma.h"
#include "tree_attn.h"

namespace llkv {
namespace {

__device__ inline bool finite_bits(uint32_t w, bool f16) {   // both halves of a pair of 16-bit values
    const uint32_t e = f16 ? 0x7C00u : 0x7F80u;
    return (w & e) != e && ((w >> 16) & e) != e;
}

// Bits j0 .. j0 + 31 of a row's mask; bits below 0 (the context) are set, those
// beyond the row's words are not.  (Without branches: a chain of conditions
// around each score compiled to a select that kept the score of a masked key.)
__device__ inline uint32_t tree_bits(const int* row, int words, int j0) {
    const int w0 = j0 >> 5, w1 = w0 + 1;
    const uint32_t a = (uint32_t)row[min(max(w0, 0), words - 1)], b = (uint32_t)row[min(max(w1, 0), words - 1)];
    const uint32_t lo = w0 < 0 ? ~0u : (w0 < words ? a : 0u), hi = w1 < 0 ? ~0u : (w1 < words ? b : 0u);
    return (uint32_t)(((uint64_t)hi << 32 | lo) >> (j0 & 31));
}

// Whether any thread of the work-group found a value of V in the tree that is not
// finite.
__device__ inline bool odd_segment(int& flag, bool odd) {
    if (threadIdx.x == 0) flag = 0;
    lds_barrier();
    if (odd) flag = 1;
    lds_barrier();
    const bool any = flag != 0;
    lds_barrier();   // before the next segment clears it
    return any;
}

// A segment's columns with plain arithmetic, one wave per column, keys that a
// column does not see left out: the answer where V has values that are not
// finite among the tree's nodes.
template <typename T, int D>
__device__ void slow_columns(const TreeArgs& a, const TreeSeg& sg, int kcols) {
    const int lane = threadIdx.x & 63, G = a.Hq / a.Hkv;
    const int64_t row_elems = (int64_t)a.Hkv * D;
    const int* bt = a.bt + (int64_t)sg.n * a.max_blocks;
    constexpr int MD = (D + 63) / 64;
    const int stop = min(sg.t1 * kTreeTile, sg.s.L);
    for (int cc = threadIdx.x >> 6; cc < kcols; cc += blockDim.x >> 6) {
        const int col = sg.c0 + cc;
        if (col >= sg.cols) break;
        const int node = col / G, hq = sg.kvh * G + (col - node * G);
        const int64_t row = sg.s.q0 + node;
        const T* q = reinterpret_cast<const T*>(a.q) + (row * a.Hq + hq) * D;
        float m = kNegBig, l = 0.0f, acc[MD];
#pragma unroll
        for (int i = 0; i < MD; ++i) acc[i] = 0.0f;
        for (int t0 = sg.t0 * kTreeTile; t0 < stop; t0 += 64) {
            const int t = t0 + lane;
            const bool seen = t < stop && (tree_bits(a.mask + row * a.words, a.words, t - sg.s.hist) & 1u) != 0;
            const int64_t at = ((int64_t)max(bt[min(t, stop - 1) / kPage], 0) * kPage + t % kPage) * row_elems + sg.kvh * D;
            float x = -INFINITY;
            if (seen) {
                float d0 = 0.0f, d1 = 0.0f, d2 = 0.0f, d3 = 0.0f;
#pragma unroll 1
                for (int d = 0; d < D; d += 4) {
                    const T* k = reinterpret_cast<const T*>(a.k) + at + d;
                    d0 = fmaf(Elem<T>::to_f32(q[d]), Elem<T>::to_f32(k[0]), d0);
                    d1 = fmaf(Elem<T>::to_f32(q[d + 1]), Elem<T>::to_f32(k[1]), d1);
                    d2 = fmaf(Elem<T>::to_f32(q[d + 2]), Elem<T>::to_f32(k[2]), d2);
                    d3 = fmaf(Elem<T>::to_f32(q[d + 3]), Elem<T>::to_f32(k[3]), d3);
                }
                x = ((d0 + d1) + (d2 + d3)) * a.scale_log2;
            }
            const float mx = fmaxf(m, wave_max(x)), corr = fast_exp2(m - mx);
            const float p = seen ? fast_exp2(x - mx) : 0.0f;
            l = l * corr + wave_sum(p);
            m = mx;
#pragma unroll
            for (int i = 0; i < MD; ++i) acc[i] *= corr;
            uint64_t left = __builtin_amdgcn_ballot_w64(seen);
            while (left != 0) {
                const int j = __builtin_ctzll(left);
                left &= left - 1;
                const float pj = __shfl(p, j, 64);
                const int64_t vj = __shfl((long long)at, j, 64);
#pragma unroll
                for (int i = 0; i < MD; ++i)
                    if (lane + 64 * i < D)
                        acc[i] = fmaf(pj, Elem<T>::to_f32(reinterpret_cast<const T*>(a.v)[vj + lane + 64 * i]), acc[i]);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t part = (int64_t)sg.slot * kcols + cc;
#pragma unroll
        for (int i = 0; i < MD; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) break;
            if (sg.direct) reinterpret_cast<T*>(a.out)[(row * a.Hq + hq) * D + d] = Elem<T>::from_f32(acc[i] * inv);
            else a.part_o[part * D + d] = acc[i] * inv;
        }
        if (lane == 0 && !sg.direct) a.part_lse[part] = l == 0.0f ? -INFINITY : m + fast_log2(l);
    }
}

template <int D_, int NCT_, bool MASS>
struct FewCols {
    using T = float;
    static constexpr int D = D_, NCT = NCT_, W = 4;
    static constexpr int kCols = 16 * NCT, kThreads = 64 * W;
    static constexpr bool kMass = MASS, kTeams = false, kStreams = false;
    using Ops = ScoreOps<T, D>;
    static constexpr int VH = (D + 63) / 64, DT = 4 * VH, MD = VH;
    // Resident waves per SIMD that the registers are held to (the loads in flight are what
    // bounds a few columns).
    static constexpr int kWavesPerEU = NCT == 1 ? (D == 64 ? 4 : (D == 256 ? 1 : (D == 128 && !MASS ? 2 : 3))) : (D == 64 ? 3 : 2);

    struct Smem {
        float acc[W][16][D];
        float ml[W][16][2];   // (max, sum)
        int odd;
    };

    __device__ static void run(const TreeArgs& a, Smem& sm, const TreeSeg& sg) {
        const int lane = threadIdx.x & 63;
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int g = lane >> 4, c = lane & 15;
        const int G = a.Hq / a.Hkv;
        const int64_t row_elems = (int64_t)a.Hkv * D;
        const int L = sg.s.L, hist = sg.s.hist;
        const T* kbase = reinterpret_cast<const T*>(a.k) + (int64_t)sg.kvh * D;
        const T* vbase = reinterpret_cast<const T*>(a.v) + (int64_t)sg.kvh * D;
        const int* bt = a.bt + (int64_t)sg.n * a.max_blocks;

        float q[NCT][Ops::NQ];
        const int* mrow[NCT];
        mf32x4 o[NCT][DT];
        float m[NCT], l[NCT];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
            const int col = sg.c0 + 16 * ct + c;
            const bool valid = col < sg.cols;
            const int node = valid ? col / G : 0;
            const int64_t row = sg.s.q0 + node;
            const T* qrow = reinterpret_cast<const T*>(a.q) + (row * a.Hq + sg.kvh * G + (valid ? col - node * G : 0)) * D;
#pragma unroll
            for (int cc = 0; cc < D / 16; ++cc) {
                const float4 x = *reinterpret_cast<const float4*>(qrow + 16 * cc + 4 * g);
                const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) q[ct][4 * cc + e] = valid ? f[e] * a.scale_log2 : 0.0f;
            }
            mrow[ct] = MASS ? nullptr : a.mask + row * a.words;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[ct][dt] = mf32x4{0.f, 0.f, 0.f, 0.f};
            m[ct] = kNegBig;
            l[ct] = 0.0f;
        }

        const int npages = (L + kPage - 1) / kPage;
        const int count = sg.t1 - sg.t0;   // this wave's pages: 4 (t0 + j) + w, j < count
        int tbl = 0;
        bool odd = false;
        for (int j = 0; j < count; ++j) {
            if ((j & 63) == 0) {   // the next 64 page ids, one per lane
                const int pg = W * (sg.t0 + j + lane) + w;
                tbl = pg < npages ? bt[pg] : 0;
            }
            const int pg = W * (sg.t0 + j) + w;
            if (pg >= npages) break;
            const int64_t phys = max(__builtin_amdgcn_readlane(tbl, j & 63), 0);

            float4 kr[Ops::NK];
            Ops::template load_k<false>(kbase + (phys * kPage + c) * row_elems, g, kr);
            float4 vr[VH][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T* vp = vbase + (phys * kPage + 4 * g + i) * row_elems + 4 * c;
#pragma unroll
                for (int h = 0; h < VH; ++h) {
                    if (D % 64 != 0 && 64 * h + 4 * c >= D) vr[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);   // past the last dim
                    else vr[h][i] = Ops::template load_v4<false>(vp + 64 * h);
                }
            }

            // Keys that some columns do not see: the last page's rest, where V may hold
            // anything and is taken as zero, and the tree's own.  A value there that is not
            // finite must reach the columns that see it and no other, which a product with
            // weights of zero does not give: such a segment is computed again (slow_columns).
            const int p0 = pg * kPage;
            const bool whole = p0 + kPage <= min(hist, L);   // uniform
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool beyond = p0 + 4 * g + i >= L;
                    const bool tree = !MASS && p0 + 4 * g + i >= hist && !beyond;
#pragma unroll
                    for (int h = 0; h < VH; ++h) {
                        odd |= tree && !(isfinite(vr[h][i].x) && isfinite(vr[h][i].y) && isfinite(vr[h][i].z) &&
                                         isfinite(vr[h][i].w));
                        if (beyond) vr[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
            }

#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
                const mf32x4 sc = Ops::scores(kr, q[ct], a.scale_log2);
                float x[4] = {sc[0], sc[1], sc[2], sc[3]};
                if (!whole) {
                    const int p4 = p0 + 4 * g;
                    uint32_t seen = ~0u;   // bit i: the lane's key i
                    if constexpr (!MASS) seen = tree_bits(mrow[ct], a.words, p4 - hist);
                    seen &= L >= p4 + 4 ? ~0u : (1u << max(L - p4, 0)) - 1u;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = seen >> i & 1u ? x[i] : -INFINITY;
                }
                if constexpr (MASS) {
                    const int col = sg.c0 + 16 * ct + c;
                    if (col < sg.cols)
                        *reinterpret_cast<float4*>(a.scores + ((int64_t)(sg.n * a.Hkv + sg.kvh) * G + col) * a.score_stride +
                                                   p0 + 4 * g) = make_float4(x[0], x[1], x[2], x[3]);
                }
                // The running maximum moves only when a column's page exceeds it by more than
                // 8, so most pages need no exchange between lanes.
                const float mt = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                if (__builtin_amdgcn_ballot_w64(mt > m[ct] + 8.0f) != 0) {
                    float mm = fmaxf(mt, __shfl_xor(mt, 16, 64));
                    mm = fmaxf(mm, __shfl_xor(mm, 32, 64));
                    const float mnew = fmaxf(m[ct], mm);
                    const float corr = fast_exp2(m[ct] - mnew);
                    m[ct] = mnew;
                    l[ct] *= corr;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[ct][dt] *= corr;
                }
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[i] = fast_exp2(x[i] - m[ct]);
                    l[ct] += p[i];
                }
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[ct][4 * h + 0] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[h][i].x, p[i], o[ct][4 * h + 0], 0, 0, 0);
                        o[ct][4 * h + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[h][i].y, p[i], o[ct][4 * h + 1], 0, 0, 0);
                        o[ct][4 * h + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[h][i].z, p[i], o[ct][4 * h + 2], 0, 0, 0);
                        o[ct][4 * h + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[h][i].w, p[i], o[ct][4 * h + 3], 0, 0, 0);
                    }
            }
        }

        if constexpr (!MASS) {
            if (odd_segment(sm.odd, odd)) {
                slow_columns<T, D>(a, sg, kCols);
                return;
            }
        }
        // Join the waves' states, 16 columns at a time.
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
            float ls = l[ct];
            ls += __shfl_xor(ls, 16, 64);
            ls += __shfl_xor(ls, 32, 64);
            if (ct > 0) lds_barrier();   // the previous columns have been read
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (D % 64 == 0 || 64 * h + 16 * g + 4 * i < D)
                        *reinterpret_cast<float4*>(&sm.acc[w][c][64 * h + 16 * g + 4 * i]) =
                            make_float4(o[ct][4 * h][i], o[ct][4 * h + 1][i], o[ct][4 * h + 2][i], o[ct][4 * h + 3][i]);
            if (g == 0) {
                sm.ml[w][c][0] = m[ct];
                sm.ml[w][c][1] = ls;
            }
            lds_barrier();
            for (int cc = w; cc < 16; cc += W) {
                const int col = sg.c0 + 16 * ct + cc;
                if (col >= sg.cols) break;
                float M = sm.ml[0][cc][0];
#pragma unroll
                for (int ww = 1; ww < W; ++ww) M = fmaxf(M, sm.ml[ww][cc][0]);
                float f[W], sum = 0.0f;
#pragma unroll
                for (int ww = 0; ww < W; ++ww) {
                    f[ww] = fast_exp2(sm.ml[ww][cc][0] - M);
                    sum = fmaf(f[ww], sm.ml[ww][cc][1], sum);
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // 0: a column that sees no key
                const int node = col / G;
                const int hq = sg.kvh * G + (col - node * G);
                T* out = reinterpret_cast<T*>(a.out) + ((int64_t)(sg.s.q0 + node) * a.Hq + hq) * D;
                float* po = a.part_o + ((int64_t)sg.slot * kCols + 16 * ct + cc) * D;
#pragma unroll
                for (int i = 0; i < MD; ++i) {
                    const int d = lane + 64 * i;
                    if (D % 64 != 0 && d >= D) break;
                    float ov = 0.0f;
#pragma unroll
                    for (int ww = 0; ww < W; ++ww) ov = fmaf(f[ww], sm.acc[ww][cc][d], ov);
                    ov *= inv;
                    if (sg.direct) out[d] = Elem<T>::from_f32(ov);
                    else po[d] = ov;
                }
                if (lane == 0) {
                    const float lse = sum == 0.0f ? -INFINITY : M + fast_log2(sum);
                    if (!sg.direct) a.part_lse[(int64_t)sg.slot * kCols + 16 * ct + cc] = lse;
                    else if constexpr (MASS) a.lse[(int64_t)sg.n * a.Hq + hq] = lse;
                }
            }
        }
        lds_barrier();
    }
};

// V_MFMA_F32_16X16X32 of a 16-bit type.
template <typename T>
__device__ inline mf32x4 mma32(const mu32x4& x, const mu32x4& y, mf32x4 c) {
    if constexpr (Elem<T>::kDtype == LLKV_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mf16x8, x), __builtin_bit_cast(mf16x8, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mbf16x8, x), __builtin_bit_cast(mbf16x8, y), c, 0, 0, 0);
}

template <typename T>
__device__ inline uint32_t pack_pair(float x, float y) {
    if constexpr (Elem<T>::kDtype == LLKV_DTYPE_F16) return pack_h2(x, y);
    else return pack_b2(x, y);
}

// K and V in LDS tiles of BN keys.  Rows are unpadded (direct loads write 1 KB
// blocks) and their 16-byte chunks XOR-ed with the row, so that the rows that an
// operand read takes together lie in different banks.  The key order of the K
// operand's rows is permuted (row 8 (c / 4) + 4 h + c % 4 of a 32-key half for
// lane c of tile h), so that a lane's scores are the 8 consecutive keys that it
// feeds to the second product; V's operand comes by transposing LDS reads.
// Instruction order of the S^T product: the K operand reads (READS per k-step) of
// the first two k-steps, then each k-step's products followed by the reads of the
// k-step after next.
template <int KS, int READS, int PRODUCTS, int I = 0>
__device__ inline void score_schedule() {
    if constexpr (I == 0) __builtin_amdgcn_sched_group_barrier(0x100, KS > 1 ? 2 * READS : READS, 0);
    if constexpr (I < KS) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
        if constexpr (I + 2 < KS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        score_schedule<KS, READS, PRODUCTS, I + 1>();
    }
}

template <typename TT, int D_, int NCW, int WV, int RING, bool MASS = false>
struct ManyCols {
    using T = TT;
    static constexpr int D = D_, W = WV, R = RING;
    static constexpr int kCols = 16 * NCW * W, kThreads = 64 * W;
    static constexpr int BN = D == 256 ? 32 : 64;
    static constexpr int KT = BN / 16, SS = BN / 32;   // key tiles, key halves of the second product
    static constexpr int KS = D / 32, DT = D / 16;
    static constexpr int CPR = D / 8;                  // 16-byte chunks per row
    // Four waves load a quarter of the rows of K and of V each; of eight, four load K's and
    // four V's, so that a part is whole 1 KB blocks.
    static constexpr int RPW = BN / 4;
    static constexpr int BPW = RPW * D * 2 / 1024;
    static constexpr int kLoads = (W == 4 ? 2 : 1) * BPW;   // of a wave per tile
    static_assert((W == 4 || W == 8) && RPW * D * 2 % 1024 == 0 && kPage % RPW == 0, "tile parts");
    static constexpr int kWavesPerEU = 2;
    // Eight waves, two per SIMD: the second four run half a tile behind (kPair), so that the
    // exponentials of the one meet the products of the other (32/8/128 fp16, 32 x 2816 keys,
    // 64 nodes: 120 us all at once, 110 so).
    static constexpr bool kPair = W == 8 && !MASS;
    static constexpr int kAhead = kPair ? R - 2 : R - 1;   // tiles loaded ahead (V of tile j - 1 is still read)
    static constexpr bool kMass = MASS, kTeams = !MASS, kStreams = true;
    static constexpr uint32_t kOnes = Elem<T>::kDtype == LLKV_DTYPE_F16 ? 0x3C003C00u : 0x3F803F80u;
    static constexpr bool kF16 = Elem<T>::kDtype == LLKV_DTYPE_F16;

    struct Smem {
        alignas(16) uint16_t k[R][BN * D];
        alignas(16) uint16_t v[R][BN * D];
        int odd;
    };

    // Place of chunk ch of row r, and the chunk at a place: XOR with row bits, or a rotation by
    // them where a row's chunks are no power of two.  K: bits 0, 1, 3, 4 (the 16 rows that an
    // operand read takes together differ there).  V: 8 rows of 32 lanes, which read pairs of
    // chunks: bits 0, 1, 3 (at head_dim 64, where two rows share the banks, 1 and 3) above the
    // pair (with K's bits, two rows' pairs met in the same banks).
    static constexpr bool kXor = (CPR & (CPR - 1)) == 0;
    template <bool V>
    __device__ static int bits(int r) {
        if (kXor && V) return CPR == 8 ? (r & 2) | ((r & 8) >> 1) : ((r & 3) << 1) | (r & 8);
        return ((r & 3) | ((r >> 1) & 0xC)) & (kXor ? CPR - 1 : ~0);
    }
    template <bool V>
    __device__ static int place(int r, int ch) { return kXor ? ch ^ bits<V>(r) : (ch + bits<V>(r)) % CPR; }
    template <bool V>
    __device__ static int chunk(int r, int pl) { return kXor ? pl ^ bits<V>(r) : (pl + 16 * CPR - bits<V>(r)) % CPR; }
    template <bool V>
    __device__ static int at(int row, int d) { return row * D + (place<V>(row, d >> 3) << 3 | (d & 7)); }

    __device__ static void run(const TreeArgs& a, Smem& sm, const TreeSeg& sg) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int g = lane >> 4, c = lane & 15;
        const int G = a.Hq / a.Hkv;
        const int L = sg.s.L, hist = sg.s.hist;
        const uint32_t row_bytes = (uint32_t)(a.Hkv * D * sizeof(T));
        const char* kp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.k) + (int64_t)sg.kvh * D);
        const char* vp = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.v) + (int64_t)sg.kvh * D);
        const int* bt = a.bt + (int64_t)sg.n * a.max_blocks;
        const int last_page = L > 0 ? (L - 1) / kPage : 0;
        // keys [begin, stop) in tiles of BN
        const int begin = sg.t0 * kTreeTile;
        const int tiles = (min(sg.t1 * kTreeTile, L) - begin + BN - 1) / BN;   // 0 or less: no key

        // The wave's rows of a tile, a page or a part of one: 16-byte units u of them, 64 per block.
        constexpr uint32_t kTileBytes = BN * D * 2;
        const int part = RPW * (w & 3);   // first row
        const bool loads_v = W == 8 && w >= 4;
        uint32_t off[BPW], off_v[BPW], to_k[BPW], to_v[BPW];   // (off: V's in the waves that load only V)
#pragma unroll
        for (int i = 0; i < BPW; ++i) {
            const int u = 64 * i + lane, r = part + u / CPR;
            const uint32_t row = (uint32_t)(r % kPage) * row_bytes;
            off_v[i] = row + (uint32_t)chunk<true>(r, u % CPR) * 16u;
            off[i] = loads_v ? off_v[i] : row + (uint32_t)chunk<false>(r, u % CPR) * 16u;
            to_k[i] = lds_addr((loads_v ? sm.v[0] : sm.k[0]) + part * D + 512 * i);
            to_v[i] = lds_addr(sm.v[0] + part * D + 512 * i);
        }
        const char* const kb = loads_v ? vp : kp;
        int tbl = 0;   // page ids of the wave's next 64 tiles, one per lane
        auto load_tile = [&](int j) {
            if ((j & 63) == 0) {
                tbl = bt[min((begin + (j + lane) * BN + part) / kPage, last_page)];
                // Waited for here: at its use, where the compiler cannot tell whether it is still
                // on the way, the wait would stand in every tile and empty the ring.
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            }
            const int phys = max(__builtin_amdgcn_readlane(tbl, j & 63), 0);
            const uint64_t base = (uint64_t)(uint32_t)phys * row_bytes * kPage;
            const uint32_t to = (uint32_t)(j % R) * kTileBytes;
            if (sg.stream) {   // (uniform)
#pragma unroll
                for (int i = 0; i < BPW; ++i) {
                    dma16_s<true>(kb + base, off[i], to_k[i] + to);
                    if constexpr (W == 4) dma16_s<true>(vp + base, off_v[i], to_v[i] + to);
                }
            } else {
#pragma unroll
                for (int i = 0; i < BPW; ++i) {
                    dma16_s(kb + base, off[i], to_k[i] + to);
                    if constexpr (W == 4) dma16_s(vp + base, off_v[i], to_v[i] + to);
                }
            }
        };
        // Where the lane's operands lie in a tile (halves): K row 8 (c / 4) + c % 4 for each
        // k-step, V row 8 g + c / 4 for each output tile.
        int koff[KS], voff[DT];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) koff[ks] = at<false>(8 * (c >> 2) + (c & 3), ks * 32 + g * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) voff[dt] = at<true>(8 * g + (c >> 2), dt * 16 + 4 * (c & 3));

        // Columns; a negative scale goes into Q's signs, so that the largest score stays the
        // largest when scaled.
        const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);
        const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
        mu32x4 q[NCW][KS];
        const int* mrow[NCW];
        // Row sums: of the rounded weights, as O's products take them, by a tile of ones; of
        // kept weights, which the log-sum-exp normalises in 32 bits, of the weights themselves.
        mf32x4 o[NCW][DT], osum[NCW];
        float m[NCW], l[NCW];
#pragma unroll
        for (int nt = 0; nt < NCW; ++nt) {
            const int col = sg.c0 + (w * NCW + nt) * 16 + c;
            const bool valid = col < sg.cols;
            const int node = valid ? col / G : 0;
            const int64_t row = sg.s.q0 + node;
            const T* qrow = reinterpret_cast<const T*>(a.q) + (row * a.Hq + sg.kvh * G + (valid ? col - node * G : 0)) * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const mu32x4 x = *reinterpret_cast<const mu32x4*>(qrow + 32 * ks + 8 * g);
                q[nt][ks] = valid ? x ^ flip : mu32x4{0u, 0u, 0u, 0u};
            }
            mrow[nt] = MASS ? nullptr : a.mask + row * a.words;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[nt][dt] = mf32x4{0.f, 0.f, 0.f, 0.f};
            osum[nt] = mf32x4{0.f, 0.f, 0.f, 0.f};
            m[nt] = kNegBig;
            l[nt] = 0.0f;
        }
        __builtin_amdgcn_sched_barrier(0);   // Q before the tiles (loads return in order)
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (j < tiles) load_tile(j);
        const mu32x4 ones = {kOnes, kOnes, kOnes, kOnes};
        bool odd = false;
        const bool idle = sg.c0 + w * NCW * 16 >= sg.cols;   // the wave has no column: it loads and waits only

        mu32x4 p[SS][NCW];   // the weights of a tile, packed
        // S^T = K Q^T of tile j, masked, the running maximum, and the weights.
        auto score = [&](int j, bool whole) {
            const uint16_t* const kt_lds = sm.k[j % R];
            const int key0 = begin + j * BN;
            __builtin_amdgcn_sched_barrier(0);   // the next tile's loads are issued first
            if constexpr (D >= 128) __builtin_amdgcn_s_setprio(1);
            // the K operands of k-step ks + 1 read behind the products of ks
            mf32x4 s[KT][NCW];
            auto k_operand = [&](int kt, int ks) {
                return *reinterpret_cast<const mu32x4*>(kt_lds + koff[ks] + (32 * (kt >> 1) + 4 * (kt & 1)) * D);
            };
            mu32x4 ka[2][KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) ka[0][kt] = k_operand(kt, 0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 1 < KS) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) ka[(ks + 1) & 1][kt] = k_operand(kt, ks + 1);
                }
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NCW; ++nt)
                        s[kt][nt] = mma32<T>(ka[ks & 1][kt], q[nt][ks], ks == 0 ? mf32x4{0.f, 0.f, 0.f, 0.f} : s[kt][nt]);
            }
            score_schedule<KS, KT, KT * NCW>();
            if constexpr (D >= 128) {
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            float mx[NCW];
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NCW; ++nt) {
                if (!whole) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        const int k4 = key0 + 32 * (kt >> 1) + 8 * g + 4 * (kt & 1);
                        uint32_t seen = ~0u;
                        if constexpr (!MASS) seen = tree_bits(mrow[nt], a.words, k4 - hist);
                        seen &= L >= k4 + 4 ? ~0u : (1u << max(L - k4, 0)) - 1u;
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kt][nt][i] = seen >> i & 1u ? s[kt][nt][i] : -INFINITY;
                    }
                }
                if constexpr (MASS) {
                    const int col = sg.c0 + (w * NCW + nt) * 16 + c;
                    float* sc = a.scores + ((int64_t)(sg.n * a.Hkv + sg.kvh) * G + col) * a.score_stride + key0 + 8 * g;
                    if (col < sg.cols) {
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
                            *reinterpret_cast<mf32x4*>(sc + 32 * (kt >> 1) + 4 * (kt & 1)) = s[kt][nt] * scale;
                    }
                }
                float v = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v = fmaxf(v, s[kt][nt][i]);
                mx[nt] = v * scale;
                grow |= mx[nt] > m[nt] + 8.0f;
            }
            // The running maximum moves only when a lane's keys exceed it by more than 8.
            if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
                for (int nt = 0; nt < NCW; ++nt) {
                    float v = fmaxf(mx[nt], __shfl_xor(mx[nt], 16, 64));
                    v = fmaxf(v, __shfl_xor(v, 32, 64));
                    const float mnew = fmaxf(m[nt], v);
                    const float corr = fast_exp2(m[nt] - mnew);
                    m[nt] = mnew;
                    if constexpr (MASS) l[nt] *= corr;
                    else osum[nt] *= corr;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= corr;
                }
            }
            // P in the pool's type (half a step of each weight, as the prefill)
#pragma unroll
            for (int ss = 0; ss < SS; ++ss)
#pragma unroll
                for (int nt = 0; nt < NCW; ++nt) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = fast_exp2(fmaf(s[2 * ss + (i >> 2)][nt][i & 3], scale, -m[nt]));
                        if constexpr (MASS) l[nt] += e[i];
                    }
                    p[ss][nt] = mu32x4{pack_pair<T>(e[0], e[1]), pack_pair<T>(e[2], e[3]), pack_pair<T>(e[4], e[5]),
                                       pack_pair<T>(e[6], e[7])};
                }
        };
        // O^T += V^T P^T of tile j, and the row sums by the same rounded weights.
        auto product = [&](int j) {
            const uint16_t* const vt_lds = sm.v[j % R];
            // V^T operand of output dims 16 dt .. + 15 and the 32-key half ss.
            auto v_operand = [&](int dt, int ss) {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                const uint16_t* at0 = vt_lds + voff[dt] + 32 * ss * D;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at0);
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at0 + 4 * D));
                const mu32x2 l2 = __builtin_bit_cast(mu32x2, lo), h2 = __builtin_bit_cast(mu32x2, hi);
                return mu32x4{l2.x, l2.y, h2.x, h2.y};
            };
            mu32x4 va[DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) va[dt] = v_operand(dt, 0);
#pragma unroll
            for (int ss = 0; ss < SS; ++ss) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                    for (int nt = 0; nt < NCW; ++nt) o[nt][dt] = mma32<T>(va[dt], p[ss][nt], o[nt][dt]);
                    if (ss + 1 < SS) {
                        va[dt] = v_operand(dt, ss + 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if constexpr (!MASS) {
#pragma unroll
                    for (int nt = 0; nt < NCW; ++nt) osum[nt] = mma32<T>(ones, p[ss][nt], osum[nt]);
                }
            }
        };
        const bool behind = kPair && w >= 4;   // (uniform over the wave)

        for (int j = 0; j < tiles; ++j) {
            // This wave's part of tile j is in LDS: all loads but those of the tiles after it.
            const int after = tiles - 1 - j;
            constexpr int kAll = vmcnt_imm(kLoads * (kAhead - 1)), kLess = vmcnt_imm(kAhead > 1 ? kLoads * (kAhead - 2) : 0);
            if (after >= kAhead - 1) __builtin_amdgcn_s_waitcnt(kAll);
            else if (after == kAhead - 2) __builtin_amdgcn_s_waitcnt(kLess);
            else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            lds_barrier();   // everyone's; and the buffer of the tile loaded next has been read
            if (j + kAhead < tiles) load_tile(j + kAhead);
            const int key0 = begin + j * BN;
            const bool whole = key0 + BN <= min(hist, L);   // uniform
            if (!whole) {
                // V beyond the last key may hold anything: zero.  Values in the tree that are not
                // finite: the segment is computed again.
                for (int i = tid; i < BN * CPR; i += kThreads) {
                    const int r = i / CPR;
                    mu32x4& x = *reinterpret_cast<mu32x4*>(sm.v[j % R] + i * 8);
                    if (key0 + r >= L) x = mu32x4{0u, 0u, 0u, 0u};
                    else if (!MASS && key0 + r >= hist)
                        odd |= !(finite_bits(x.x, kF16) && finite_bits(x.y, kF16) && finite_bits(x.z, kF16) && finite_bits(x.w, kF16));
                }
                lds_barrier();
            }
            if (idle) continue;   // (uniform over the wave)
            if (behind && j > 0) product(j - 1);
            score(j, whole);
            if (!behind) product(j);
        }
        if (behind && !idle && tiles > 0) product(tiles - 1);
        if constexpr (MASS) {
            lds_barrier();   // the last tile has been read: the next segment loads into the ring
        } else if (odd_segment(sm.odd, odd)) {
            slow_columns<T, D>(a, sg, kCols);
            return;
        }
#pragma unroll
        for (int nt = 0; nt < NCW; ++nt) {
            const int cc = (w * NCW + nt) * 16 + c, col = sg.c0 + cc;
            float sum = osum[nt][0];
            if constexpr (MASS) {
                sum = l[nt] + __shfl_xor(l[nt], 16, 64);
                sum += __shfl_xor(sum, 32, 64);
            }
            if (col >= sg.cols) continue;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int node = col / G;
            T* out = reinterpret_cast<T*>(a.out) + ((int64_t)(sg.s.q0 + node) * a.Hq + sg.kvh * G + (col - node * G)) * D;
            const int64_t part = (int64_t)sg.slot * kCols + cc;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const mf32x4 x = o[nt][dt] * inv;
                const int d = dt * 16 + 4 * g;
                if (sg.direct)
                    *reinterpret_cast<mu32x2*>(out + d) = mu32x2{pack_pair<T>(x[0], x[1]), pack_pair<T>(x[2], x[3])};
                else
                    *reinterpret_cast<mf32x4*>(a.part_o + part * D + d) = x;
            }
            if (g == 0) {
                const float lse = sum == 0.0f ? -INFINITY : m[nt] + fast_log2(sum);
                if (!sg.direct) a.part_lse[part] = lse;
                else if constexpr (MASS) a.lse[(int64_t)sg.n * a.Hq + sg.kvh * G + (col - node * G)] = lse;
            }
        }
    }
};

// Log-sum-exp join of a cut unit's parts.  LR lanes hold a row, 16 bytes each, and a
// work-group as many rows as it has lanes for: of a column's parts kBatch per lane
// and as many lane groups as that takes (parts_groups), so that most joins are one
// round trip; the rest are other columns (join_width).  (A wave per column with its
// parts one after the other: 54 us for 8 units of 64 columns of 64 parts, 17 us the
// kernel that wrote them.)
constexpr int kBatch = 4;

// Lanes of a row.
constexpr int join_lanes(int D) { return D <= 64 ? 16 : (D <= 128 ? 32 : 64); }

template <int LR>
__device__ inline int part_groups(int parts) {
    int sp = 1;
    while (sp * kBatch < parts && sp < 256 / LR) sp *= 2;
    return sp;
}

// Columns at once.
template <int LR>
__device__ inline int join_width(int parts) { return 256 / LR / part_groups<LR>(parts); }

constexpr int kXcds = 8;
constexpr int64_t kTreeStreamBytes = 192ll << 20;

// Whether page pg of sequence n is another sequence's too: a prefix lies at the same
// place of each table, so one entry per sequence tells.  The same in every wave.
__device__ inline bool shared_page(const TreeArgs& a, int n, int pg) {
    pg = min(pg, a.max_blocks - 1);
    const int id = a.bt[(int64_t)n * a.max_blocks + pg];
    bool same = false;
    for (int j = threadIdx.x & 63; j < a.N; j += 64) {
        const int l = a.lens[j];
        same |= (a.bt[(int64_t)j * a.max_blocks + pg] == id) & (l > pg * kPage) & (j != n);
    }
    return __builtin_amdgcn_ballot_w64(same) != 0;
}

template <class B>
__global__ __launch_bounds__(B::kThreads) __attribute__((amdgpu_waves_per_eu(B::kWavesPerEU))) void tree_kernel(TreeArgs a) {
    __shared__ typename B::Smem sm;
    __shared__ int64_t sP[kTreeSeqs + 1];
    __shared__ int64_t sT[B::kTeams ? kTreeSeqs + 1 : 1];
    __shared__ int s_most;
    const int most = tree_scan<B::kCols>(a, sP, B::kTeams ? sT : nullptr);
    int team = 1;
    const int64_t* S = sP;
    if constexpr (B::kTeams) {
        if (threadIdx.x == 0) s_most = most;
        lds_barrier();
        const int b = s_most;
        // teams where at most a fifth of the members' work is a block that a sequence does not have
        if (b > 1 && b <= a.nwg && 4 * b * sT[a.N] <= 5 * sP[a.N]) {
            team = b;
            S = sT;
        }
    }
    if (B::kMass && blockIdx.x == 0)
        for (int i = threadIdx.x; i <= a.N; i += blockDim.x) a.plan[i] = sP[i];
    const int64_t T = a.Hkv * S[a.N];
    const int shares = (int)min(T, (int64_t)(a.nwg / team)), used = shares * team;
    if ((int)blockIdx.x >= used) {
        if (!B::kMass && threadIdx.x == 0) a.rounds[blockIdx.x] = 0;
        return;
    }
    // Work-groups go to the 8 XCDs in turn: neighbours, which may read the same keys for
    // other columns, to one XCD's L2.
    const int xcd = blockIdx.x % kXcds;
    const int w = xcd * (used / kXcds) + min(xcd, used % kXcds) + blockIdx.x / kXcds;
    const int share = w / team, member = w - share * team;
    const int64_t r0 = share_begin(share, T, shares), r1 = share_begin(share + 1, T, shares);
    const int G = a.Hq / a.Hkv;
    // Beyond three quarters of the last-level cache K and V are streamed, where no other column
    // block and no other sequence (a cached prefix) reads them again; as in the plain decode.
    const int64_t tiles = a.Hkv * (B::kTeams ? sT : sP)[a.N];
    const bool big = B::kStreams && tiles * (kTreeTile * 2 * B::D * (int64_t)sizeof(typename B::T)) > kTreeStreamBytes;
    TreeCut cut = {};
    for (int64_t p = r0; p < r1;) {
        TreeSeg sg;
        sg.n = tree_find(S, a.N, a.Hkv, p);
        sg.s = tree_seq(a, sg.n);
        const TreeUnit u = tree_unit(a, S, sg.n, tree_tiles(sg.s), p);
        const int64_t end = u.begin + u.tiles, stop = end < r1 ? end : r1;
        sg.kvh = u.kvh;
        sg.cols = sg.s.P * G;
        sg.c0 = (u.cb + member) * B::kCols;
        sg.t0 = (int)(p - u.begin);
        sg.t1 = (int)(stop - u.begin);
        sg.direct = p == u.begin && stop == end;
        sg.slot = 2 * w + (p == r0 ? 0 : 1);
        sg.stream = false;
        if (big) sg.stream = sg.s.P * G <= B::kCols && !shared_page(a, sg.n, (sg.t0 + sg.t1) / 2 * (kTreeTile / kPage));
        if (sg.c0 < sg.cols) {   // (uniform; a team's member may have no block of this sequence)
            if (p == u.begin && stop < end)
                cut = TreeCut{sg.s.q0, sg.cols, sg.c0, sg.kvh, sg.slot, (int)(wg_of(end - 1, T, shares) - share) + 1, team};
            B::run(a, sm, sg);
        }
        p = stop;
    }
    if (!B::kMass && threadIdx.x == 0) {
        const int width = join_width<join_lanes(B::D)>(cut.parts);   // a power of two
        a.rounds[w] = cut.parts > 0 ? (min(B::kCols, cut.cols - cut.c0) + width - 1) >> (31 - __builtin_clz(width)) : 0;
        a.cuts[w] = cut;
    }
}

// Slot of part j of a cut unit that begins in work-group w.
__device__ inline int part_slot(int w, int first_slot, int step, int j) { return j == 0 ? first_slot : 2 * (w + j * step); }

struct JoinSmem {
    mf32x4 o[256];
    float ml[64][2];   // (max, sum) per row
};

// Columns c0 .. c0 + join_width - 1 (those below `here`); out_row(c): the output row.
template <typename T, int LR, class OutRow>
__device__ inline void join_columns(const TreeArgs& a, JoinSmem& sm, int cols, int w, const TreeCut& u, int c0, int here,
                                    OutRow out_row) {
    const int r = threadIdx.x / LR, l = threadIdx.x % LR;
    const int sp = part_groups<LR>(u.parts), sub = r % sp;
    const bool lane_on = 4 * l < a.D;
    const int c = c0 + r / sp;
    float M = -INFINITY, sum = 0.0f;
    mf32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (c < here) {
        for (int j0 = sub; j0 < u.parts; j0 += kBatch * sp) {
            float lv[kBatch];
            mf32x4 pv[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int j = j0 + b * sp;
                const bool ok = j < u.parts;
                const int64_t row = (int64_t)part_slot(w, u.slot, u.step, ok ? j : j0) * cols + c;
                lv[b] = ok ? a.part_lse[row] : -INFINITY;
                pv[b] = *reinterpret_cast<const mf32x4*>(a.part_o + row * a.D + (lane_on ? 4 * l : 0));
            }
            float mb = M;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) mb = fmaxf(mb, lv[b]);
            // (no key seen so far: weights of zero; a part that is no number stays one)
            const float base = mb == -INFINITY ? 0.0f : mb;
            const float sc = fast_exp2(M - base);
            sum *= sc;
            o *= sc;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const float f = fast_exp2(lv[b] - base);
                sum += f;
                o += f * pv[b];
            }
            M = mb;
        }
    }
    if (sp > 1) {   // uniform
        sm.o[threadIdx.x] = o;
        if (l == 0) {
            sm.ml[r][0] = M;
            sm.ml[r][1] = sum;
        }
        __syncthreads();
        if (sub == 0) {
            float top = M;
            for (int i = 1; i < sp; ++i) top = fmaxf(top, sm.ml[r + i][0]);
            const float base = top == -INFINITY ? 0.0f : top;
            float f = fast_exp2(M - base);
            sum *= f;
            o *= f;
            for (int i = 1; i < sp; ++i) {
                f = fast_exp2(sm.ml[r + i][0] - base);
                sum = fmaf(f, sm.ml[r + i][1], sum);
                o += f * sm.o[threadIdx.x + i * LR];
            }
        }
        __syncthreads();
    }
    if (sub == 0 && c < here && lane_on) {
        o *= sum == 0.0f ? 0.0f : 1.0f / sum;
        T* out = out_row(c) + 4 * l;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<mf32x4*>(out) = o;
        else *reinterpret_cast<mu32x2*>(out) = mu32x2{pack_pair<T>(o[0], o[1]), pack_pair<T>(o[2], o[3])};
    }
}

// The cut units' columns shared by the whole grid: every work-group sums up the
// rounds of join_columns that the units take and runs rounds blockIdx.x,
// + gridDim.x ..  (With work-groups tied to the units, a few long units were joined
// by a few work-groups.)
constexpr int kMostShares = 2048;   // work-groups of the first kernel

template <typename T, int LR>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int cols) {
    __shared__ JoinSmem sm;
    __shared__ int start[kMostShares + 1];   // rounds before unit w
    __shared__ int wave_total[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    constexpr int kPer = kMostShares / 256;
    int mine[kPer], sum = 0;   // of units kPer tid ..
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        mine[i] = kPer * tid + i < a.nwg ? a.rounds[kPer * tid + i] : 0;
        sum += mine[i];
    }
    const int incl = wave_incl_scan(sum);
    if (lane == 63) wave_total[wv] = incl;
    __syncthreads();
    int run = incl - sum;
    for (int i = 0; i < wv; ++i) run += wave_total[i];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        start[kPer * tid + i] = run;
        run += mine[i];
    }
    if (tid == 255) start[kMostShares] = run;
    __syncthreads();
    const int rounds = start[kMostShares], G = a.Hq / a.Hkv;
    for (int x = blockIdx.x; x < rounds; x += gridDim.x) {
        int lo = 0, hi = kMostShares;   // start[lo] <= x < start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= x) lo = mid;
            else hi = mid;
        }
        const int w = __builtin_amdgcn_readfirstlane(lo);
        const TreeCut u = a.cuts[w];
        join_columns<T, LR>(a, sm, cols, w, u, (x - start[w]) * join_width<LR>(u.parts), min(cols, u.cols - u.c0), [&](int c) {
            const int col = u.c0 + c, node = col / G;
            return reinterpret_cast<T*>(a.out) + ((int64_t)(u.q0 + node) * a.Hq + u.kvh * G + (col - node * G)) * a.D;
        });
    }
}

// Kept weights: grid (kMassJoins + key blocks of kMassKeys, Hkv, N).  The first blocks
// join the output rows of a cut unit.  The others take the unit's log2-sum-exp2 per query
// head (of a cut unit, from its parts) and add
// sum over the group's heads of 2^(score - lse) to their keys' totals, four keys
// per thread; the first heads' scores are loaded before the log-sum-exps are known.
constexpr int kMassKeys = 1024;
constexpr int kMassGroup = 64;   // query heads of a kv head, at most
constexpr int kMassAhead = 8;    // heads whose scores are in flight
constexpr int kMassJoins = 2;

template <typename T, int LR>
__global__ __launch_bounds__(256) void mass_join_kernel(TreeArgs a, int cols) {
    __shared__ JoinSmem sm;
    __shared__ float lse[kMassGroup];
    const int n = blockIdx.z, kvh = blockIdx.y, G = a.Hq / a.Hkv;
    const TreeSeq s = tree_seq(a, n);
    const int first = ((int)blockIdx.x - kMassJoins) * kMassKeys;
    if (first >= s.L) return;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j0 = first + 4 * (int)threadIdx.x;
    const bool keys = first >= 0;
    const float* sc = a.scores + ((int64_t)n * a.Hkv + kvh) * G * a.score_stride + j0;
    float* mass = a.mass + n * a.mass_bs + kvh * a.mass_hs + j0;
    mf32x4 x[kMassAhead];
    float old[4] = {0.f, 0.f, 0.f, 0.f};
    auto load = [&](int h0) {
#pragma unroll
        for (int h = 0; h < kMassAhead; ++h)
            if (j0 < s.L && h0 + h < G) x[h] = *reinterpret_cast<const mf32x4*>(sc + (h0 + h) * a.score_stride);
    };
    if (keys) {
        load(0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j0 + i < s.L) old[i] = mass[i];
    }
    const int64_t T_ = a.Hkv * a.plan[a.N];
    const int nwg = (int)min(T_, (int64_t)a.nwg);
    const int tiles = tree_tiles(s);
    const int64_t begin = a.Hkv * a.plan[n] + (int64_t)kvh * tiles, end = begin + tiles;   // one column block
    const int w = (int)wg_of(begin, T_, nwg), parts = (int)wg_of(end - 1, T_, nwg) - w + 1;
    const TreeCut u{n, G, 0, kvh, 2 * w + (begin == share_begin(w, T_, nwg) ? 0 : 1), parts, 1};
    if (!keys) {
        const int width = join_width<LR>(parts);
        for (int c0 = blockIdx.x * width; c0 < G && parts > 1; c0 += kMassJoins * width)
            join_columns<T, LR>(a, sm, cols, w, u, c0, G, [&](int c) {
                return reinterpret_cast<T*>(a.out) + ((int64_t)n * a.Hq + kvh * G + c) * a.D;
            });
        return;
    }
    for (int c = wv; c < G; c += 4) {
        float v;
        if (parts == 1) {
            v = a.lse[(int64_t)n * a.Hq + kvh * G + c];
        } else {
            float M = -INFINITY, sum = 0.0f;
            for (int j = lane; j < parts; j += 64) {
                const float y = a.part_lse[(int64_t)part_slot(w, u.slot, 1, j) * cols + c];
                const float mb = fmaxf(M, y), base = mb == -INFINITY ? 0.0f : mb;
                sum = sum * fast_exp2(M - base) + fast_exp2(y - base);
                M = mb;
            }
            const float top = wave_max(M);
            sum = wave_sum(sum * fast_exp2(M - (top == -INFINITY ? 0.0f : top)));
            v = top + fast_log2(sum);
        }
        if (lane == 0) lse[c] = v == -INFINITY ? INFINITY : v;   // no finite score: no weight
    }
    __syncthreads();
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int h0 = 0; h0 < G; h0 += kMassAhead) {
        if (h0 > 0) load(h0);
#pragma unroll
        for (int h = 0; h < kMassAhead; ++h) {
            if (h0 + h >= G) break;
            const float l = lse[h0 + h];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += fast_exp2(x[h][i] - l);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (j0 + i < s.L) mass[i] = old[i] + sum[i];
}

// Any head_dim up to 256, any page size and alignment.  Tree: one wave per
// (row, query head).  MASS: one wave per (sequence, kv head), head after head,
// the scores kept, then the totals.
template <typename T, bool MASS>
__global__ __launch_bounds__(64) void tree_generic_kernel(TreeArgs a) {
    __shared__ float q_s[256];
    __shared__ float p_s[64];
    __shared__ int64_t row_s[64];
    __shared__ float lse_s[kMassGroup];
    const int lane = threadIdx.x, D = a.D, G = a.Hq / a.Hkv;
    const int kvh = MASS ? blockIdx.y : blockIdx.y / G;
    int n = blockIdx.x;
    if (!MASS) {   // the sequence of row blockIdx.x: the last with cu_q[n] <= row
        int lo = 0, hi = a.N - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.cu_q[mid] <= (int)blockIdx.x) lo = mid;
            else hi = mid - 1;
        }
        n = lo;
    }
    const TreeSeq s = tree_seq(a, n);
    const int64_t row = MASS ? n : blockIdx.x;
    if (!MASS && (row < s.q0 || row >= s.q0 + s.P)) return;   // no sequence's row
    const int* bt = a.bt + (int64_t)n * a.max_blocks;
    const T* kp = reinterpret_cast<const T*>(a.k);
    const T* vp = reinterpret_cast<const T*>(a.v);
    const int64_t row_elems = (int64_t)a.Hkv * D;
    const int* mrow = MASS ? nullptr : a.mask + row * a.words;
    float* sc = MASS ? a.scores + ((int64_t)n * a.Hkv + kvh) * G * a.score_stride : nullptr;
    for (int h = 0; h < (MASS ? G : 1); ++h) {
        const int hq = MASS ? kvh * G + h : blockIdx.y;
        const int64_t off = (row * a.Hq + hq) * D;
        const T* qp = reinterpret_cast<const T*>(a.q) + off;
        __syncthreads();
        for (int d = lane; d < D; d += 64) q_s[d] = Elem<T>::to_f32(qp[d]) * a.scale_log2;
        __syncthreads();
        float m = kNegBig, l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int t0 = 0; t0 < s.L; t0 += 64) {
            const int t = t0 + lane;
            const bool seen = t < s.L && (MASS || (tree_bits(mrow, a.words, t - s.hist) & 1u) != 0);
            int64_t at = 0;
            float x = -INFINITY;
            if (seen) {
                at = ((int64_t)max(bt[t / a.bs], 0) * a.bs + t % a.bs) * row_elems + (int64_t)kvh * D;
                float d0 = 0.0f, d1 = 0.0f, d2 = 0.0f, d3 = 0.0f;   // four sums, added pairwise
                int d = 0;
                for (; d + 3 < D; d += 4) {
                    d0 = fmaf(q_s[d], Elem<T>::to_f32(kp[at + d]), d0);
                    d1 = fmaf(q_s[d + 1], Elem<T>::to_f32(kp[at + d + 1]), d1);
                    d2 = fmaf(q_s[d + 2], Elem<T>::to_f32(kp[at + d + 2]), d2);
                    d3 = fmaf(q_s[d + 3], Elem<T>::to_f32(kp[at + d + 3]), d3);
                }
                for (; d < D; ++d) d0 = fmaf(q_s[d], Elem<T>::to_f32(kp[at + d]), d0);
                x = (d0 + d1) + (d2 + d3);
            }
            if (MASS && t < s.L) sc[h * a.score_stride + t] = x;
            const float mx = fmaxf(m, wave_max(x));
            const float corr = fast_exp2(m - mx);
            const float p = seen ? fast_exp2(x - mx) : 0.0f;
            l = l * corr + wave_sum(p);
            m = mx;
            p_s[lane] = seen ? p : -1.0f;
            row_s[lane] = at;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= corr;
            const int cnt = min(64, s.L - t0);
            for (int j = 0; j < cnt; ++j) {
                const float pj = p_s[j];
                if (pj < 0.0f) continue;   // not seen (uniform)
                const int64_t rj = row_s[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = lane + 64 * i;
                    if (d < D) acc[i] = fmaf(pj, Elem<T>::to_f32(vp[rj + d]), acc[i]);
                }
            }
            __syncthreads();
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* op = reinterpret_cast<T*>(a.out) + off;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d < D) op[d] = Elem<T>::from_f32(acc[i] * inv);
        }
        if (MASS && lane == 0) lse_s[h] = l == 0.0f ? INFINITY : m + fast_log2(l);
    }
    if constexpr (MASS) {
        __syncthreads();
        float* mass = a.mass + n * a.mass_bs + kvh * a.mass_hs;
        for (int j = lane; j < s.L; j += 64) {   // each lane reads the scores that it wrote
            float sum = 0.0f;
            for (int h = 0; h < G; ++h) sum += fast_exp2(sc[h * a.score_stride + j] - lse_s[h]);
            mass[j] += sum;
        }
    }
}

// Ancestor masks and positions from parent indices, one work-group per
// sequence, one thread per node walking up its branch.  A parent outside [0, i)
// makes node i a root, so that every walk ends.
constexpr int kStagedNodes = 4096;

__global__ __launch_bounds__(256) void build_tree_kernel(int* mask, int words, int* positions, const int* parents,
                                                         const int* cu_q, const int* lens) {
    __shared__ int up_s[kStagedNodes];
    const int n = blockIdx.x, q0 = cu_q[n], P = cu_q[n + 1] - q0;
    const bool staged = P <= kStagedNodes;
    if (staged)
        for (int i = threadIdx.x; i < P; i += blockDim.x) up_s[i] = parents[q0 + i];
    __syncthreads();
    for (int i = threadIdx.x; i < P; i += blockDim.x) {
        int* row = mask + (int64_t)(q0 + i) * words;
        int depth = -1, word = words - 1;
        uint32_t bits = 0;   // of `word`; ancestors come in falling order
        for (int j = i; j >= 0;) {
            for (; word > j >> 5; --word) {
                row[word] = (int)bits;
                bits = 0;
            }
            if (word == j >> 5) bits |= 1u << (j & 31);   // (a node beyond the row's words has no bit)
            ++depth;
            const int up = staged ? up_s[j] : parents[q0 + j];
            j = up < j ? up : -1;
        }
        for (; word >= 0; --word) {
            row[word] = (int)bits;
            bits = 0;
        }
        if (positions) positions[q0 + i] = lens[n] - P + depth;
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
typedef void (*TreeKernel)(TreeArgs);

// The kernel of a shape and its columns per unit.
struct TreeChoice {
    TreeKernel fn = nullptr;
    int cols = 0, threads = 0;
};

template <class B>
TreeChoice choice() {
    return TreeChoice{tree_kernel<B>, B::kCols, B::kThreads};
}

// By the most columns that a sequence of the call has and the tiles of all
// (sequence, kv head) pairs.  mass: one unit per (sequence, kv head); wider groups
// than the kernels' columns take the generic one.
template <int D>
TreeChoice choose_f32(int64_t cols, int64_t tiles, bool mass) {
    if (mass) {
        if (cols <= 16) return choice<FewCols<D, 1, true>>();
        if constexpr (D < 256)
            if (cols <= 32) return choice<FewCols<D, 2, true>>();
        return TreeChoice();
    }
    // Two tiles of columns where there are tiles for 16 a compute unit (32/8/128, 16 x 2000
    // keys, 64 columns: 105 us, 112 by single ones); below that single ones (14/2/64, 64 x
    // 1000, 28 columns: 37 us and 46).
    if constexpr (D < 256)
        if (cols > 16 && tiles >= 16 * device_cus()) return choice<FewCols<D, 2, false>>();
    return choice<FewCols<D, 1, false>>();
}

// 16-bit pools.  From 129 columns on, units of 256 where there are tiles for 16 a
// compute unit and most of the last unit is columns (32/8/128, 16 x 4500 keys, 64
// nodes: 102 us, 117 by units of 64; 16 x 500 keys: 41 us and 27), else units of 64.  Up
// to 128, and at head_dim 256, one unit of 128 with eight waves and four tiles in the ring
// (16 x 4500 keys, 8 nodes: 61 us, 64 by units of 64 on four waves; 16/8/256, 61 x 1100
// keys, 8 nodes: 102 us and 110).
template <typename T, int D>
TreeChoice choose_16(int64_t cols, int64_t tiles, bool mass) {
    if (mass) return choice<ManyCols<T, D, 1, 8, 4, true>>();
    if constexpr (D <= 128) {
        if (cols > 128) {
            if (tiles >= 16 * device_cus() && (cols - 1) % 256 >= 192) return choice<ManyCols<T, D, 2, 8, 4>>();
            return choice<ManyCols<T, D, 1, 4, 2>>();
        }
    }
    return choice<ManyCols<T, D, 1, 8, 4>>();
}

template <typename T, int D>
TreeChoice choose(int64_t cols, int64_t tiles, bool mass) {
    if constexpr (Elem<T>::kDtype == LLKV_DTYPE_F32) return choose_f32<D>(cols, tiles, mass);
    else return choose_16<T, D>(cols, tiles, mass);
}

template <typename T>
TreeChoice choose(int D, int64_t cols, int64_t tiles, bool mass) {
    if (D == 64) return choose<T, 64>(cols, tiles, mass);
    if (D == 96) return choose<T, 96>(cols, tiles, mass);
    if (D == 128) return choose<T, 128>(cols, tiles, mass);
    return choose<T, 256>(cols, tiles, mass);
}

TreeChoice choose(int dtype, int D, int64_t cols, int64_t tiles, bool mass) {
    if (dtype == LLKV_DTYPE_F32) return choose<float>(D, cols, tiles, mass);
    if (dtype == LLKV_DTYPE_F16) return choose<_Float16>(D, cols, tiles, mass);
    return choose<bf16_t>(D, cols, tiles, mass);
}

template <typename T, int LR>
void launch_join(const TreeArgs& a, int cols, bool mass, hipStream_t st) {
    if (mass) {
        const dim3 grid((unsigned)(kMassJoins + (a.max_len + kMassKeys - 1) / kMassKeys), a.Hkv, a.N);
        mass_join_kernel<T, LR><<<grid, 256, 0, st>>>(a, cols);
    } else {
        // at most a round for each column of each work-group's one cut unit
        const int grid = (int)std::min<int64_t>((int64_t)a.nwg * cols, 1024);
        tree_join_kernel<T, LR><<<grid, 256, 0, st>>>(a, cols);
    }
}

template <typename T>
void launch_join(const TreeArgs& a, int cols, bool mass, hipStream_t st) {
    if (a.D == 64) launch_join<T, 16>(a, cols, mass, st);
    else if (a.D <= 128) launch_join<T, 32>(a, cols, mass, st);
    else launch_join<T, 64>(a, cols, mass, st);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a shape runs: on the matrix kernels (fn) with nwg work-groups at most, or on
// the generic one, and where its workspace's parts begin.
struct TreePlan {
    TreeKernel fn = nullptr;
    int cols = 0, threads = 0, nwg = 0;
    int64_t score_stride = 0;
    size_t rounds = 0, plan = 0, lse = 0, part_lse = 0, part_o = 0, scores = 0, total = 0;
};

TreePlan make_plan(int N, int rows_most, int Hq, int Hkv, int D, int bs, int max_len, int dtype, bool mass) {
    TreePlan p;
    const int n1 = std::min(N, kTreeSeqs);
    const int64_t cols = (int64_t)rows_most * (Hq / Hkv);
    const int64_t tiles = std::max<int64_t>(1, ((int64_t)max_len + kTreeTile - 1) / kTreeTile);
    TreeChoice c;
    if (bs == kPage && (D == 64 || D == 96 || D == 128 || D == 256)) c = choose(dtype, D, cols, tiles * n1 * Hkv, mass);
    p.fn = c.fn;
    if (c.fn) {
        p.cols = c.cols;
        p.threads = c.threads;
        const int64_t blocks = (cols + c.cols - 1) / c.cols;
        const int64_t all = (int64_t)n1 * Hkv * blocks * tiles;
        p.nwg = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(resident_workgroups((const void*)c.fn, c.threads), kMostShares), all));
        p.rounds = up256((size_t)p.nwg * sizeof(TreeCut));
        p.plan = p.rounds + up256((size_t)p.nwg * sizeof(int));
        p.lse = p.plan + up256((size_t)(n1 + 1) * sizeof(int64_t));
        p.part_lse = p.lse + (mass ? up256((size_t)n1 * Hq * 4) : 0);
        p.part_o = p.part_lse + up256((size_t)2 * p.nwg * p.cols * 4);
        p.scores = p.part_o + up256((size_t)2 * p.nwg * p.cols * D * 4);
    }
    p.total = p.scores;
    if (mass) {
        p.score_stride = ((int64_t)max_len + kTreeTile - 1) / kTreeTile * kTreeTile;
        p.total += (size_t)n1 * Hq * p.score_stride * 4;
    }
    return p;
}

bool aligned16(const void* a, const void* b, const void* c, const void* d) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0;
}

// One launch's worth of sequences at a time; a.N is the whole batch.
int run_tree(const char* fn, const TreeArgs& all, int rows, int rows_most, int max_len, int dtype, bool mass,
             void* workspace, size_t workspace_bytes, hipStream_t st) {
    const TreePlan p = make_plan(all.N, rows_most, all.Hq, all.Hkv, all.D, all.bs, max_len, dtype, mass);
    if (workspace_bytes < p.total || (p.total > 0 && !workspace))
        return set_error(LLKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, p.total);
    if (((uintptr_t)workspace & 15) != 0) return set_error(LLKV_ERR_INVALID, "%s: workspace not 16-byte aligned", fn);
    char* ws = reinterpret_cast<char*>(workspace);
    const size_t es = dtype_bytes(dtype);
    const bool tuned = p.fn != nullptr && aligned16(all.q, all.k, all.v, all.out);
    for (int n0 = 0; n0 < all.N; n0 += kTreeSeqs) {
        TreeArgs a = all;
        a.N = std::min(all.N - n0, kTreeSeqs);
        a.bt += (int64_t)n0 * a.max_blocks;
        a.lens += n0;
        if (a.cu_q) a.cu_q += n0;
        if (mass) {
            const int64_t off = (int64_t)n0 * a.Hq * a.D * es;
            a.q = reinterpret_cast<const char*>(a.q) + off;
            a.out = reinterpret_cast<char*>(a.out) + off;
            a.mass += n0 * a.mass_bs;
            a.scores = reinterpret_cast<float*>(ws + p.scores);
            a.score_stride = p.score_stride;
        }
        if (!tuned) {
            const dim3 grid(mass ? a.N : rows, mass ? a.Hkv : a.Hq);
            if (dtype == LLKV_DTYPE_F32)
                mass ? tree_generic_kernel<float, true><<<grid, 64, 0, st>>>(a)
                     : tree_generic_kernel<float, false><<<grid, 64, 0, st>>>(a);
            else if (dtype == LLKV_DTYPE_F16)
                mass ? tree_generic_kernel<_Float16, true><<<grid, 64, 0, st>>>(a)
                     : tree_generic_kernel<_Float16, false><<<grid, 64, 0, st>>>(a);
            else
                mass ? tree_generic_kernel<bf16_t, true><<<grid, 64, 0, st>>>(a)
                     : tree_generic_kernel<bf16_t, false><<<grid, 64, 0, st>>>(a);
            continue;
        }
        a.nwg = p.nwg;
        a.cuts = reinterpret_cast<TreeCut*>(ws);
        a.rounds = reinterpret_cast<int*>(ws + p.rounds);
        a.plan = reinterpret_cast<int64_t*>(ws + p.plan);
        a.lse = reinterpret_cast<float*>(ws + p.lse);
        a.part_lse = reinterpret_cast<float*>(ws + p.part_lse);
        a.part_o = reinterpret_cast<float*>(ws + p.part_o);
        p.fn<<<p.nwg, p.threads, 0, st>>>(a);
        if (dtype == LLKV_DTYPE_F32) launch_join<float>(a, p.cols, mass, st);
        else if (dtype == LLKV_DTYPE_F16) launch_join<_Float16>(a, p.cols, mass, st);
        else launch_join<bf16_t>(a, p.cols, mass, st);
    }
    return check_launch(fn);
}

int check_shapes(const char* fn, int N, int Hq, int Hkv, int D, int bs, int max_blocks, int max_len, int dtype) {
    if (N < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || bs <= 0 || max_blocks <= 0 || max_len < 0)
        return set_error(LLKV_ERR_INVALID, "%s: bad shape arguments", fn);
    if (D > 256) return set_error(LLKV_ERR_UNSUPPORTED, "%s: head_dim too large (%d > 256)", fn, D);
    if (Hq % Hkv != 0)
        return set_error(LLKV_ERR_INVALID, "%s: num_q_heads %d not a multiple of num_kv_heads %d", fn, Hq, Hkv);
    if (dtype_bytes(dtype) == 0) return set_error(LLKV_ERR_INVALID, "%s: unsupported dtype %d", fn, dtype);
    if ((int64_t)max_blocks * bs > INT32_MAX - kTreeTile || (int64_t)N * max_blocks > INT32_MAX)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: block table too large", fn);
    if (Hkv > 65535) return set_error(LLKV_ERR_UNSUPPORTED, "%s: more than 65535 kv heads", fn);
    return LLKV_OK;
}

}  // namespace
}  // namespace llkv

using namespace llkv;

extern "C" size_t llkv_paged_tree_attention_workspace_size(int num_seqs, int max_q_len, int num_q_heads,
                                                           int num_kv_heads, int head_dim, int block_size,
                                                           int max_seq_len, int dtype) {
    if (num_seqs <= 0 || max_q_len <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
        dtype_bytes(dtype) == 0)
        return 0;
    return make_plan(num_seqs, max_q_len, num_q_heads, num_kv_heads, head_dim, block_size, std::max(max_seq_len, 0),
                     dtype, false)
        .total;
}

extern "C" int llkv_paged_tree_attention(void* out, const void* q, const void* k_pool, const void* v_pool,
                                         const int* block_table, int max_blocks_per_seq, const int* cu_q,
                                         const int* seq_lens, const int* tree_mask, int mask_words, int num_seqs,
                                         int total_q, int max_q_len, int max_seq_len, int num_q_heads,
                                         int num_kv_heads, int head_dim, int block_size, float scale, int dtype,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "llkv_paged_tree_attention";
    if (num_seqs == 0 || total_q == 0) return LLKV_OK;
    const int rc = check_shapes(fn, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                                max_seq_len, dtype);
    if (rc != LLKV_OK) return rc;
    if (total_q < 0 || max_q_len <= 0 || mask_words <= 0 || (int64_t)mask_words * 32 < max_q_len)
        return set_error(LLKV_ERR_INVALID, "%s: mask rows of %d words for up to %d rows", fn, mask_words, max_q_len);
    if (!out || !q || !k_pool || !v_pool || !block_table || !cu_q || !seq_lens || !tree_mask)
        return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    if ((int64_t)total_q * (num_q_heads / num_kv_heads) > INT32_MAX - 256 || num_q_heads > 65535)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: too many rows and heads", fn);
    TreeArgs a = {};
    a.out = out;
    a.q = q;
    a.k = k_pool;
    a.v = v_pool;
    a.bt = block_table;
    a.cu_q = cu_q;
    a.lens = seq_lens;
    a.mask = tree_mask;
    a.words = mask_words;
    a.max_blocks = max_blocks_per_seq;
    a.N = num_seqs;
    a.Hq = num_q_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.bs = block_size;
    a.max_len = INT32_MAX;   // shares and tiles follow the actual lengths; the bound only sizes the launch
    a.scale_log2 = scale * kLog2e;
    return run_tree(fn, a, total_q, max_q_len, max_seq_len, dtype, false, workspace, workspace_bytes,
                    (hipStream_t)stream);
}

extern "C" size_t llkv_paged_decode_mass_workspace_size(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                                        int block_size, int max_seq_len, int dtype) {
    if (num_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
        dtype_bytes(dtype) == 0)
        return 0;
    return make_plan(num_seqs, 1, num_q_heads, num_kv_heads, head_dim, block_size, std::max(max_seq_len, 0), dtype, true)
        .total;
}

extern "C" int llkv_paged_decode_mass(void* out, float* mass, int64_t mass_seq_stride, int64_t mass_head_stride,
                                      const void* q, const void* k_pool, const void* v_pool, const int* block_table,
                                      const int* seq_lens, int num_seqs, int num_q_heads, int num_kv_heads,
                                      int head_dim, int block_size, int max_blocks_per_seq, int max_seq_len,
                                      float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "llkv_paged_decode_mass";
    if (num_seqs == 0) return LLKV_OK;
    const int rc = check_shapes(fn, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                                max_seq_len, dtype);
    if (rc != LLKV_OK) return rc;
    if (num_q_heads / num_kv_heads > kMassGroup)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: more than %d query heads per kv head", fn, kMassGroup);
    if (!out || !mass || !q || !k_pool || !v_pool || !block_table || !seq_lens)
        return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    if (mass_head_stride < max_seq_len || (num_seqs > 1 && mass_seq_stride < (int64_t)num_kv_heads * mass_head_stride))
        return set_error(LLKV_ERR_INVALID, "%s: totals of %lld keys a head for up to %d", fn,
                         (long long)mass_head_stride, max_seq_len);
    TreeArgs a = {};
    a.out = out;
    a.q = q;
    a.k = k_pool;
    a.v = v_pool;
    a.bt = block_table;
    a.lens = seq_lens;
    a.max_blocks = max_blocks_per_seq;
    a.N = num_seqs;
    a.Hq = num_q_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.bs = block_size;
    a.max_len = max_seq_len;   // scores and totals have room for so many
    a.scale_log2 = scale * kLog2e;
    a.mass = mass;
    a.mass_bs = mass_seq_stride;
    a.mass_hs = mass_head_stride;
    return run_tree(fn, a, num_seqs, 1, max_seq_len, dtype, true, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int llkv_build_tree(int* tree_mask, int mask_words, int* positions, const int* parents, const int* cu_q,
                               const int* seq_lens, int num_seqs, int total_q, int max_q_len, void* stream) {
    const char* fn = "llkv_build_tree";
    if (num_seqs == 0 || total_q == 0) return LLKV_OK;
    if (num_seqs < 0 || total_q < 0 || max_q_len <= 0 || mask_words <= 0 || (int64_t)mask_words * 32 < max_q_len)
        return set_error(LLKV_ERR_INVALID, "%s: mask rows of %d words for up to %d rows", fn, mask_words, max_q_len);
    if (!tree_mask || !parents || !cu_q || (positions && !seq_lens))
        return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    build_tree_kernel<<<num_seqs, 256, 0, (hipStream_t)stream>>>(tree_mask, mask_words, positions, parents, cu_q,
                                                                 seq_lens);
    return check_launch(fn);
}
