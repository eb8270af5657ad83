// Attention for trees of drafted tokens over the paged cache, and the decode
// step that adds its attention weights to each key's total (gfx950).  The
// schedule is in tree_attn.h.
//
// Body of one wave (FewCols): a page of 16 keys at a time, K and V straight
// into the operand registers of the matrix instructions in the decode's layouts
// (decode_mfma.h), NCT tiles of 16 columns against each.  The four waves of a
// work-group take the four pages of a tile and join their softmax states
// through LDS at the end of a segment.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

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

template <typename TT, int D_, int NCT_, bool MASS>
struct FewCols {
    using T = TT;
    static constexpr int D = D_, NCT = NCT_, W = 4;
    static constexpr int kCols = 16 * NCT;
    static constexpr bool kMass = MASS;
    static constexpr bool k16 = Elem<T>::kDtype != LLKV_DTYPE_F32;
    static constexpr bool kF16 = Elem<T>::kDtype == LLKV_DTYPE_F16;
    using Ops = ScoreOps<T, D>;
    static constexpr int VH = (D + 63) / 64, DT = 4 * VH, MD = VH;

    struct Smem {
        float acc[W][16][D];
        float ml[W][16][2];   // (max, sum)
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

        typename Ops::QReg q[NCT][Ops::NQ];
        const int* mrow[NCT];
        mf32x4 o[NCT][DT];
        float m[NCT], l[NCT];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
            const int col = sg.c0 + 16 * ct + c;
            const bool valid = col < sg.cols;
            const int node = valid ? col / G : 0;
            const int64_t row = sg.s.q0 + node;
            Ops::load_q(reinterpret_cast<const T*>(a.q) + (row * a.Hq + sg.kvh * G + (col - node * G)) * D, valid, g,
                        a.scale_log2, q[ct]);
            mrow[ct] = MASS ? nullptr : a.mask + row * a.words;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[ct][dt] = mf32x4{0.f, 0.f, 0.f, 0.f};
            m[ct] = kNegBig;
            l[ct] = 0.0f;
        }

        const int npages = (L + kPage - 1) / kPage;
        const int count = sg.t1 - sg.t0;   // this wave's pages: 4 (t0 + j) + w, j < count
        int tbl = 0;
        for (int j = 0; j < count; ++j) {
            if ((j & 63) == 0) {   // the next 64 page ids, one per lane
                const int pg = W * (sg.t0 + j + lane) + w;
                tbl = pg < npages ? bt[pg] : 0;
            }
            const int pg = W * (sg.t0 + j) + w;
            if (pg >= npages) break;
            const int64_t phys = max(__builtin_amdgcn_readlane(tbl, j & 63), 0);

            typename Ops::KReg kr[Ops::NK];
            Ops::template load_k<false>(kbase + (phys * kPage + c) * row_elems, g, kr);
            float4 vr[VH][4];
            mu32x2 vh[VH][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T* vp = vbase + (phys * kPage + 4 * g + i) * row_elems + 4 * c;
#pragma unroll
                for (int h = 0; h < VH; ++h) {
                    if (D % 64 != 0 && 64 * h + 4 * c >= D) {   // past the head's last dim
                        vh[h][i] = mu32x2{0u, 0u};
                        vr[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    } else if constexpr (k16) {
                        vh[h][i] = load_vec<false, mu32x2>(vp + 64 * h);
                    } else {
                        vr[h][i] = Ops::template load_v4<false>(vp + 64 * h);
                    }
                }
            }

            // Keys that some columns do not see: the last page's rest, where V may hold
            // anything and is taken as zero, and the tree's own, where a value that is not
            // finite must reach the columns that see it and no other.
            const int p0 = pg * kPage;
            const bool whole = p0 + kPage <= min(hist, L);   // uniform
            bool odd = false;
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool beyond = p0 + 4 * g + i >= L, tree = p0 + 4 * g + i >= hist;
#pragma unroll
                    for (int h = 0; h < VH; ++h) {
                        if constexpr (k16) {
                            const bool bad = !finite_bits(vh[h][i].x, kF16) || !finite_bits(vh[h][i].y, kF16);
                            odd |= bad && tree && !beyond;
                            if (beyond || (bad && tree)) vh[h][i] = mu32x2{0u, 0u};
                        } else {
                            const bool bad = !(isfinite(vr[h][i].x) && isfinite(vr[h][i].y) && isfinite(vr[h][i].z) &&
                                               isfinite(vr[h][i].w));
                            odd |= bad && tree && !beyond;
                            if (beyond || (bad && tree)) vr[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                    }
                }
            }
            const bool any_odd = !whole && __builtin_amdgcn_ballot_w64(odd) != 0;

            mu32x2 av[VH][4];   // V^T operands of the 16-bit product
            if constexpr (k16) {
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        const unsigned sel = (jj & 1) ? 0x07060302u : 0x05040100u;
                        const int wd = jj >> 1;
                        av[h][jj] = mu32x2{__builtin_amdgcn_perm(vh[h][1][wd], vh[h][0][wd], sel),
                                           __builtin_amdgcn_perm(vh[h][3][wd], vh[h][2][wd], sel)};
                    }
            }

#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
                const mf32x4 sc = Ops::scores(kr, q[ct], a.scale_log2);
                float x[4] = {sc[0], sc[1], sc[2], sc[3]};
                uint32_t seen = ~0u;   // bit i: the lane's key i
                if (!whole) {
                    const int p4 = p0 + 4 * g;
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
                // 8 (2^8 fits every type), so most pages need no exchange between lanes.
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
                if constexpr (k16) {
                    // P in the pool's type, as the prefill: at most half a step of each weight.
                    const mu32x2 pb = kF16 ? mu32x2{pack_h2(p[0], p[1]), pack_h2(p[2], p[3])}
                                           : mu32x2{pack_b2(p[0], p[1]), pack_b2(p[2], p[3])};
#pragma unroll
                    for (int h = 0; h < VH; ++h)
#pragma unroll
                        for (int jj = 0; jj < 4; ++jj) {
                            mf32x4& acc = o[ct][4 * h + jj];
                            if constexpr (kF16)
                                acc = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(mf16x4, av[h][jj]),
                                                                            __builtin_bit_cast(mf16x4, pb), acc, 0, 0, 0);
                            else
                                acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(ms16x4, av[h][jj]),
                                                                                __builtin_bit_cast(ms16x4, pb), acc, 0, 0, 0);
                        }
                } else {
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
                if (any_odd) add_odd(vbase + phys * kPage * row_elems, row_elems, p0, hist, L, seen, p, o[ct]);
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

    // The products of V's values that are not finite, which the matrix instructions took as
    // zero, added for the columns that see their keys (a masked weight of zero times infinity
    // would be NaN).  vrow0: row 0 of the page.
    __device__ static void add_odd(const T* vrow0, int64_t row_elems, int p0, int hist, int L, uint32_t seen,
                                   const float (&p)[4], mf32x4 (&o)[DT]) {
        const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
        for (int tg = 0; tg < 4; ++tg)
#pragma unroll
            for (int ti = 0; ti < 4; ++ti) {
                const float pt = __shfl(seen >> ti & 1u ? p[ti] : -1.0f, 16 * tg + c, 64);
                const int pos = p0 + 4 * tg + ti;
                if (pos < hist || pos >= L) continue;   // uniform
                const T* vrow = vrow0 + (4 * tg + ti) * row_elems;
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int jj = 0; jj < 4; ++jj) {
                            const int d = 64 * h + 16 * g + 4 * i + jj;
                            if (D % 64 != 0 && d >= D) continue;
                            // the four dims that one lane loaded were taken as zero together
                            bool bad = false;
#pragma unroll
                            for (int e = 0; e < 4; ++e) bad |= !isfinite(Elem<T>::to_f32(vrow[d - jj + e]));
                            if (bad && pt >= 0.0f) o[4 * h + jj][i] += pt * Elem<T>::to_f32(vrow[d]);
                        }
            }
    }
};

template <class B>
__global__ __launch_bounds__(256) void tree_kernel(TreeArgs a) {
    __shared__ typename B::Smem sm;
    __shared__ int64_t sP[kTreeSeqs + 1];
    tree_scan<B::kCols>(a, sP);
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= a.N; i += blockDim.x) a.plan[i] = sP[i];
    const int64_t T = a.Hkv * sP[a.N];
    const int nwg = tree_shares(a, T);
    const int w = blockIdx.x;
    if (w >= nwg) return;
    const int64_t r0 = share_begin(w, T, nwg), r1 = share_begin(w + 1, T, nwg);
    const int G = a.Hq / a.Hkv;
    for (int64_t p = r0; p < r1;) {
        TreeSeg sg;
        sg.n = tree_find(sP, a.N, a.Hkv, p);
        sg.s = tree_seq(a, sg.n);
        const TreeUnit u = tree_unit(a, sP, sg.n, tree_tiles(sg.s), p);
        const int64_t end = u.begin + u.tiles, stop = end < r1 ? end : r1;
        sg.kvh = u.kvh;
        sg.cols = sg.s.P * G;
        sg.c0 = u.cb * B::kCols;
        sg.t0 = (int)(p - u.begin);
        sg.t1 = (int)(stop - u.begin);
        sg.direct = p == u.begin && stop == end;
        sg.slot = 2 * w + (p == r0 ? 0 : 1);
        B::run(a, sm, sg);
        p = stop;
    }
}

// The unit that begins in share w and is cut at its end, with the shares
// w .. last that hold the rest of it; false when there is none.
__device__ inline bool cut_unit(const TreeArgs& a, int w, TreeUnit& u, int& first_slot, int& parts) {
    const int64_t T = a.Hkv * a.plan[a.N];
    const int nwg = tree_shares(a, T);
    if (w >= nwg - 1) return false;   // the last share's units end with it
    const int64_t r0 = share_begin(w, T, nwg), r1 = share_begin(w + 1, T, nwg);
    const int n = tree_find(a.plan, a.N, a.Hkv, r1 - 1);
    u = tree_unit(a, a.plan, n, tree_tiles(tree_seq(a, n)), r1 - 1);
    const int64_t end = u.begin + u.tiles;
    if (u.begin < r0 || end <= r1) return false;
    first_slot = 2 * w + (u.begin == r0 ? 0 : 1);
    parts = (int)(wg_of(end - 1, T, nwg) - w) + 1;
    return true;
}

// Slot of part j of a cut unit whose first share is w.
__device__ inline int part_slot(int w, int first_slot, int j) { return j == 0 ? first_slot : 2 * (w + j); }

// Log-sum-exp join of one column's parts: a wave, lane owning dims lane + 64 i.
// Returns the column's log2-sum-exp2.
template <typename T, int MD>
__device__ inline float join_parts(const TreeArgs& a, int cols, int w, int first_slot, int parts, int col, T* out) {
    constexpr int kBatch = 8;
    const int lane = threadIdx.x & 63;
    float M = -INFINITY, sum = 0.0f, o[MD];
#pragma unroll
    for (int i = 0; i < MD; ++i) o[i] = 0.0f;
    for (int j0 = 0; j0 < parts; j0 += kBatch) {
        float lv[kBatch], pv[kBatch][MD];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const bool ok = j0 + j < parts;
            const int64_t row = (int64_t)part_slot(w, first_slot, j0 + (ok ? j : 0)) * cols + col;
            lv[j] = ok ? a.part_lse[row] : -INFINITY;
#pragma unroll
            for (int i = 0; i < MD; ++i) pv[j][i] = a.part_o[row * a.D + min(lane + 64 * i, a.D - 1)];
        }
        float mb = M;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) mb = fmaxf(mb, lv[j]);
        if (mb == -INFINITY) continue;   // no key seen so far
        const float sc = fast_exp2(M - mb);
        sum *= sc;
#pragma unroll
        for (int i = 0; i < MD; ++i) o[i] *= sc;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float f = fast_exp2(lv[j] - mb);
            sum += f;
#pragma unroll
            for (int i = 0; i < MD; ++i) o[i] = fmaf(f, pv[j][i], o[i]);
        }
        M = mb;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < MD; ++i)
        if (lane + 64 * i < a.D) out[lane + 64 * i] = Elem<T>::from_f32(o[i] * inv);
    return sum == 0.0f ? -INFINITY : M + fast_log2(sum);
}

// Grid (shares, columns / 4), a wave per column.
template <typename T, int MD>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int cols) {
    TreeUnit u;
    int slot, parts;
    if (!cut_unit(a, blockIdx.x, u, slot, parts)) return;
    const int G = a.Hq / a.Hkv;
    const int lc = blockIdx.y * 4 + (threadIdx.x >> 6), col = u.cb * cols + lc;
    const TreeSeq s = tree_seq(a, u.n);
    if (col >= s.P * G) return;
    const int node = col / G;
    T* out = reinterpret_cast<T*>(a.out) + ((int64_t)(s.q0 + node) * a.Hq + u.kvh * G + (col - node * G)) * a.D;
    join_parts<T, MD>(a, cols, blockIdx.x, slot, parts, lc, out);
}

// Kept weights: grid (key blocks of kMassKeys, Hkv, N).  Each work-group takes
// the unit's log2-sum-exp2 per query head (joining the parts of a cut unit; the
// first key block joins its output rows as well), then adds
// sum over the group's heads of 2^(score - lse) to its keys' totals.
constexpr int kMassKeys = 1024;
constexpr int kMassGroup = 64;   // query heads of a kv head (tree_cols' most columns)

template <typename T, int MD>
__global__ __launch_bounds__(256) void mass_join_kernel(TreeArgs a, int cols) {
    __shared__ float lse[kMassGroup];
    const int n = blockIdx.z, kvh = blockIdx.y, G = a.Hq / a.Hkv;
    const TreeSeq s = tree_seq(a, n);
    if (blockIdx.x > 0 && (int)blockIdx.x * kMassKeys >= s.L) return;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t T_ = a.Hkv * a.plan[a.N];
    const int nwg = tree_shares(a, T_);
    const int tiles = tree_tiles(s);
    const int64_t begin = a.Hkv * a.plan[n] + (int64_t)kvh * tiles, end = begin + tiles;   // one column block
    const int w = (int)wg_of(begin, T_, nwg), last = (int)wg_of(end - 1, T_, nwg);
    const int slot = 2 * w + (begin == share_begin(w, T_, nwg) ? 0 : 1);
    for (int c = wv; c < G; c += 4) {
        const int64_t hq = (int64_t)n * a.Hq + kvh * G + c;
        float v;
        if (w == last) {
            v = a.lse[hq];
        } else if (blockIdx.x == 0) {
            v = join_parts<T, MD>(a, cols, w, slot, last - w + 1, c, reinterpret_cast<T*>(a.out) + hq * a.D);
        } else {
            float M = -INFINITY, sum = 0.0f;
            for (int j = lane; j < last - w + 1; j += 64) {
                const float x = a.part_lse[(int64_t)part_slot(w, slot, j) * cols + c];
                const float mb = fmaxf(M, x);
                if (mb == -INFINITY) continue;
                sum = sum * fast_exp2(M - mb) + fast_exp2(x - mb);
                M = mb;
            }
            const float top = wave_max(M);
            sum = wave_sum(top == -INFINITY ? 0.0f : sum * fast_exp2(M - top));
            v = top + fast_log2(sum);
        }
        if (lane == 0) lse[c] = v == -INFINITY ? INFINITY : v;   // no finite score: no weight
    }
    __syncthreads();
    float* mass = a.mass + n * a.mass_bs + kvh * a.mass_hs;
    const float* sc = a.scores + ((int64_t)n * a.Hkv + kvh) * G * a.score_stride;
    const int stop = min(s.L, ((int)blockIdx.x + 1) * kMassKeys);
    for (int j = blockIdx.x * kMassKeys + threadIdx.x; j < stop; j += 256) {
        float sum = 0.0f;
        for (int c = 0; c < G; ++c) sum += fast_exp2(sc[c * a.score_stride + j] - lse[c]);
        mass[j] += sum;
    }
}

// Any head_dim up to 256, any page size and alignment.  Tree: one wave per
// (row, query head).  MASS: one wave per (sequence, kv head), head after head,
// the scores kept, then the totals.
template <typename T, bool MASS>
__global__ __launch_bounds__(64) void tree_generic_kernel(TreeArgs a, int rows) {
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

// Most column tiles whose accumulators and queries a wave's registers hold.
template <typename T, int D>
constexpr int most_tiles() {
    constexpr bool k16 = Elem<T>::kDtype != LLKV_DTYPE_F32;
    return k16 ? (D == 256 ? 2 : 4) : (D == 64 ? 4 : (D == 256 ? 1 : 2));
}

template <typename T, int D>
TreeKernel kernel_for(int nct, bool mass) {
    constexpr int most = most_tiles<T, D>();
    if (mass) {
        if (nct == 1) return tree_kernel<FewCols<T, D, 1, true>>;
        if constexpr (most >= 2) if (nct == 2) return tree_kernel<FewCols<T, D, 2, true>>;
        if constexpr (most >= 4) if (nct == 4) return tree_kernel<FewCols<T, D, 4, true>>;
    } else {
        if (nct == 1) return tree_kernel<FewCols<T, D, 1, false>>;
        if constexpr (most >= 2) if (nct == 2) return tree_kernel<FewCols<T, D, 2, false>>;
        if constexpr (most >= 4) if (nct == 4) return tree_kernel<FewCols<T, D, 4, false>>;
    }
    return nullptr;
}

template <typename T>
TreeKernel kernel_for(int D, int nct, bool mass) {
    if (D == 64) return kernel_for<T, 64>(nct, mass);
    if (D == 96) return kernel_for<T, 96>(nct, mass);
    if (D == 128) return kernel_for<T, 128>(nct, mass);
    return kernel_for<T, 256>(nct, mass);
}

TreeKernel kernel_for(int dtype, int D, int nct, bool mass) {
    if (dtype == LLKV_DTYPE_F32) return kernel_for<float>(D, nct, mass);
    if (dtype == LLKV_DTYPE_F16) return kernel_for<_Float16>(D, nct, mass);
    return kernel_for<bf16_t>(D, nct, mass);
}

template <typename T>
void launch_join(const TreeArgs& a, int cols, bool mass, hipStream_t st) {
    const int md = (a.D + 63) / 64;
    if (mass) {
        const dim3 grid((unsigned)std::max(1, (a.max_len + kMassKeys - 1) / kMassKeys), a.Hkv, a.N);
        if (md == 1) mass_join_kernel<T, 1><<<grid, 256, 0, st>>>(a, cols);
        else if (md == 2) mass_join_kernel<T, 2><<<grid, 256, 0, st>>>(a, cols);
        else mass_join_kernel<T, 4><<<grid, 256, 0, st>>>(a, cols);
        return;
    }
    const dim3 grid(a.nwg, cols / 4);
    if (md == 1) tree_join_kernel<T, 1><<<grid, 256, 0, st>>>(a, cols);
    else if (md == 2) tree_join_kernel<T, 2><<<grid, 256, 0, st>>>(a, cols);
    else tree_join_kernel<T, 4><<<grid, 256, 0, st>>>(a, cols);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a shape runs: on the matrix kernels (nct > 0) with nwg work-groups at most,
// and where its workspace's parts begin.
struct TreePlan {
    int nct = 0, cols = 0, nwg = 0;
    int64_t score_stride = 0;
    size_t plan = 0, lse = 0, part_lse = 0, part_o = 0, scores = 0, total = 0;
};

// The schedule does not depend on pointers: unaligned calls use the scores alone.
TreePlan make_plan(int N, int rows_most, int Hq, int Hkv, int D, int bs, int max_len, int dtype, bool mass) {
    TreePlan p;
    const int G = Hq / Hkv;
    const int n1 = std::min(N, kTreeSeqs);
    if (bs == kPage && (D == 64 || D == 96 || D == 128 || D == 256)) {
        int most = 4;
        while (most > 1 && !kernel_for(dtype, D, most, mass)) most /= 2;
        const int64_t cols = (int64_t)rows_most * G;
        p.nct = cols <= 16 ? 1 : (cols <= 32 ? std::min(2, most) : most);
        if (mass && cols > 16 * p.nct) p.nct = 0;   // a unit is one column block there
    }
    if (p.nct > 0) {
        p.cols = 16 * p.nct;
        const int64_t blocks = ((int64_t)rows_most * G + p.cols - 1) / p.cols;
        const int64_t tiles = std::max<int64_t>(1, ((int64_t)max_len + kTreeTile - 1) / kTreeTile);
        const int64_t all = (int64_t)n1 * Hkv * blocks * tiles;
        const int res = resident_workgroups((const void*)kernel_for(dtype, D, p.nct, mass), 256);
        p.nwg = (int)std::max<int64_t>(1, std::min<int64_t>(res, all));
        p.lse = up256((size_t)(n1 + 1) * sizeof(int64_t));
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
    const bool tuned = p.nct > 0 && aligned16(all.q, all.k, all.v, all.out);
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
            const int nrows = rows;
            if (dtype == LLKV_DTYPE_F32)
                mass ? tree_generic_kernel<float, true><<<grid, 64, 0, st>>>(a, nrows)
                     : tree_generic_kernel<float, false><<<grid, 64, 0, st>>>(a, nrows);
            else if (dtype == LLKV_DTYPE_F16)
                mass ? tree_generic_kernel<_Float16, true><<<grid, 64, 0, st>>>(a, nrows)
                     : tree_generic_kernel<_Float16, false><<<grid, 64, 0, st>>>(a, nrows);
            else
                mass ? tree_generic_kernel<bf16_t, true><<<grid, 64, 0, st>>>(a, nrows)
                     : tree_generic_kernel<bf16_t, false><<<grid, 64, 0, st>>>(a, nrows);
            continue;
        }
        a.nwg = p.nwg;
        a.plan = reinterpret_cast<int64_t*>(ws);
        a.lse = reinterpret_cast<float*>(ws + p.lse);
        a.part_lse = reinterpret_cast<float*>(ws + p.part_lse);
        a.part_o = reinterpret_cast<float*>(ws + p.part_o);
        kernel_for(dtype, a.D, p.nct, mass)<<<p.nwg, 256, 0, st>>>(a);
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
