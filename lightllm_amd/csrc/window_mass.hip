// The attention weight that the last rows of each sequence give to each of its
// keys, summed over rows and query heads and added to the keys' totals (gfx950).
//
// For a sequence of L keys whose last P rows are given, row i (at position
// L - P + i) seeing keys j <= L - P + i:
//     total[h][j] += sum over rows i and the heads c of kv head h of
//                    exp(x_ijc - lse_ic),   x = scale q_ic . k_j.
// The scores (4 bytes for each of the P G columns of a key) are more than the
// key's K row, so they are computed twice rather than stored: once for each
// column's log-sum-exp, once for the sums.  Both passes hold a block of keys in
// the operand registers of the matrix instructions (K as in the decode) and run
// over the columns, so that K is read once a pass, a key's sum stays in one
// wave's registers and nothing is added atomically.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_common.h"
#include "decode_mfma.h"
#include "lds_dma.h"

namespace llkv {
namespace {

struct WindowArgs {
    const void* q;
    const void* k;
    const int* bt;
    const int* cu_q;
    const int* lens;
    int max_blocks, N, Hq, Hkv, D, bs, max_len;
    float scale_log2;
    int nblk;          // key blocks of a sequence, a wave's keys each (by the bound)
    int64_t cols;      // rows x (Hq / Hkv) of the call
    float* part;       // [nblk][Hkv][cols] log2-sum-exp2 per key block
    float* lse;        // [Hkv][cols] (the generic kernels: [rows][Hq])
    float* mass;
    int64_t mass_bs, mass_hs;
};

struct WindowSeq {
    int q0, P, L, hist;
};

__device__ inline WindowSeq window_seq(const WindowArgs& a, int n) {
    WindowSeq s;
    s.q0 = a.cu_q[n];
    s.P = max(a.cu_q[n + 1] - s.q0, 0);
    const int l = a.lens[n], cap = min(a.max_blocks * a.bs, a.max_len);
    s.L = l < 0 ? 0 : (l > cap ? cap : l);
    s.hist = s.L - s.P;
    return s;
}

// Keys per wave: as many 16-key tiles as leave registers for two waves per SIMD.
template <typename T>
constexpr int key_tiles() { return Elem<T>::kDtype == LLKV_DTYPE_F32 ? 2 : 4; }
template <typename T>
constexpr int wave_keys() { return 16 * key_tiles<T>(); }

// Columns per LDS chunk: 16 KB of rows (24 KB at head_dim 96, where a chunk has to be
// whole loads of a work-group).
template <typename T, int D>
constexpr int chunk_cols() { return D == 96 ? 512 / (int)sizeof(T) / 2 : 16384 / (D * (int)sizeof(T)); }

// x and the value of the lane 16 (32) away, reduced: the four lanes of a column, which
// lie in different rows of 16, by swaps of rows between two registers.
template <class F>
__device__ inline float over_rows(float x, F f) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// SUM false: the log2-sum-exp2 of each column over a wave's keys, part[wave][kv head][column].
// SUM true: the totals, from the columns' log2-sum-exp2.
// Grid (nblk / W, Hkv, N), W waves.  The columns' rows go through LDS by direct loads,
// a ring of three chunks that all waves read: read by each wave from the caches, they
// took 6 TB/s from L2 and set the time (28/4/128 bf16, 2 x 30001 keys, 64 rows: 72 and
// 100 us the two passes).  A row's 16-byte units are XOR-ed with the column (rotated by
// it at head_dim 96), so that the 16 columns of an operand lie in different banks.  The
// second pass has its columns' log2-sum-exp2 in the ring as well, and the first stores a
// chunk's results a chunk later, before it issues the loads of another one: vector
// memory returns in order, so a load or store of its own behind those of the ring made
// every step wait for the ring (53 us a pass).
template <typename T, int D, int W, bool SUM>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D == 256 ? (sizeof(T) == 2 ? 2 : 1) : (D == 128 && sizeof(T) == 4 ? 3 : 4))))
void window_kernel(WindowArgs a) {
    using Ops = ScoreOps<T, D>;
    constexpr int KT = key_tiles<T>();
    constexpr bool k16 = Elem<T>::kDtype != LLKV_DTYPE_F32;
    constexpr int NC = chunk_cols<T, D>(), CPR = D * (int)sizeof(T) / 16, R = 3;
    constexpr int NS = NC / 16, NK = (NC + 63) / 64;   // steps of 16 columns, column blocks of 64
    constexpr int LPW = NC * CPR / (64 * W) + (SUM ? NK : 0);   // loads of a lane per chunk
    static_assert(NC % 16 == 0 && NC * CPR % (64 * W) == 0, "chunks are whole loads");
    __shared__ mu32x4 rows[R][NC * CPR];
    __shared__ float lse_s[SUM ? R : 1][SUM ? 64 * NK : 1];
    const int n = blockIdx.z, kvh = blockIdx.y;
    const WindowSeq s = window_seq(a, n);
    if ((int)blockIdx.x * W * wave_keys<T>() >= s.L || s.P == 0) return;   // uniform over the work-group
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int blk = blockIdx.x * W + w;
    const int k0 = blk * wave_keys<T>();
    const bool idle = k0 >= s.L;   // the wave has no key: it loads and waits only
    const int G = a.Hq / a.Hkv, cols = s.P * G, chunks = (cols + NC - 1) / NC;
    const int64_t row_elems = (int64_t)a.Hkv * D;
    const float* const lse = a.lse + kvh * a.cols + (int64_t)s.q0 * G;
    float* const part = a.part + ((int64_t)blk * a.Hkv + kvh) * a.cols + (int64_t)s.q0 * G;

    auto place = [](int col, int u) { return (CPR & (CPR - 1)) == 0 ? u ^ (col & (CPR - 1)) : (u + col) % CPR; };
    auto unit_at = [](int col, int pl) {
        return (CPR & (CPR - 1)) == 0 ? pl ^ (col & (CPR - 1)) : (pl + CPR * NC - col) % CPR;
    };
    const char* const qbase = reinterpret_cast<const char*>(a.q) + ((int64_t)s.q0 * a.Hq + kvh * G) * D * (int)sizeof(T);
    constexpr int RL = NC * CPR / (64 * W);   // of them rows
    uint32_t lds[RL], lds_lse[NK];
#pragma unroll
    for (int i = 0; i < RL; ++i) lds[i] = lds_addr(&rows[0][64 * (RL * w + i)]);
#pragma unroll
    for (int i = 0; i < NK; ++i) lds_lse[i] = lds_addr(&lse_s[0][SUM ? 64 * i : 0]);
    auto load_chunk = [&](int ch) {
#pragma unroll
        for (int i = 0; i < RL; ++i) {
            const int x = 64 * (RL * w + i) + lane, r = x / CPR;
            const int col = min(ch * NC + r, cols - 1), node = col / G;   // (beyond the last: not used)
            const int64_t off = ((int64_t)node * a.Hq + (col - node * G)) * D * (int)sizeof(T) + unit_at(r, x % CPR) * 16;
            dma16(qbase + off, lds[i] + (uint32_t)(ch % R) * (NC * CPR * 16));
        }
        if constexpr (SUM) {   // every wave the same values: its own wait covers them
#pragma unroll
            for (int i = 0; i < NK; ++i)
                dma4(lse + min(ch * NC + 64 * i + lane, cols - 1), lds_lse[i] + (uint32_t)(ch % R) * (64 * NK * 4));
        }
    };
    load_chunk(0);
    if (chunks > 1) load_chunk(1);

    typename Ops::KReg kr[KT][Ops::NK];
    if (!idle) {
        const int* bt = a.bt + (int64_t)n * a.max_blocks;
        const int last_page = (s.L - 1) / kPage;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            const int64_t phys = max(bt[min(k0 / kPage + kt, last_page)], 0);   // (beyond the last page: masked)
            Ops::template load_k<false>(reinterpret_cast<const T*>(a.k) + (int64_t)kvh * D + (phys * kPage + c) * row_elems,
                                        g, kr[kt]);
        }
        // fp32 keys are scaled here, 16-bit scores in the exponent; a negative scale goes into
        // the keys' signs, so that the largest score stays the largest when scaled.
        if constexpr (k16) {
            if (a.scale_log2 < 0.0f) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < Ops::NK; ++i) kr[kt][i] ^= 0x80008000u;
            }
        } else {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int i = 0; i < Ops::NK; ++i) {
                    kr[kt][i].x *= a.scale_log2;
                    kr[kt][i].y *= a.scale_log2;
                    kr[kt][i].z *= a.scale_log2;
                    kr[kt][i].w *= a.scale_log2;
                }
        }
    }
    const bool whole = k0 + wave_keys<T>() <= s.hist;   // every row sees all of the wave's keys (uniform)
    const float scale = k16 ? fabsf(a.scale_log2) : 1.0f;

    float sum[KT][4];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[kt][i] = 0.0f;
    // The keys have arrived: left open, the compiler's waits for them stayed in the loop, where
    // they meet the ring's loads.
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));

    // First pass: the maximum and the sum of column 64 k + lane of a chunk.
    float top_of[NK], sum_of[NK];
    auto store_chunk = [&](int ch) {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int x = 64 * k + lane, col = ch * NC + x;
            if (x < NC && col < cols) part[col] = sum_of[k] == 0.0f ? -INFINITY : top_of[k] + fast_log2(sum_of[k]);
        }
    };

    for (int ch = 0; ch < chunks; ++ch) {
        if (ch + 1 < chunks) __builtin_amdgcn_s_waitcnt(vmcnt_imm(LPW));   // all but the next chunk's loads
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        lds_barrier();   // the chunk is there for all, and the one before it has been read
        if constexpr (!SUM) {
            if (ch > 0 && !idle) store_chunk(ch - 1);
        }
        if (ch + 2 < chunks) load_chunk(ch + 2);
        if (idle) continue;
        const mu32x4* const here = rows[ch % R];
        const int stop = min(NC, cols - ch * NC);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const int c0 = 16 * st;
            if (c0 >= stop) break;   // (uniform)
            typename Ops::QReg q[Ops::NQ];
#pragma unroll
            for (int i = 0; i < CPR / 4; ++i) {
                const mu32x4 x = here[(c0 + c) * CPR + place(c0 + c, 4 * i + g)];
                if constexpr (k16) {
                    q[i] = x;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[4 * i + e] = __uint_as_float(x[e]);
                }
            }
            mf32x4 x[KT];
            if constexpr (k16) {   // k-step by k-step: four products that do not wait for each other
#pragma unroll
                for (int ks = 0; ks < Ops::NK; ++ks) {
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
                        x[kt] = Ops::mma(kr[kt][ks], q[ks], ks == 0 ? mf32x4{0.f, 0.f, 0.f, 0.f} : x[kt]);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, Ops::NK, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, Ops::NK * KT, 0);
            } else {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) x[kt] = Ops::scores(kr[kt], q, 1.0f);
            }
            float f = scale;
            if (!whole) {
                const int node = (ch * NC + c0 + c) / G;
                const int last = min(s.hist + node, s.L - 1) - k0 - 4 * g;   // the last key that the column sees
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[kt][i] = 16 * kt + i <= last ? x[kt][i] * scale : -INFINITY;
                f = 1.0f;   // (a masked score stays what it is under a scale of zero)
            }
            if constexpr (SUM) {
                const float here_lse = lse_s[ch % R][c0 + c], l = c0 + c < stop ? here_lse : INFINITY;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[kt][i] += fast_exp2(fmaf(x[kt][i], f, -l));
            } else {
                // exp2 of the scores as they are: while a column's sum lies well within fp32's
                // range, no maximum has to be taken off, which would not change its precision.
                float top = 0.0f;
                auto exps = [&]() {
                    float l[4];
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = fast_exp2(fmaf(x[kt][i], f, -top));
                            l[i] = kt == 0 ? e : l[i] + e;
                        }
                    return over_rows((l[0] + l[1]) + (l[2] + l[3]), [](float u, float v) { return u + v; });
                };
                float all = exps();
                if (__builtin_amdgcn_ballot_w64(!(all >= 0x1p-60f && all <= 0x1p100f)) != 0) {
                    float m = kNegBig;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) m = fmaxf(fmaxf(m, x[kt][i]), x[kt][i + 1]);
                    top = over_rows(m * f, [](float u, float v) { return fmaxf(u, v); });
                    all = exps();
                }
                const bool mine = g == (st & 3);
                top_of[st / 4] = mine ? top : top_of[st / 4];
                sum_of[st / 4] = mine ? all : sum_of[st / 4];
            }
        }
    }
    if (idle) return;
    if constexpr (!SUM) {
        store_chunk(chunks - 1);
    } else {
        float* mass = a.mass + n * a.mass_bs + kvh * a.mass_hs;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float t = group_sum<16>(sum[kt][i]);
                const int pos = k0 + 16 * kt + 4 * g + i;
                if (c == 0 && pos < s.L) mass[pos] += t;
            }
    }
}

// Per column: the log2-sum-exp2 over its key blocks, +inf for a column that sees
// no key (every weight is then zero).  Grid (groups of 16 columns, Hkv, N): 16 columns,
// 16 threads each, with four blocks in flight.
__global__ __launch_bounds__(256) void window_lse_kernel(WindowArgs a, int keys) {
    __shared__ float part_m[16][17], part_s[16][17];
    const int n = blockIdx.z, kvh = blockIdx.y, c = threadIdx.x & 15, t = threadIdx.x >> 4;
    const WindowSeq s = window_seq(a, n);
    const int nblk = (s.L + keys - 1) / keys, cols = s.P * (a.Hq / a.Hkv);
    const int64_t at = (int64_t)s.q0 * (a.Hq / a.Hkv), step = a.Hkv * a.cols;
    for (int c0 = 16 * blockIdx.x; c0 < cols; c0 += 16 * gridDim.x) {   // (uniform)
        const bool on = c0 + c < cols;
        const float* part = a.part + kvh * a.cols + at + (on ? c0 + c : c0);
        float M = -INFINITY, S = 0.0f;
        for (int j = t; j < nblk; j += 64) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = j + 16 * i < nblk ? part[(j + 16 * i) * step] : -INFINITY;
            const float mb = fmaxf(fmaxf(M, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
            const float base = mb == -INFINITY ? 0.0f : mb;   // (a score that is no number stays one in the sum)
            S *= fast_exp2(M - base);
#pragma unroll
            for (int i = 0; i < 4; ++i) S += fast_exp2(x[i] - base);
            M = mb;
        }
        __syncthreads();   // the columns before have been read
        part_m[c][t] = M;
        part_s[c][t] = S;
        __syncthreads();
        if (t == 0 && on) {
            for (int i = 1; i < 16; ++i) M = fmaxf(M, part_m[c][i]);
            const float base = M == -INFINITY ? 0.0f : M;
            float sum = 0.0f;
            for (int i = 0; i < 16; ++i) sum = fmaf(part_s[c][i], fast_exp2(part_m[c][i] - base), sum);
            a.lse[kvh * a.cols + at + c0 + c] = sum == 0.0f ? INFINITY : M + fast_log2(sum);
        }
    }
}

// Any head_dim up to 256, any page size and alignment: a wave per (row, query
// head) for the log-sum-exp, then a thread per (key, kv head) for the totals.
template <typename T>
__device__ inline float dot(const T* q, const T* k, int D) {
    float d0 = 0.0f, d1 = 0.0f, d2 = 0.0f, d3 = 0.0f;   // four sums, added pairwise
    int d = 0;
    for (; d + 3 < D; d += 4) {
        d0 = fmaf(Elem<T>::to_f32(q[d]), Elem<T>::to_f32(k[d]), d0);
        d1 = fmaf(Elem<T>::to_f32(q[d + 1]), Elem<T>::to_f32(k[d + 1]), d1);
        d2 = fmaf(Elem<T>::to_f32(q[d + 2]), Elem<T>::to_f32(k[d + 2]), d2);
        d3 = fmaf(Elem<T>::to_f32(q[d + 3]), Elem<T>::to_f32(k[d + 3]), d3);
    }
    for (; d < D; ++d) d0 = fmaf(Elem<T>::to_f32(q[d]), Elem<T>::to_f32(k[d]), d0);
    return (d0 + d1) + (d2 + d3);
}

template <typename T>
__device__ inline const T* key_row(const WindowArgs& a, int n, int kvh, int pos) {
    const int64_t phys = max(a.bt[(int64_t)n * a.max_blocks + pos / a.bs], 0);
    return reinterpret_cast<const T*>(a.k) + ((phys * a.bs + pos % a.bs) * a.Hkv + kvh) * a.D;
}

template <typename T>
__global__ __launch_bounds__(256) void window_lse_generic_kernel(WindowArgs a) {
    const int n = blockIdx.y, lane = threadIdx.x & 63, G = a.Hq / a.Hkv;
    const WindowSeq s = window_seq(a, n);
    for (int64_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < (int64_t)s.P * a.Hq; r += gridDim.x * 4) {
        const int64_t at = (int64_t)s.q0 * a.Hq + r;
        const int node = (int)(r / a.Hq), kvh = (int)(r - (int64_t)node * a.Hq) / G;
        const T* q = reinterpret_cast<const T*>(a.q) + at * a.D;
        const int stop = min(s.hist + node + 1, s.L);
        float M = -INFINITY, S = 0.0f;
        for (int j = lane; j < stop; j += 64) {
            const float x = dot(q, key_row<T>(a, n, kvh, j), a.D) * a.scale_log2;
            const float mb = fmaxf(M, x), base = mb == -INFINITY ? 0.0f : mb;
            S = S * fast_exp2(M - base) + fast_exp2(x - base);
            M = mb;
        }
        const float top = wave_max(M);
        S = wave_sum(S * fast_exp2(M - (top == -INFINITY ? 0.0f : top)));
        if (lane == 0) a.lse[at] = S == 0.0f ? INFINITY : top + fast_log2(S);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void window_sum_generic_kernel(WindowArgs a) {
    const int n = blockIdx.z, kvh = blockIdx.y, G = a.Hq / a.Hkv;
    const WindowSeq s = window_seq(a, n);
    for (int j = blockIdx.x * 256 + threadIdx.x; j < s.L; j += gridDim.x * 256) {
        const T* k = key_row<T>(a, n, kvh, j);
        float sum = 0.0f;
        for (int i = max(0, j - s.hist); i < s.P; ++i)
            for (int h = 0; h < G; ++h) {
                const int64_t at = (int64_t)(s.q0 + i) * a.Hq + kvh * G + h;
                sum += fast_exp2(dot(reinterpret_cast<const T*>(a.q) + at * a.D, k, a.D) * a.scale_log2 - a.lse[at]);
            }
        a.mass[n * a.mass_bs + kvh * a.mass_hs + j] += sum;
    }
}

bool tuned_shape(int D, int bs) { return bs == kPage && (D == 64 || D == 96 || D == 128 || D == 256); }

int keys_of(int dtype) { return dtype == LLKV_DTYPE_F32 ? wave_keys<float>() : wave_keys<_Float16>(); }

template <typename T, int D, int W>
void launch_waves(const WindowArgs& a, int max_q_len, hipStream_t st) {
    const dim3 grid((a.nblk + W - 1) / W, a.Hkv, a.N);
    const int lse_wgs = (int)std::min<int64_t>(((int64_t)max_q_len * (a.Hq / a.Hkv) + 15) / 16, 65535);
    window_kernel<T, D, W, false><<<grid, 64 * W, 0, st>>>(a);
    window_lse_kernel<<<dim3(lse_wgs, a.Hkv, a.N), 256, 0, st>>>(a, wave_keys<T>());
    window_kernel<T, D, W, true><<<grid, 64 * W, 0, st>>>(a);
}

// Eight waves share a work-group's rows where that leaves work-groups for every
// compute unit.
template <typename T, int D>
void launch_tuned(const WindowArgs& a, int max_q_len, hipStream_t st) {
    if ((int64_t)a.nblk * a.Hkv * a.N >= 8ll * device_cus()) launch_waves<T, D, 8>(a, max_q_len, st);
    else launch_waves<T, D, 4>(a, max_q_len, st);
}

template <typename T>
void launch_window(const WindowArgs& a, int max_q_len, bool tuned, hipStream_t st) {
    if (tuned) {
        if (a.D == 64) launch_tuned<T, 64>(a, max_q_len, st);
        else if (a.D == 96) launch_tuned<T, 96>(a, max_q_len, st);
        else if (a.D == 128) launch_tuned<T, 128>(a, max_q_len, st);
        else launch_tuned<T, 256>(a, max_q_len, st);
        return;
    }
    const int lse_wgs = (int)std::min<int64_t>(((int64_t)max_q_len * a.Hq + 3) / 4, 65535);
    window_lse_generic_kernel<T><<<dim3(lse_wgs, a.N), 256, 0, st>>>(a);
    const int blocks = std::max(1, std::min((a.max_len + 255) / 256, 65535));
    window_sum_generic_kernel<T><<<dim3(blocks, a.Hkv, a.N), 256, 0, st>>>(a);
}

struct WindowPlan {
    int nblk;
    size_t lse, total;
};

WindowPlan window_plan(int64_t total_q, int Hq, int max_len, int dtype) {
    WindowPlan p;
    const int keys = keys_of(dtype);
    p.nblk = (int)std::max<int64_t>(1, ((int64_t)max_len + keys - 1) / keys);
    const size_t rows = (size_t)total_q * Hq * sizeof(float);
    p.lse = (rows * p.nblk + 255) & ~(size_t)255;
    p.total = p.lse + rows;
    return p;
}

}  // namespace
}  // namespace llkv

using namespace llkv;

extern "C" size_t llkv_paged_window_mass_workspace_size(int total_q, int num_q_heads, int max_seq_len, int dtype) {
    if (total_q <= 0 || num_q_heads <= 0 || max_seq_len < 0 || dtype_bytes(dtype) == 0) return 0;
    return window_plan(total_q, num_q_heads, max_seq_len, dtype).total;
}

extern "C" int llkv_paged_window_mass(float* mass, int64_t mass_seq_stride, int64_t mass_head_stride, const void* q,
                                      const void* k_pool, const int* block_table, int max_blocks_per_seq,
                                      const int* cu_q, const int* seq_lens, int num_seqs, int total_q, int max_q_len,
                                      int max_seq_len, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                      float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "llkv_paged_window_mass";
    if (num_seqs == 0 || total_q == 0) return LLKV_OK;
    if (num_seqs < 0 || total_q < 0 || max_q_len <= 0 || max_seq_len < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
        head_dim <= 0 || block_size <= 0 || max_blocks_per_seq <= 0)
        return set_error(LLKV_ERR_INVALID, "%s: bad shape arguments", fn);
    if (head_dim > 256) return set_error(LLKV_ERR_UNSUPPORTED, "%s: head_dim too large (%d > 256)", fn, head_dim);
    if (num_q_heads % num_kv_heads != 0)
        return set_error(LLKV_ERR_INVALID, "%s: num_q_heads %d not a multiple of num_kv_heads %d", fn, num_q_heads,
                         num_kv_heads);
    if (dtype_bytes(dtype) == 0) return set_error(LLKV_ERR_INVALID, "%s: unsupported dtype %d", fn, dtype);
    if ((int64_t)max_blocks_per_seq * block_size > INT32_MAX - 1024 || (int64_t)num_seqs * max_blocks_per_seq > INT32_MAX ||
        num_kv_heads > 65535 || (int64_t)total_q * num_q_heads > INT32_MAX - 256)
        return set_error(LLKV_ERR_UNSUPPORTED, "%s: block table or rows too large", fn);
    if (!mass || !q || !k_pool || !block_table || !cu_q || !seq_lens)
        return set_error(LLKV_ERR_INVALID, "%s: null pointer", fn);
    if (mass_head_stride < max_seq_len || (num_seqs > 1 && mass_seq_stride < (int64_t)num_kv_heads * mass_head_stride))
        return set_error(LLKV_ERR_INVALID, "%s: totals of %lld keys a head for up to %d", fn,
                         (long long)mass_head_stride, max_seq_len);
    const WindowPlan p = window_plan(total_q, num_q_heads, max_seq_len, dtype);
    if (!workspace || workspace_bytes < p.total)
        return set_error(LLKV_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, p.total);
    if (((uintptr_t)workspace & 15) != 0) return set_error(LLKV_ERR_INVALID, "%s: workspace not 16-byte aligned", fn);
    WindowArgs a = {};
    a.q = q;
    a.k = k_pool;
    a.cu_q = cu_q;
    a.max_blocks = max_blocks_per_seq;
    a.Hq = num_q_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.bs = block_size;
    a.max_len = max_seq_len;
    a.scale_log2 = scale * kLog2e;
    a.nblk = p.nblk;
    a.cols = (int64_t)total_q * (num_q_heads / num_kv_heads);
    a.part = reinterpret_cast<float*>(workspace);
    a.lse = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + p.lse);
    a.mass_bs = mass_seq_stride;
    a.mass_hs = mass_head_stride;
    const bool tuned = tuned_shape(head_dim, block_size) && (((uintptr_t)q | (uintptr_t)k_pool) & 15) == 0;
    hipStream_t st = (hipStream_t)stream;
    constexpr int kMost = 32768;   // sequences per launch (a grid's extent in z)
    for (int n0 = 0; n0 < num_seqs; n0 += kMost) {
        a.N = std::min(num_seqs - n0, kMost);
        a.bt = block_table + (int64_t)n0 * max_blocks_per_seq;
        a.cu_q = cu_q + n0;
        a.lens = seq_lens + n0;
        a.mass = mass + n0 * mass_seq_stride;
        if (dtype == LLKV_DTYPE_F32) launch_window<float>(a, max_q_len, tuned, st);
        else if (dtype == LLKV_DTYPE_F16) launch_window<_Float16>(a, max_q_len, tuned, st);
        else launch_window<bf16_t>(a, max_q_len, tuned, st);
    }
    return check_launch(fn);
}
