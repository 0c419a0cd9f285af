// rules_mi355.hip — decoding rules on logits for MI355X (gfx950): penalties for repeated tokens, biases and masks of
// allowed tokens, applied on the way to the argmax and its log-probability, or written out.
//
// The reference's searches take the maximum of the raw logits (src/rnnt/model.py:152-153,
// src/rnnt/beam_searcher.py:91-93).  Here the logits of a row pass once through registers:
//     c = count of v in the row's history
//     v' = c > 0 ? (v > 0 ? v / r : v r) : v;   v' -= f c;   v' -= p (c > 0);   v' += bias;   not allowed: -inf
// in fp32 and in this order, so that a near-tie is decided as the formula decides it.
// One workgroup per row (argmax; per kTileSplit columns where a row is longer than kTilePick, joined by a second launch)
// or per kTileOut columns of a row (written out).  How often each token stands in the
// history is counted first, in LDS, 16 bits per token (integer LDS atomics: any order, the same counts).
// Rows are read in the 16-byte pieces that memory has, wherever a row begins (an odd vocabulary puts most rows off 16
// bytes): piece c of a row holds its columns c E - o .. c E - o + E - 1, E elements to a piece, o the row's first element
// within its piece; the counters are numbered the same way.  Only the two pieces at a row's ends are read by elements.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/rnnt_mi355.h"
#include "elem_types.h"

namespace {

using namespace rnnt_mi355_detail;

constexpr int kTilePick = 16384;  // columns whose counts are in LDS at once: 32 KiB
constexpr int kTileSplit = 4096;  // columns per workgroup where a row is shared out
constexpr int kTileOut = 4096;    // columns that a workgroup writes
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16-byte loads need 4-byte alignment only

// running {max, sum of 2^((x - max) log2e)} of two parts
__device__ __forceinline__ void join_sums(float &m, float &s, float mo, float so) {
    const float mn = fmaxf(m, mo);
    const float a = (s == 0.0f || m == -INFINITY) ? 0.0f : s * __builtin_amdgcn_exp2f((m - mn) * kLog2e);
    const float b = (so == 0.0f || mo == -INFINITY) ? 0.0f : so * __builtin_amdgcn_exp2f((mo - mn) * kLog2e);
    s = a + b;
    m = mn;
}

// A value and its index as one number whose maximum is the argmax: NaN above all, the two zeros equal, the lower index
// first among equals.
__device__ __forceinline__ unsigned long long rank_of(float v, int i) {
    const unsigned bits = __float_as_uint(v + 0.f);
    const unsigned order = v != v ? 0xffffffffu : (bits & 0x80000000u ? ~bits : bits | 0x80000000u);
    return (unsigned long long)order << 32 | (unsigned)~i;
}

template <typename DT>
struct RowRules {
    static constexpr int E = DT::EPC;
    typedef typename DT::elem elem;
    struct Piece {
        float x[E], bias[E];
        unsigned allowed;
    };
    const elem *row;          // column 0
    int V, off;               // off: column 0's place in its piece
    const float *bias;        // of the context; NULL: none
    const unsigned *allowed;  // NULL: all
    float repetition, presence, frequency;

    __device__ __forceinline__ int pieces() const { return (off + V + E - 1) / E; }
    __device__ __forceinline__ bool whole(int c) const { return c * E >= off && c * E - off + E <= V; }

    __device__ __forceinline__ void load(int c, Piece &p) const {
        const int v0 = c * E - off;
        if (whole(c)) {
            DT::unpack(reinterpret_cast<const u32x4 *>(row - off)[c], p.x);
#pragma unroll
            for (int j = 0; j < E; j += 4) {
                f32x4_any b = {0.f, 0.f, 0.f, 0.f};
                if (bias) b = *reinterpret_cast<const f32x4_any *>(bias + v0 + j);
                p.bias[j] = b.x;
                p.bias[j + 1] = b.y;
                p.bias[j + 2] = b.z;
                p.bias[j + 3] = b.w;
            }
            p.allowed = ~0u;
            if (allowed) {  // E bits from bit v0 % 32 on, perhaps of two words
                const int w = v0 >> 5, last = (v0 + E - 1) >> 5;
                p.allowed = (unsigned)(((unsigned long long)allowed[last] << 32 | allowed[w]) >> (v0 & 31));
                if (last == w) p.allowed = allowed[w] >> (v0 & 31);
            }
        } else {
            p.allowed = 0u;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int v = v0 + j;
                const bool in = v >= 0 && v < V;
                p.x[j] = in ? DT::to_float(row[v]) : 0.f;
                p.bias[j] = in && bias ? bias[v] : 0.f;
                if (in && (allowed == nullptr || (allowed[v >> 5] >> (v & 31) & 1u))) p.allowed |= 1u << j;
            }
        }
    }
    // count2: the counts of the piece's columns, two to a word
    __device__ __forceinline__ void apply(Piece &p, const unsigned (&count2)[E / 2]) const {
        unsigned any = 0u;
#pragma unroll
        for (int j = 0; j < E / 2; ++j) any |= count2[j];
        if (any) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const unsigned count = j & 1 ? count2[j / 2] >> 16 : count2[j / 2] & 0xffffu;
                if (count) {
                    float v = p.x[j];
                    v = v > 0.f ? v / repetition : v * repetition;
                    v = v - frequency * (float)count;
                    p.x[j] = v - presence;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float v = p.x[j] + p.bias[j];
            p.x[j] = p.allowed >> j & 1u ? v : -INFINITY;
        }
    }
};

template <typename DT>
__device__ __forceinline__ RowRules<DT> rules_of_row(const typename DT::elem *x, int V, const rnntRules &rules, int r, int context) {
    RowRules<DT> q;
    q.row = x + (size_t)r * V;
    q.V = V;
    q.off = (int)((reinterpret_cast<uintptr_t>(q.row) & 15u) / sizeof(typename DT::elem));
    q.bias = rules.bias ? rules.bias + (size_t)context * rules.bias_stride : nullptr;
    q.allowed = rules.allowed ? reinterpret_cast<const unsigned *>(rules.allowed) + (size_t)context * rules.allowed_stride : nullptr;
    q.repetition = rules.repetition_penalty;
    q.presence = rules.presence_penalty;
    q.frequency = rules.frequency_penalty;
    return q;
}

__device__ __forceinline__ int history_length(const rnntRules &rules, int context) {
    if (rules.history == nullptr) return 0;
    const int n = rules.history_lens ? rules.history_lens[context] : rules.history_stride;
    return n < 0 ? 0 : (n > rules.history_stride ? rules.history_stride : n);
}

// counts of the columns [first, first + slots) (numbered as in pieces: column + off), all threads of the workgroup
__device__ __forceinline__ void count_history(unsigned *s_count, const int *history, int n, int V, int off, int first, int slots) {
    for (int i = threadIdx.x; i < slots / 2; i += blockDim.x) s_count[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int v = history[i];
        if (v < 0 || v >= V) continue;
        const int k = v + off - first;
        if (k >= 0 && k < slots) atomicAdd(&s_count[k >> 1], 1u << ((k & 1) * 16));
    }
    __syncthreads();
}

template <typename DT>
__device__ __forceinline__ void read_counts(const unsigned *s_count, bool counted, int slot, unsigned (&count2)[DT::EPC / 2]) {
    if constexpr (DT::EPC == 8) {
        u32x4 w = {0u, 0u, 0u, 0u};
        if (counted) w = *reinterpret_cast<const u32x4 *>(s_count + slot / 2);
        count2[0] = w.x;
        count2[1] = w.y;
        count2[2] = w.z;
        count2[3] = w.w;
    } else {
        u32x2 w = {0u, 0u};
        if (counted) w = *reinterpret_cast<const u32x2 *>(s_count + slot / 2);
        count2[0] = w.x;
        count2[1] = w.y;
    }
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_(unsigned v) {
    return __builtin_amdgcn_update_dpp(0u, v, CTRL, 0xf, 0xf, true);
}
// what another lane of the wave holds, over the six steps of a reduction (lane xor 1, 2, 7, row rotation by 8, xor 16, 32)
template <int STEP>
__device__ __forceinline__ unsigned from_lane(unsigned v) {
    if constexpr (STEP == 0) return dpp_<0xB1>(v);
    if constexpr (STEP == 1) return dpp_<0x4E>(v);
    if constexpr (STEP == 2) return dpp_<0x141>(v);
    if constexpr (STEP == 3) return dpp_<0x128>(v);
    if constexpr (STEP == 4) return __shfl_xor(v, 16, kWave);
    return __shfl_xor(v, 32, kWave);
}
template <int STEP, int STEPS>
__device__ __forceinline__ void reduce_lanes(unsigned long long &rank, float &m, float &s, bool sums) {
    if constexpr (STEP < STEPS) {
        const unsigned long long other = (unsigned long long)from_lane<STEP>((unsigned)(rank >> 32)) << 32 | from_lane<STEP>((unsigned)rank);
        rank = other > rank ? other : rank;
        if (sums) {
            const float mo = __uint_as_float(from_lane<STEP>(__float_as_uint(m))), so = __uint_as_float(from_lane<STEP>(__float_as_uint(s)));
            join_sums(m, s, mo, so);
        }
        reduce_lanes<STEP + 1, STEPS>(rank, m, s, sums);
    }
}

struct RowPart {  // of a row's argmax and sum of exponentials
    unsigned long long rank;
    float m, s;
};

// the answer of a row: m - m is NaN for an infinite maximum, as in torch; a NaN among the values is the rank's maximum
__device__ __forceinline__ void store_answer(const RowPart &p, int *out, float *logp, int r) {
    out[r] = (int)~(unsigned)p.rank;
    if (logp == nullptr) return;
    const bool nan = (unsigned)(p.rank >> 32) == 0xffffffffu;
    logp[r] = nan ? __builtin_nanf("") : (p.m - p.m) - kLn2 * __builtin_amdgcn_logf(p.s);
}

// Bound by latency: one load of a thread's two pieces behind the counting, then the reduction.  512 rows of 4232 fp32 logits
// (16 contexts with history, bias and mask) 8 us, one row of 5455 fp16 logits 6 us (10 us by elements, with the whole
// row off 16 bytes).
template <typename DT, bool SPLIT>
__global__ __launch_bounds__(1024) void row_rules_kernel(const typename DT::elem *__restrict__ x, int V, const rnntRules rules,
                                                         int rows_per_context, int *__restrict__ out, float *__restrict__ logp,
                                                         int splits, RowPart *__restrict__ parts) {
    constexpr int E = DT::EPC, kTile = SPLIT ? kTileSplit : kTilePick;
    extern __shared__ u32x4 s_words[];  // the counts of the row's (the part's) columns: no more than it has, so that short
                                        // rows share a CU with many others
    __shared__ unsigned long long s_rank[16];
    __shared__ float s_max[16], s_sum[16];
    unsigned *s_count = reinterpret_cast<unsigned *>(s_words);
    const int r = SPLIT ? blockIdx.x / splits : blockIdx.x, context = r / rows_per_context;
    const int first = SPLIT ? (int)(blockIdx.x - (unsigned)r * splits) * kTile : 0;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, threads = blockDim.x;
    const RowRules<DT> q = rules_of_row<DT>(x, V, rules, r, context);
    const int *history = rules.history ? rules.history + (size_t)context * rules.history_stride : nullptr;
    const int n_hist = history_length(rules, context);
    const int pieces = q.pieces(), stop = first / E + kTile / E < pieces ? first / E + kTile / E : pieces;

    float best = -INFINITY, m = -INFINITY, s = 0.f;
    int at = 0x7fffffff;
    typename RowRules<DT>::Piece next;
    int c = first / E + threadIdx.x;
    if (c < stop) q.load(c, next);  // (before the counting: its latency is the counting's)
    if (n_hist > 0) count_history(s_count, history, n_hist, V, q.off, first, SPLIT ? kTile : (stop * E + 7) & ~7);
    for (; c < stop; c += threads) {
        typename RowRules<DT>::Piece p = next;
        if (c + threads < stop) q.load(c + threads, next);
        unsigned count2[E / 2];
        read_counts<DT>(s_count, n_hist > 0, c * E - first, count2);
        q.apply(p, count2);
        const int v0 = c * E - q.off;
        float cm = -INFINITY;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            // greater, or the first NaN; columns outside the row are -inf and never taken
            const bool take = !(p.x[j] <= best) && best == best;
            best = take ? p.x[j] : best;
            at = take ? v0 + j : at;
            cm = fmaxf(cm, p.x[j]);
        }
        const float mn = fmaxf(m, cm);
        if (logp != nullptr && mn != -INFINITY) {  // (all -inf so far: nothing to add)
            float acc = s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f((m - mn) * kLog2e);
#pragma unroll
            for (int j = 0; j < E; ++j) acc += __builtin_amdgcn_exp2f((p.x[j] - mn) * kLog2e);
            s = acc;
            m = mn;
        }
    }
    // (a thread that saw only -inf has no index: token 0 then is the answer, as of a row of -inf)
    unsigned long long rank = rank_of(best, at == 0x7fffffff ? 0 : at);
    const bool sums = logp != nullptr;
    reduce_lanes<0, 6>(rank, m, s, sums);
    if (lane == 0) {
        s_rank[wave] = rank;
        s_max[wave] = m;
        s_sum[wave] = s;
    }
    __syncthreads();
    if (wave != 0) return;
    const int w = lane & 15;  // (the sixteen lanes of a row: at most as many waves)
    const bool held = w < threads / kWave;
    rank = held ? s_rank[w] : 0ull;
    m = held ? s_max[w] : -INFINITY;
    s = held ? s_sum[w] : 0.f;
    reduce_lanes<0, 4>(rank, m, s, sums);
    if (lane != 0) return;
    const RowPart part = {rank, m, s};
    if (SPLIT)
        parts[blockIdx.x] = part;
    else
        store_answer(part, out, logp, r);
}

// the parts of a shared-out row, a wave per row
__global__ __launch_bounds__(kWave) void row_rules_join_kernel(const RowPart *__restrict__ parts, int splits, int *__restrict__ out,
                                                               float *__restrict__ logp) {
    unsigned long long rank = 0ull;
    float m = -INFINITY, s = 0.f;
    for (int k = threadIdx.x; k < splits; k += kWave) {
        const RowPart p = parts[(size_t)blockIdx.x * splits + k];
        rank = p.rank > rank ? p.rank : rank;
        join_sums(m, s, p.m, p.s);
    }
    reduce_lanes<0, 6>(rank, m, s, true);
    if (threadIdx.x == 0) store_answer(RowPart{rank, m, s}, out, logp, blockIdx.x);
}

// Bound by memory once there are rows enough: 64 rows of 70 001 bf16 logits 11 us (37 MB with bias, mask and histories:
// 3.4 TB/s); a workgroup per row, by elements, took 38.
template <typename DT>
__global__ __launch_bounds__(256) void process_logits_kernel(const typename DT::elem *x, int V, const rnntRules rules,
                                                             int rows_per_context, typename DT::elem *processed, int tiles) {
    constexpr int E = DT::EPC;
    __shared__ u32x4 s_words[kTileOut / 8];
    unsigned *s_count = reinterpret_cast<unsigned *>(s_words);
    const int r = blockIdx.x / tiles, first = (int)(blockIdx.x - (unsigned)r * tiles) * kTileOut, context = r / rows_per_context;
    const RowRules<DT> q = rules_of_row<DT>(x, V, rules, r, context);
    const int n_hist = history_length(rules, context);
    const int pieces = q.pieces(), stop = first / E + kTileOut / E < pieces ? first / E + kTileOut / E : pieces;
    typename DT::elem *dst = processed + (size_t)r * V;
    const bool same = ((reinterpret_cast<uintptr_t>(dst) ^ reinterpret_cast<uintptr_t>(q.row)) & 15u) == 0;
    typename RowRules<DT>::Piece next;
    int c = first / E + threadIdx.x;
    if (c < stop) q.load(c, next);
    if (n_hist > 0)
        count_history(s_count, rules.history + (size_t)context * rules.history_stride, n_hist, V, q.off, first, kTileOut);
    for (; c < stop; c += 256) {
        typename RowRules<DT>::Piece p = next;
        if (c + 256 < stop) q.load(c + 256, next);
        unsigned count2[E / 2];
        read_counts<DT>(s_count, n_hist > 0, c * E - first, count2);
        q.apply(p, count2);
        const int v0 = c * E - q.off;
        if (same && q.whole(c)) {
            reinterpret_cast<u32x4 *>(dst - q.off)[c] = DT::pack(p.x);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (v0 + j >= 0 && v0 + j < V) dst[v0 + j] = DT::from_float(p.x[j]);
        }
    }
}

// (a launch has less than 2^32 threads: at most 512 to 4096 columns where there are many rows)
inline bool rows_ok(int rows, int V) {
    return rows >= 1 && V >= 1 && V <= 0x40000000 && (long long)rows * (V / kTileSplit + 2) < (1ll << 23);
}

bool rules_ok(const rnntRules *r, int rows, int V) {
    if (r == nullptr || r->contexts < 1 || rows % r->contexts != 0) return false;
    if (r->history && (r->history_stride < 1 || r->history_stride > RNNT_MAX_HISTORY)) return false;
    if (r->bias && r->bias_stride != 0 && r->bias_stride < V) return false;
    if (r->allowed && r->allowed_stride != 0 && r->allowed_stride < (V + 31) / 32) return false;
    return r->repetition_penalty > 0.f && r->repetition_penalty < INFINITY && r->presence_penalty == r->presence_penalty &&
           r->frequency_penalty == r->frequency_penalty;
}

// Threads of a row's workgroup: one to three pieces each.  1058 pieces (4232 fp32 logits), 512 rows: 8.9, 8.0 and 8.8 us with
// 256, 512 and 1024 threads; 682 pieces, one row: 7.3, 6.0 and 5.8; 2000 pieces, 16 rows: 12.8, 8.9 and 8.1.
inline int pick_threads(int rows, int pieces) { return pieces <= 512 ? 256 : (pieces <= 1536 || rows > 256 ? 512 : 1024); }

// 0: a workgroup per row; otherwise workgroups per row.  One workgroup reads a row of 70 001 logits in 24 us whether there
// is one row or 64; shared out among 18 and joined by a second launch one fp32 row takes 11 us, 64 bf16 rows 15 us.
inline int pick_splits(int V, int per_piece) {
    const long long slots = (long long)V + per_piece - 1;  // (a row's pieces may begin up to per_piece - 1 before it)
    return slots <= kTilePick ? 0 : (int)((slots + kTileSplit - 1) / kTileSplit);
}

template <typename DT>
rnntStatus_t launch_pick(const void *x, int rows, int V, const rnntRules &r, int *out, float *logp, void *workspace, hipStream_t st) {
    typedef typename DT::elem E;
    const int splits = pick_splits(V, DT::EPC);
    if (splits == 0) {
        const size_t counts = r.history ? (((size_t)V + 2 * DT::EPC + 7) & ~(size_t)7) * 2 : 0;  // (whole pieces at both ends)
        hipLaunchKernelGGL((row_rules_kernel<DT, false>), dim3(rows), dim3(pick_threads(rows, V / DT::EPC + 1)), counts, st,
                           static_cast<const E *>(x), V, r, rows / r.contexts, out, logp, 1, static_cast<RowPart *>(nullptr));
    } else {
        if (workspace == nullptr || !aligned16(workspace)) return RNNT_STATUS_INVALID_VALUE;
        RowPart *parts = static_cast<RowPart *>(workspace);
        hipLaunchKernelGGL((row_rules_kernel<DT, true>), dim3((unsigned)(rows * (long long)splits)), dim3(512), kTileSplit * 2, st,
                           static_cast<const E *>(x), V, r, rows / r.contexts, out, logp, splits, parts);
        hipLaunchKernelGGL(row_rules_join_kernel, dim3(rows), dim3(kWave), 0, st, static_cast<const RowPart *>(parts), splits, out, logp);
    }
    return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED;
}

template <typename DT>
rnntStatus_t launch_process(const void *x, int rows, int V, const rnntRules &r, void *processed, hipStream_t st) {
    typedef typename DT::elem E;
    const long long tiles = ((long long)V + DT::EPC - 1 + kTileOut - 1) / kTileOut;  // (a row's pieces may begin up to EPC - 1 before it)
    hipLaunchKernelGGL((process_logits_kernel<DT>), dim3((unsigned)(tiles * rows)), dim3(256), 0, st, static_cast<const E *>(x), V, r,
                       rows / r.contexts, static_cast<E *>(processed), (int)tiles);
    return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED;
}

}  // namespace

extern "C" {

rnntStatus_t rnnt_row_rules_workspace_size(int rows, int V, rnntDtype_t dtype, size_t *size_bytes) {
    if (size_bytes == nullptr || !rows_ok(rows, V) || dtype < RNNT_DTYPE_F32 || dtype > RNNT_DTYPE_F16)
        return RNNT_STATUS_INVALID_VALUE;
    *size_bytes = (size_t)rows * pick_splits(V, dtype == RNNT_DTYPE_F32 ? F32::EPC : F16::EPC) * sizeof(RowPart);
    return RNNT_STATUS_SUCCESS;
}

rnntStatus_t rnnt_row_rules(const void *x, int rows, int V, rnntDtype_t dtype, const rnntRules *rules, int *out, float *logp,
                            void *workspace, void *stream) {
    if (x == nullptr || out == nullptr || !rows_ok(rows, V) || !rules_ok(rules, rows, V)) return RNNT_STATUS_INVALID_VALUE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RNNT_DTYPE_F32: return launch_pick<F32>(x, rows, V, *rules, out, logp, workspace, st);
        case RNNT_DTYPE_BF16: return launch_pick<BF16>(x, rows, V, *rules, out, logp, workspace, st);
        case RNNT_DTYPE_F16: return launch_pick<F16>(x, rows, V, *rules, out, logp, workspace, st);
        default: return RNNT_STATUS_INVALID_VALUE;
    }
}

rnntStatus_t rnnt_process_logits(const void *x, int rows, int V, rnntDtype_t dtype, const rnntRules *rules, void *processed,
                                 void *stream) {
    if (x == nullptr || processed == nullptr || !rows_ok(rows, V) || !rules_ok(rules, rows, V)) return RNNT_STATUS_INVALID_VALUE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RNNT_DTYPE_F32: return launch_process<F32>(x, rows, V, *rules, processed, st);
        case RNNT_DTYPE_BF16: return launch_process<BF16>(x, rows, V, *rules, processed, st);
        case RNNT_DTYPE_F16: return launch_process<F16>(x, rows, V, *rules, processed, st);
        default: return RNNT_STATUS_INVALID_VALUE;
    }
}

}  // extern "C"
