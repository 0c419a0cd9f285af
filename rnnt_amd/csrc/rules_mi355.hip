// rules_mi355.hip — decoding rules on logits for MI355X (gfx950): penalties for repeated tokens, biases and masks of
// allowed tokens, applied on the way to the argmax and its log-probability, or written out.
//
// The reference's searches take the maximum of the raw logits (src/rnnt/model.py:152-153,
// src/rnnt/beam_searcher.py:91-93).  Here the logits of a row pass once through registers:
//     c = count of v in the row's history
//     v' = c > 0 ? (v > 0 ? v / r : v r) : v;   v' -= f c;   v' -= p (c > 0);   v' += bias;   not allowed: -inf
// in fp32 and in this order, so that a near-tie is decided as the formula decides it.
// One workgroup per row.  How often each token stands in the history is counted first, in LDS, 16 bits per token and
// kTile tokens at a time (integer LDS atomics: any order, the same counts); then the tile's logits are read.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/rnnt_mi355.h"
#include "elem_types.h"

namespace {

using namespace rnnt_mi355_detail;

constexpr int kTile = 16384;  // columns whose counts are in LDS at once: 32 KiB
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct Best {
    float v;  // NaN mapped to +inf
    int nan;  // 1 if the value was a NaN (ranks above +inf)
    int i;
};
__device__ __forceinline__ bool better(const Best &a, const Best &b) {  // a beats b; the lower index wins a tie
    if (a.nan != b.nan) return a.nan > b.nan;
    if (a.v != b.v) return a.v > b.v;
    return a.i < b.i;
}

// running {max, sum of 2^((x - max) log2e)} of two parts, the first part's share added first
__device__ __forceinline__ void join_sums(float &m, float &s, float mo, float so) {
    const float mn = fmaxf(m, mo);
    const float a = (s == 0.0f || m == -INFINITY) ? 0.0f : s * __builtin_amdgcn_exp2f((m - mn) * kLog2e);
    const float b = (so == 0.0f || mo == -INFINITY) ? 0.0f : so * __builtin_amdgcn_exp2f((mo - mn) * kLog2e);
    s = a + b;
    m = mn;
}

struct RowContext {
    const float *bias;        // NULL: none
    const unsigned *allowed;  // NULL: all
    float repetition, presence, frequency;
    __device__ __forceinline__ float apply(float v, unsigned count, float bias_v, bool ok) const {
        if (count) {
            const float c = (float)count;
            v = v > 0.f ? v / repetition : v * repetition;
            v = v - frequency * c;
            v = v - presence;
        }
        v = v + bias_v;
        return ok ? v : -INFINITY;
    }
};

// VEC: 16-byte pieces (rows of x, of the result and of the bias start on 16 bytes); otherwise element by element
template <typename DT, int VEC, bool PICK>
__global__ __launch_bounds__(1024) void row_rules_kernel(const typename DT::elem *x, int rows, int V,
                                                         const rnntRules rules, int rows_per_context, int *__restrict__ out,
                                                         float *__restrict__ logp, typename DT::elem *processed) {
    typedef typename DT::elem E;
    __shared__ unsigned s_count[kTile / 2];
    __shared__ Best s_best[16];
    __shared__ float s_max[16], s_sum[16];
    const int r = blockIdx.x, context = r / rows_per_context;
    const int tid = threadIdx.x, threads = blockDim.x;
    const int lane = tid & (kWave - 1), wave = tid / kWave;
    const E *row = x + (size_t)r * V;
    E *dst = PICK ? nullptr : processed + (size_t)r * V;
    const int *history = rules.history ? rules.history + (size_t)context * rules.history_stride : nullptr;
    int n_hist = 0;
    if (history) {
        n_hist = rules.history_lens ? rules.history_lens[context] : rules.history_stride;
        n_hist = n_hist < 0 ? 0 : (n_hist > rules.history_stride ? rules.history_stride : n_hist);
    }
    const RowContext ctx = {rules.bias ? rules.bias + (size_t)context * rules.bias_stride : nullptr,
                            rules.allowed ? reinterpret_cast<const unsigned *>(rules.allowed) + (size_t)context * rules.allowed_stride
                                          : nullptr,
                            rules.repetition_penalty, rules.presence_penalty, rules.frequency_penalty};
    Best best = {-INFINITY, 0, 0x7fffffff};
    float m = -INFINITY, s = 0.f;
    for (int c0 = 0; c0 < V; c0 += kTile) {
        const int cols = V - c0 < kTile ? V - c0 : kTile;
        if (n_hist > 0) {  // (the same for the whole workgroup)
            __syncthreads();
            for (int i = tid; i < (cols + 1) / 2; i += threads) s_count[i] = 0;
            __syncthreads();
            for (int i = tid; i < n_hist; i += threads) {
                const int k = history[i] - c0;
                if (history[i] >= 0 && k >= 0 && k < cols) atomicAdd(&s_count[k >> 1], 1u << ((k & 1) * 16));
            }
            __syncthreads();
        }
        for (int k = tid * VEC; k < cols; k += threads * VEC) {
            float f[VEC], bias[VEC];
            unsigned count[VEC], ok = ~0u;
            const int v0 = c0 + k;
            if constexpr (VEC == 1) {
                f[0] = DT::to_float(row[v0]);
                bias[0] = ctx.bias ? ctx.bias[v0] : 0.f;
                count[0] = n_hist > 0 ? (s_count[k >> 1] >> ((k & 1) * 16)) & 0xffffu : 0u;
                if (ctx.allowed) ok = ctx.allowed[v0 >> 5] >> (v0 & 31);
            } else {
                DT::unpack(reinterpret_cast<const u32x4 *>(row)[v0 / VEC], f);
#pragma unroll
                for (int j = 0; j < VEC; j += 4) {
                    u32x4 raw = {0u, 0u, 0u, 0u};
                    if (ctx.bias) raw = *reinterpret_cast<const u32x4 *>(ctx.bias + v0 + j);
                    bias[j] = __uint_as_float(raw.x);
                    bias[j + 1] = __uint_as_float(raw.y);
                    bias[j + 2] = __uint_as_float(raw.z);
                    bias[j + 3] = __uint_as_float(raw.w);
                }
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    const unsigned both = n_hist > 0 ? s_count[(k + j) >> 1] : 0u;
                    count[j] = both & 0xffffu;
                    count[j + 1] = both >> 16;
                }
                if (ctx.allowed) ok = ctx.allowed[v0 >> 5] >> (v0 & 31);  // (VEC divides 32)
            }
            float cm = -INFINITY;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                f[j] = ctx.apply(f[j], count[j], bias[j], (ok >> j) & 1u);
                if (PICK) {
                    const Best cand = {f[j] != f[j] ? INFINITY : f[j], f[j] != f[j] ? 1 : 0, v0 + j};
                    if (better(cand, best)) best = cand;
                    cm = fmaxf(cm, f[j]);
                }
            }
            if (PICK) {
                const float mn = fmaxf(m, cm);
                if (logp != nullptr && mn != -INFINITY) {  // (all -inf so far: nothing to add)
                    float acc = s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f((m - mn) * kLog2e);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc += __builtin_amdgcn_exp2f((f[j] - mn) * kLog2e);
                    s = acc;
                    m = mn;
                }
            } else if constexpr (VEC == 1) {
                dst[v0] = DT::from_float(f[0]);
            } else {
                reinterpret_cast<u32x4 *>(dst)[v0 / VEC] = DT::pack(f);
            }
        }
    }
    if (!PICK) return;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        Best o;
        o.v = __shfl_xor(best.v, off, kWave);
        o.nan = __shfl_xor(best.nan, off, kWave);
        o.i = __shfl_xor(best.i, off, kWave);
        if (better(o, best)) best = o;
    }
    if (logp != nullptr) {
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            float mo = __shfl_xor(m, off, kWave), so = __shfl_xor(s, off, kWave);
            if (lane & off) {  // both lanes of a pair add the lower lane's share first
                join_sums(mo, so, m, s);
                m = mo;
                s = so;
            } else {
                join_sums(m, s, mo, so);
            }
        }
    }
    if (lane == 0) {
        s_best[wave] = best;
        s_max[wave] = m;
        s_sum[wave] = s;
    }
    __syncthreads();
    if (tid != 0) return;
    for (int w = 1; w < threads / kWave; ++w) {
        if (better(s_best[w], best)) best = s_best[w];
        if (logp != nullptr) join_sums(m, s, s_max[w], s_sum[w]);
    }
    out[r] = best.i;
    if (logp == nullptr) return;
    const float mm = best.nan ? __builtin_nanf("") : best.v;
    logp[r] = (mm - mm) - kLn2 * __builtin_amdgcn_logf(s);  // mm - mm: NaN for an infinite maximum, as torch
}

bool rules_ok(const rnntRules *r, int rows, int V) {
    if (r == nullptr || r->contexts < 1 || rows % r->contexts != 0) return false;
    if (r->history && (r->history_stride < 1 || r->history_stride > RNNT_MAX_HISTORY)) return false;
    if (r->bias && r->bias_stride != 0 && r->bias_stride < V) return false;
    if (r->allowed && r->allowed_stride != 0 && r->allowed_stride < (V + 31) / 32) return false;
    return r->repetition_penalty > 0.f && r->repetition_penalty < INFINITY && r->presence_penalty == r->presence_penalty &&
           r->frequency_penalty == r->frequency_penalty;
}

template <typename DT, bool PICK>
rnntStatus_t launch_rules(const void *x, int rows, int V, const rnntRules &r, int *out, float *logp, void *processed,
                          hipStream_t st) {
    typedef typename DT::elem E;
    constexpr int EPC = DT::EPC;
    const bool vec = V % EPC == 0 && aligned16(x) && (PICK || aligned16(processed)) &&
                     (r.bias == nullptr || (aligned16(r.bias) && r.bias_stride % 4 == 0));
    const int work = vec ? V / EPC : V;
    const int threads = work > 1024 && rows < 512 ? 1024 : 256;
    if (vec)
        hipLaunchKernelGGL((row_rules_kernel<DT, EPC, PICK>), dim3(rows), dim3(threads), 0, st, static_cast<const E *>(x), rows, V,
                           r, rows / r.contexts, out, logp, static_cast<E *>(processed));
    else
        hipLaunchKernelGGL((row_rules_kernel<DT, 1, PICK>), dim3(rows), dim3(threads), 0, st, static_cast<const E *>(x), rows, V, r,
                           rows / r.contexts, out, logp, static_cast<E *>(processed));
    return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED;
}

template <bool PICK>
rnntStatus_t dispatch(const void *x, int rows, int V, rnntDtype_t dtype, const rnntRules *r, int *out, float *logp,
                      void *processed, void *stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RNNT_DTYPE_F32: return launch_rules<F32, PICK>(x, rows, V, *r, out, logp, processed, st);
        case RNNT_DTYPE_BF16: return launch_rules<BF16, PICK>(x, rows, V, *r, out, logp, processed, st);
        case RNNT_DTYPE_F16: return launch_rules<F16, PICK>(x, rows, V, *r, out, logp, processed, st);
        default: return RNNT_STATUS_INVALID_VALUE;
    }
}

}  // namespace

extern "C" {

rnntStatus_t rnnt_row_rules(const void *x, int rows, int V, rnntDtype_t dtype, const rnntRules *rules, int *out, float *logp,
                            void *stream) {
    if (x == nullptr || out == nullptr || rows < 1 || V < 1 || !rules_ok(rules, rows, V)) return RNNT_STATUS_INVALID_VALUE;
    return dispatch<true>(x, rows, V, dtype, rules, out, logp, nullptr, stream);
}

rnntStatus_t rnnt_process_logits(const void *x, int rows, int V, rnntDtype_t dtype, const rnntRules *rules, void *processed,
                                 void *stream) {
    if (x == nullptr || processed == nullptr || rows < 1 || V < 1 || !rules_ok(rules, rows, V)) return RNNT_STATUS_INVALID_VALUE;
    return dispatch<false>(x, rows, V, dtype, rules, nullptr, nullptr, processed, stream);
}

}  // extern "C"
