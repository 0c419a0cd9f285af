// state_space_mi355.hip — the recurrent layer of a state-space prediction network on MI355X (gfx950): the short causal
// convolution and the selective scan, each for whole sequences (forward and backward) and for single tokens.
//
// The reference's prediction network is embedding -> LSTM -> Linear (src/decoder/decoder.py:5-44) and its decoding loops
// carry that layer's state from emission to emission (src/rnnt/model.py:145-165).  These kernels compute a layer of
// the same place and interface:
//     convolution   p_t = bias + sum_k w_k x_{t-W+1+k},  y_t = p_t sigmoid(p_t)
//     scan          delta_t = softplus(dt_t + dt_bias),  h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t x_t B_t[n],
//                   y_t = (sum_n C_t[n] h_t[n] + D x_t) z_t sigmoid(z_t)
// for every channel d of every sequence b; B_t and C_t are shared by all channels of a sequence.
// Everything between loads and stores is fp32.  No atomics: two runs give the same bits.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/rnnt_mi355.h"
#include "elem_types.h"

namespace {

using namespace rnnt_mi355_detail;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.925963033500e-08f, kLn2 = 0.6931471805599453f;

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float rcp_(float v) { return __builtin_amdgcn_rcpf(v); }
__device__ __forceinline__ float sigmoid_(float v) { return rcp_(1.f + exp2_(-kLog2e * v)); }

// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1], and its derivative sigmoid(v) in `sig`.
// log1p(e) = e P(e), P the degree-9 Chebyshev interpolant of log1p(e) / e on [0, 1] (fit 1.2e-8 relative): rounding
// 1 + e first would cost 6e-8 / delta, and steps of delta = 1e-3 are ordinary.  v log2(e) is formed in two parts, since
// an exponent of 10 would pass its rounding on to delta tenfold.
__device__ __forceinline__ float softplus_(float v, float &sig) {
    const float w = -fabsf(v), hi = w * kLog2e;
    float lo = fma_(w, kLog2e, -hi);
    lo = w > -128.f ? fma_(w, kLog2eLow, lo) * kLn2 : 0.f;
    float e = exp2_(hi);
    e = fma_(e, lo, e);
    float p = -3.176057013e-03f;
    p = fma_(p, e, 1.954252832e-02f);
    p = fma_(p, e, -5.637361482e-02f);
    p = fma_(p, e, 1.054362357e-01f);
    p = fma_(p, e, -1.526966691e-01f);
    p = fma_(p, e, 1.966327429e-01f);
    p = fma_(p, e, -2.495161593e-01f);
    p = fma_(p, e, 3.332971036e-01f);
    p = fma_(p, e, -4.999989271e-01f);
    p = fma_(p, e, 1.0f);
    const float r = rcp_(1.f + e);
    sig = v > 0.f ? r : e * r;
    return fma_(e, p, fmaxf(v, 0.f));  // (NaN comes through e)
}

// ---------------------------------------------------------------------------------------------
// B_t and C_t are the same for all channels of a sequence, so for a whole wave: the scan kernels read them through the
// scalar cache into scalar registers, and the recurrence's multiply-adds take them as scalar operands: no vector load,
// no LDS, no register per lane.  Scalar loads are whole aligned words, the scalar unit has no half-precision conversion,
// and unpacking bf16 there costs as many issue slots as the recurrence itself (16 states: 100 scalar beside 105 vector
// instructions a step, 0.73 us a step).  So a first small kernel lays both out as fp32, four states of B beside the
// same four of C: a row is whole 32-byte loads for any wave, whatever type, stride or alignment the caller's have.
// Rows from a sequence's length on, up to a multiple of 16 (and one row more at the end), are zero.
// ---------------------------------------------------------------------------------------------
typedef const __attribute__((address_space(4))) float *scalar_floats;

template <int N>
struct ScalarRow {  // N states of B and of C
    float v[2 * N];
    __device__ __forceinline__ void load(const float *p) {
        scalar_floats q = (scalar_floats) reinterpret_cast<unsigned long long>(p);
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) v[i] = q[i];
    }
    __device__ __forceinline__ float B(int n) const { return v[n / 4 * 8 + n % 4]; }
    __device__ __forceinline__ float C(int n) const { return v[n / 4 * 8 + 4 + n % 4]; }
};

// ---------------------------------------------------------------------------------------------
// selective scan
// ---------------------------------------------------------------------------------------------
constexpr int kChunk = 16;  // steps between saved states; steps a backward wave holds in registers
constexpr int kAhead = 4;   // steps whose inputs a forward wave loads ahead

// A channel's constants and where a wave works.  Segments cut the time axis so that few sequences fill the chip:
// pass 1 walks every segment from a zero state (`local`), pass 2 joins the segments' ends in order, pass 3 walks them
// again from the right states.  A single segment needs pass 3 alone.
struct ScanGeom {
    int groups;    // of 64 channels
    int segments;  // per sequence
    int seg_len;   // steps per segment, a multiple of kChunk
    int blocks;    // per sequence: what a workgroup of the backward proper takes, `joined` segments each
    int joined;
    float *seg_state;  // [batch][segments][state / 4][dim][4]: a segment's end from zero, then the state it starts from
    float *seg_delta;  // [batch][segments][dim]: sum of delta over the segment
    float *rows;       // B and C: [batch][length rounded up to kChunk][2 state], and one row more
    int padded;        // length rounded up to kChunk
};

__device__ __forceinline__ int clamp_len(const int *lengths, int b, int length) {
    if (lengths == nullptr) return length;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > length ? length : n);
}

// (5 us for 16 x 1500 steps of 16 states.)
template <typename DT, int N>
__global__ __launch_bounds__(256) void scan_rows_kernel(const rnntScan a, const ScanGeom g) {
    typedef typename DT::elem E;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int k = (int)(i % (2 * N));
    const long long row = i / (2 * N);
    const long long b = row / g.padded;
    if (row > (long long)a.batch * g.padded) return;
    const int t = (int)(row - b * g.padded);
    float v = 0.f;
    if (b < a.batch && t < clamp_len(a.lengths, (int)b, a.length)) {
        const int n = k / 8 * 4 + k % 4;
        v = DT::to_float(k % 8 < 4 ? static_cast<const E *>(a.B)[b * a.B_batch + t * a.B_time + n]
                                   : static_cast<const E *>(a.C)[b * a.C_batch + t * a.C_time + n]);
    }
    g.rows[i] = v;
}

// N adjacent floats at any address (16-byte loads need no more than 4-byte alignment)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <int N>
__device__ __forceinline__ void load_row(const float *p, float (&v)[N]) {
#pragma unroll
    for (int n = 0; n < N; n += 4) {
        const f32x4_any w = *reinterpret_cast<const f32x4_any *>(p + n);
        v[n] = w.x;
        v[n + 1] = w.y;
        v[n + 2] = w.z;
        v[n + 3] = w.w;
    }
}
template <int N>
__device__ __forceinline__ void store_row(float *p, const float (&v)[N]) {
#pragma unroll
    for (int n = 0; n < N; n += 4) *reinterpret_cast<f32x4_any *>(p + n) = f32x4_any{v[n], v[n + 1], v[n + 2], v[n + 3]};
}
template <int N>
__device__ __forceinline__ void load_rates(const float *A, int d, float (&A2)[N]) {
    load_row<N>(A + (size_t)d * N, A2);
#pragma unroll
    for (int n = 0; n < N; ++n) A2[n] *= kLog2e;
}

// state tiles between kernels: [N / 4][dim][4] per (sequence, time)
template <int N>
__device__ __forceinline__ void load_tile(const float *tile, int dim, int d, float (&h)[N]) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        const f32x4 v = reinterpret_cast<const f32x4 *>(tile + (size_t)q * dim * 4)[(unsigned)d];
#pragma unroll
        for (int n = 0; n < 4; ++n) h[4 * q + n] = v[n];
    }
}
template <int N>
__device__ __forceinline__ void store_tile(float *tile, int dim, int d, const float (&h)[N]) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q)
        reinterpret_cast<f32x4 *>(tile + (size_t)q * dim * 4)[(unsigned)d] = f32x4{h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]};
}

// One wave walks 64 channels of one segment; lane = channel, all N states of it in registers: loads and stores are whole
// 128-byte lines, the sum over the states needs no other lane.  LOCAL: from zero, gives the segment's end and its sum of
// delta.  Otherwise: the outputs.
// Bound by the vector units: 16 states take 93 vector instructions and 19 quarter-rate ones (17 exponentials) a step.
// 16 sequences of up to 1500 steps (62 % of them live), 1024 channels, 16 states, bf16: 93 us, local 65 us, the
// instructions alone 62 and 49; memory would allow 42 (training, the states kept for backward among it).  One sequence of 4095 x 1536 fp32: 35 and 26 us.
// Four steps of inputs are under way (with eight the registers of a wave cost more than the loads: 80 against 73 us for the
// latter, all passes).
template <typename DT, int N, bool LOCAL>
__global__ __launch_bounds__(64) void scan_forward_kernel(const rnntScan a, const ScanGeom g) {
    typedef typename DT::elem E;
    const int lane = threadIdx.x;
    const int group = blockIdx.x % g.groups;
    const int rest = blockIdx.x / g.groups;
    const int seg = rest % g.segments, b = rest / g.segments;
    const int d0 = group * kWave + lane;
    const bool ok = d0 < a.dim;
    const int d = ok ? d0 : a.dim - 1;
    const unsigned lo = d;  // (a lane's offset from an address that the wave shares)
    const int t0 = seg * g.seg_len;
    const int t1 = t0 + g.seg_len < a.length ? t0 + g.seg_len : a.length;
    const int len = clamp_len(a.lengths, b, a.length);
    const int te = len < t1 ? (len > t0 ? len : t0) : t1;  // steps of this segment: [t0, te)

    float A2[N], h[N];
    load_rates<N>(a.A, d, A2);
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f;
    float *seg_state = g.segments > 1 ? g.seg_state + ((size_t)b * g.segments + seg) * N * a.dim : nullptr;
#pragma unroll
    for (int n = 0; n < N; ++n) h[n] = 0.f;
    if (!LOCAL) {
        if (seg_state) {
            load_tile<N>(seg_state, a.dim, d, h);
        } else if (a.initial_state) {
            load_row<N>(a.initial_state + ((size_t)b * a.dim + d) * N, h);
        }
    }
    const float skip = !LOCAL && a.D ? a.D[d] : 0.f;
    const E *xp = static_cast<const E *>(a.x) + b * a.x_batch;
    const E *dtp = static_cast<const E *>(a.dt) + b * a.dt_batch;
    const bool gated = a.z != nullptr;  // (without a gate its loads repeat x's: no branch between loads)
    const E *zp = gated ? static_cast<const E *>(a.z) + b * a.z_batch : xp;
    const long long z_time = gated ? a.z_time : a.x_time;
    const float *rows = g.rows + ((size_t)b * g.padded + t0) * 2 * N;
    E *yp = LOCAL ? nullptr : static_cast<E *>(a.y) + (size_t)b * a.length * a.dim;
    const int chunks = (a.length + kChunk - 1) / kChunk;
    float sum_delta = 0.f;

    E xn[kAhead], dtn[kAhead], zn[kAhead];
    auto fetch = [&](int t) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const long long tt = t + j < te ? t + j : te - 1;
            xn[j] = (xp + tt * a.x_time)[lo];
            dtn[j] = (dtp + tt * a.dt_time)[lo];
            if (!LOCAL) zn[j] = (zp + tt * z_time)[lo];
        }
    };
    // the next step's row is under way while a step is computed (32 states of two rows would not fit the scalar registers)
    constexpr bool kNext = N <= 16;
    ScalarRow<N> next;
    if (te > t0) {
        fetch(t0);
        if (kNext) next.load(rows);
    }
    for (int tb = t0; tb < te; tb += kAhead) {
        E xc[kAhead], dtc[kAhead], zc[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            xc[j] = xn[j];
            dtc[j] = dtn[j];
            if (!LOCAL) zc[j] = zn[j];
        }
        if (!LOCAL && a.chunk_states && tb % kChunk == 0 && ok)
            store_tile<N>(a.chunk_states + ((size_t)b * chunks + tb / kChunk) * N * a.dim, a.dim, d, h);
        fetch(tb + kAhead);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int t = tb + j;
            if (t >= te) break;
            ScalarRow<N> row = next;
            if (!kNext) row.load(rows);
            rows += 2 * N;
            if (kNext) next.load(rows);
            float sig;
            const float x = DT::to_float(xc[j]);
            const float delta = softplus_(DT::to_float(dtc[j]) + bias, sig);
            const float dx = delta * x;
            float y0 = 0.f, y1 = 0.f;  // (two chains)
#pragma unroll
            for (int n = 0; n < N; n += 2) {
                h[n] = fma_(exp2_(delta * A2[n]), h[n], dx * row.B(n));
                h[n + 1] = fma_(exp2_(delta * A2[n + 1]), h[n + 1], dx * row.B(n + 1));
                if (!LOCAL) {
                    y0 = fma_(row.C(n), h[n], y0);
                    y1 = fma_(row.C(n + 1), h[n + 1], y1);
                }
            }
            if (LOCAL) {
                sum_delta += delta;
            } else {
                float y = fma_(skip, x, y0 + y1);
                if (gated) {
                    const float z = DT::to_float(zc[j]);
                    y *= z * sigmoid_(z);
                }
                if (ok) (yp + (size_t)t * a.dim)[lo] = DT::from_float(y);
            }
        }
    }
    if (LOCAL) {
        if (ok) {
            store_tile<N>(seg_state, a.dim, d, h);
            g.seg_delta[((size_t)b * g.segments + seg) * a.dim + d] = sum_delta;
        }
        return;
    }
    if (ok) {
        for (int t = te; t < t1; ++t) (yp + (size_t)t * a.dim)[lo] = DT::from_float(0.f);
        // the segment that holds the last step (segment 0 of an empty sequence) has the final state
        const bool last = len > t0 ? len <= t1 : (seg == 0 && len == 0);
        if (a.final_state && last) store_row<N>(a.final_state + ((size_t)b * a.dim + d) * N, h);
    }
}

// Pass 2: the state (forward) or the state's gradient (backward) at every segment's border, in order.
//   forward:  seg_state[s] <- state before segment s;      state <- exp(A sum_delta[s]) state + end[s]
//   backward: seg_state[s] <- gradient after segment s;    the same towards smaller s, the start grad_final
// A lane has 4 states of a channel.  The waves of a workgroup share the segments: each joins its range from zero, which
// gives a decay and an end for the range, and walks it again from what the ranges before it give.  Loads of kJoinAhead
// segments are under way at once: alone they are a chain of two loads and an exponential per segment.
// 32 segments of 16 x 1024 x 16 states: 18 us (two reads and a write of 34 MB: 5.6 TB/s); 128 segments of 1536 x 16: 14 us
// (64 of them, a thread per 4 states and no loads ahead: 24).
// Up to kJoinAhead segments one wave does it alone, once.
// A segment's factor exp(A sum_delta) is applied in two halves, each of them at most 2^127: a state may grow (A > 0) from 1e-30
// by more than fp32 holds, and 0 stays 0 where the factor alone would be infinite.
constexpr int kJoinWaves = 8, kJoinAhead = 8;

__device__ __forceinline__ float carried(float delta, float half_A2, float h) {
    const float e = exp2_(fminf(delta * half_A2, 127.f));
    return e * (e * h);
}

template <int N, bool BACKWARD, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void scan_join_kernel(const rnntScan a, const ScanGeom g) {
    __shared__ float s_end[WAVES][4][kWave], s_delta[WAVES][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const long long i = (long long)blockIdx.x * kWave + lane;
    const int d = (int)(i % a.dim);
    const long long r = i / a.dim;
    const int q = (int)(r % (N / 4));
    const long long b = r / (N / 4);
    const bool ok = b < a.batch;
    const int per = (g.segments + WAVES - 1) / WAVES;
    const int k0 = wave * per, k1 = !ok ? k0 : (k0 + per < g.segments ? k0 + per : g.segments);
    float A2[4] = {}, h[4] = {}, start[4] = {};
    const float *from = BACKWARD ? a.grad_final : a.initial_state;
    if (ok) {
        load_row<4>(a.A + (size_t)d * N + q * 4, A2);
        if (from) load_row<4>(from + ((size_t)b * a.dim + d) * N + q * 4, start);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) A2[n] *= 0.5f * kLog2e;
    f32x4 *tiles = reinterpret_cast<f32x4 *>(g.seg_state) + ((size_t)b * g.segments * (N / 4) + q) * a.dim + d;
    const float *deltas = g.seg_delta + (size_t)b * g.segments * a.dim + d;
    auto walk = [&](bool write) {
        float sum = 0.f;
        for (int kb = k0; kb < k1; kb += kJoinAhead) {
            f32x4 end[kJoinAhead];
            float delta[kJoinAhead];
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                const int k = kb + j < k1 ? kb + j : k1 - 1, s = BACKWARD ? g.segments - 1 - k : k;
                end[j] = tiles[(size_t)s * (N / 4) * a.dim];
                delta[j] = deltas[(size_t)s * a.dim];
            }
#pragma unroll
            for (int j = 0; j < kJoinAhead; ++j) {
                if (kb + j >= k1) break;
                const int s = BACKWARD ? g.segments - 1 - (kb + j) : kb + j;
                if (write) tiles[(size_t)s * (N / 4) * a.dim] = f32x4{h[0], h[1], h[2], h[3]};
                sum += delta[j];
#pragma unroll
                for (int n = 0; n < 4; ++n) h[n] = carried(delta[j], A2[n], h[n]) + end[j][n];
            }
        }
        return sum;
    };
    if (WAVES > 1) {
        s_delta[wave][lane] = walk(false);
#pragma unroll
        for (int n = 0; n < 4; ++n) s_end[wave][n][lane] = h[n];
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        h[n] = start[n];
        for (int w = 0; w < wave; ++w) h[n] = carried(s_delta[w][lane], A2[n], h[n]) + s_end[w][n][lane];
    }
    walk(true);
}

// Pass 1 of the backward: the gradient of a segment's first state that its own outputs give.
//   G <- exp(delta_t A) (G + C_t gy_t), t from the segment's last step to its first
// (83 us at the shape above; the same walk as the forward's, bound in the same way.)
template <typename DT, int N>
__global__ __launch_bounds__(64) void scan_backward_local_kernel(const rnntScan a, const ScanGeom g) {
    typedef typename DT::elem E;
    const int lane = threadIdx.x;
    const int group = blockIdx.x % g.groups;
    const int rest = blockIdx.x / g.groups;
    const int seg = rest % g.segments, b = rest / g.segments;
    const int d0 = group * kWave + lane;
    const bool ok = d0 < a.dim;
    const int d = ok ? d0 : a.dim - 1;
    const unsigned lo = d;  // (a lane's offset from an address that the wave shares)
    const int t0 = seg * g.seg_len;
    const int t1 = t0 + g.seg_len < a.length ? t0 + g.seg_len : a.length;
    const int len = clamp_len(a.lengths, b, a.length);
    const int te = len < t1 ? (len > t0 ? len : t0) : t1;

    float A2[N], G[N];
    load_rates<N>(a.A, d, A2);
#pragma unroll
    for (int n = 0; n < N; ++n) G[n] = 0.f;
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f;
    const E *dtp = static_cast<const E *>(a.dt) + b * a.dt_batch;
    const bool gated = a.z != nullptr;
    const E *zp = gated ? static_cast<const E *>(a.z) + b * a.z_batch : dtp;
    const long long z_time = gated ? a.z_time : a.dt_time;
    const E *gp = static_cast<const E *>(a.grad_y) + b * a.grad_y_batch;
    const float *rows = g.rows + ((size_t)b * g.padded + te) * 2 * N;  // one past the step
    float sum_delta = 0.f;
    E dtn[kAhead], zn[kAhead], gn[kAhead];
    auto fetch = [&](int t) {  // steps t, t - 1, ...
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const long long tt = t - j > t0 ? t - j : t0;
            dtn[j] = (dtp + tt * a.dt_time)[lo];
            gn[j] = (gp + tt * a.grad_y_time)[lo];
            zn[j] = (zp + tt * z_time)[lo];
        }
    };
    if (te > t0) fetch(te - 1);
    for (int tb = te - 1; tb >= t0; tb -= kAhead) {
        E dtc[kAhead], zc[kAhead], gc[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            dtc[j] = dtn[j];
            gc[j] = gn[j];
            zc[j] = zn[j];
        }
        fetch(tb - kAhead);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int t = tb - j;
            if (t < t0) break;
            rows -= 2 * N;
            ScalarRow<N> row;
            row.load(rows);
            float sig;
            const float delta = softplus_(DT::to_float(dtc[j]) + bias, sig);
            float gy = DT::to_float(gc[j]);
            if (gated) {
                const float z = DT::to_float(zc[j]);
                gy *= z * sigmoid_(z);
            }
            sum_delta += delta;
#pragma unroll
            for (int n = 0; n < N; ++n) G[n] = exp2_(delta * A2[n]) * fma_(row.C(n), gy, G[n]);
        }
    }
    if (ok) {
        store_tile<N>(g.seg_state + ((size_t)b * g.segments + seg) * N * a.dim, a.dim, d, G);
        g.seg_delta[((size_t)b * g.segments + seg) * a.dim + d] = sum_delta;
    }
}

// ---- sums over the 64 lanes ------------------------------------------------------------------------------------------
// 8 values of each of 8 steps are summed over the lanes as one tree: every stage halves the values and the lanes that
// share one, 18 instructions a step where 8 separate butterflies would take 48.
template <int CTRL>
__device__ __forceinline__ float dpp_(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E, kHalfMirror = 0x141, kRowRor8 = 0x128;

// lanes without `up` keep a's sums, the others b's; CTRL exchanges the two kinds of lanes
template <int CTRL>
__device__ __forceinline__ float fold(float a, float b, bool up) {
    return (up ? b : a) + dpp_<CTRL>(up ? a : b);
}

// 8 values over the lane bits 5, 4, 3: lane l then has the sums of value l / 8 over 8 of the 64 lanes
__device__ __forceinline__ float fold_values(float (&v)[8], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 2]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return fold<kRowRor8>(v[0], v[1], lane & 8);
}

// The steps of a chunk, taken from the last to the first, over the lane bits 2, 1, 0: when step 8 j comes, lane l gets the
// sums of step 8 j + (l >> 2 & 1) + 2 (l >> 1 & 1) + 4 (l & 1).
struct FoldSteps {
    float held[3];
    template <int I>
    __device__ __forceinline__ float take(float v, int lane) {
        if constexpr (I & 1) {
            held[0] = v;
        } else {
            v = fold<kHalfMirror>(v, held[0], lane & 4);
            if constexpr (I & 2) {
                held[1] = v;
            } else {
                v = fold<kQuadXor2>(v, held[1], lane & 2);
                if constexpr (I & 4)
                    held[2] = v;
                else
                    v = fold<kQuadXor1>(v, held[2], lane & 1);
            }
        }
        return v;
    }
};

// The backward proper.  The N / 4 waves of a workgroup share 64 channels of one segment; wave w owns the states
// [4 w, 4 w + 4) of all of them, so that a chunk of 16 steps of h and of exp(delta A) stays in registers (2 x 16 x 4).
// B and C come from LDS, 16 bytes at an address that the wave shares: scalar loads return out of order, so that each use
// would wait for all of them.  Per chunk, from the last to the first:
//   1. each wave turns its share of the steps' inputs into delta, x, gy (LDS), keeping what its outputs need;
//   2. each wave walks its states forwards from the saved state, then backwards, summing dB, dC over the 64 lanes and
//      leaving its share of the sums over n in LDS;
//   3. each wave adds the waves' shares of its steps and writes dx, ddt, dz.
// 275 us at the shape above, 28 us for 32 sequences of 41 steps.  Bound by the vector units: some 1600 vector instructions
// a wave and chunk (17 + 55 a step for 4 states, 18 of them the sums over lanes), issuing 66 % of the time with the two waves
// per SIMD that 239 registers and 64 KiB of LDS leave.  Chunks of 8 steps leave three (249 us) but keep twice the states for
// the backward pass; B and C as scalar operands, each use of which waits for all scalar loads, took 90 us more.
template <int I>
struct Index {
    static constexpr int value = I;
};
template <int I, typename F>
__device__ __forceinline__ void down(F &&f) {  // f at I - 1, I - 2, ..., 0, each a constant
    if constexpr (I > 0) {
        f(Index<I - 1>());
        down<I - 1>(f);
    }
}

struct ScanPartials {
    float *BC;      // [batch][length][groups][2 N]
    float *A;       // [batch * blocks][dim * N]
    float *D;       // [batch * blocks][2][dim]: D, dt_bias
};

template <typename DT, int N>
__global__ __launch_bounds__(N * 16, 2) void scan_backward_kernel(const rnntScan a, const ScanGeom g, const ScanPartials out) {
    typedef typename DT::elem E;
    constexpr int S = 4, W = N / S, kMine = kChunk / W;
    constexpr int kShare = kChunk * 2 * N / (W * kWave);  // values of a chunk's rows, and of its dB and dC, per thread
    __shared__ float s_delta[kChunk][kWave], s_x[kChunk][kWave], s_gy[kChunk][kWave];
    __shared__ float s_part[3][W][kChunk][kWave];
    __shared__ float s_bc[kChunk][2 * N];
    __shared__ f32x4 s_rows[kChunk][N / 2];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = blockIdx.x % g.groups;
    const int rest = blockIdx.x / g.groups;
    const int block = rest % g.blocks, b = rest / g.blocks;
    const int d0 = group * kWave + lane;
    const bool ok = d0 < a.dim;
    const int d = ok ? d0 : a.dim - 1;
    const unsigned lo = d;  // (a lane's offset from an address that the wave shares)
    const int steps_per = g.joined * g.seg_len, t0 = block * steps_per;
    const int t1 = t0 + steps_per < a.length ? t0 + steps_per : a.length;
    const int len = clamp_len(a.lengths, b, a.length);
    const int te = len < t1 ? (len > t0 ? len : t0) : t1;
    const int chunks = (a.length + kChunk - 1) / kChunk;

    float A2[S], G[S], dA[S];
#pragma unroll
    for (int n = 0; n < S; ++n) {
        A2[n] = a.A[(size_t)d * N + wave * S + n] * kLog2e;
        G[n] = 0.f;
        dA[n] = 0.f;
    }
    // (states of 4 to a tile row: state n of the layer is element n % 4 of row n / 4)
    auto tile_at = [&](const float *tile, int n) { return tile + ((size_t)(n / 4) * a.dim + d) * 4 + n % 4; };
    if (g.segments > 1) {
        const int last = block < g.blocks - 1 ? (block + 1) * g.joined - 1 : g.segments - 1;
        const float *tile = g.seg_state + ((size_t)b * g.segments + last) * N * a.dim;
#pragma unroll
        for (int n = 0; n < S; ++n) G[n] = *tile_at(tile, wave * S + n);
    } else if (a.grad_final) {
#pragma unroll
        for (int n = 0; n < S; ++n) G[n] = a.grad_final[((size_t)b * a.dim + d) * N + wave * S + n];
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f;
    const float skip = a.D ? a.D[d] : 0.f;
    const E *xp = static_cast<const E *>(a.x) + b * a.x_batch;
    const E *dtp = static_cast<const E *>(a.dt) + b * a.dt_batch;
    const bool gated = a.z != nullptr;
    const E *zp = gated ? static_cast<const E *>(a.z) + b * a.z_batch : xp;
    const long long z_time = gated ? a.z_time : a.x_time;
    const E *gp = static_cast<const E *>(a.grad_y) + b * a.grad_y_batch;
    const float *rows = g.rows + (size_t)b * g.padded * 2 * N + threadIdx.x;
    const size_t out0 = (size_t)b * a.length * a.dim;
    E *dxp = static_cast<E *>(a.grad_x) + out0, *ddtp = static_cast<E *>(a.grad_dt) + out0;
    E *dzp = gated ? static_cast<E *>(a.grad_z) + out0 : nullptr;
    float dD = 0.f, dbias = 0.f;

    if (ok) {
        for (int t = te + wave; t < t1; t += W) {
            (dxp + (size_t)t * a.dim)[lo] = DT::from_float(0.f);
            (ddtp + (size_t)t * a.dim)[lo] = DT::from_float(0.f);
            if (dzp) (dzp + (size_t)t * a.dim)[lo] = DT::from_float(0.f);
        }
    }
    // A chunk's inputs are under way while the chunk after it is computed.  With 8 states a wave has 8 of its steps, whose inputs
    // beside a whole chunk of h and decay spill 12 registers; half the walk back there is more room (5; 16 x 1500 x 1024 x 8 bf16, a
    // training pass: 412 and 385 us; with 16 and 32 states, which do not spill, late loads cost 0.5 %).
    constexpr bool kLate = N == 8;
    E xn[kMine], dtn[kMine], zn[kMine], gn[kMine];
    f32x4 hn;
    float rn[kShare];
    auto fetch = [&](int c) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int t = c * kChunk + wave * kMine + j;
            const long long tt = t < te ? t : te - 1;
            xn[j] = (xp + tt * a.x_time)[lo];
            dtn[j] = (dtp + tt * a.dt_time)[lo];
            zn[j] = (zp + tt * z_time)[lo];
            gn[j] = (gp + tt * a.grad_y_time)[lo];
        }
#pragma unroll
        for (int j = 0; j < kShare; ++j) rn[j] = rows[(size_t)c * (kChunk * 2 * N) + j * W * kWave];
        hn = reinterpret_cast<const f32x4 *>(a.chunk_states + ((size_t)b * chunks + c) * N * a.dim + (size_t)wave * a.dim * 4)[lo];
    };
    const int c0 = t0 / kChunk;
    if (te > t0) fetch((te - 1) / kChunk);
    for (int c = (te - 1) / kChunk; te > t0 && c >= c0; --c) {
        const int tc = c * kChunk;
        float sigv[kMine], dzf[kMine];
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int i = wave * kMine + j, t = tc + i;
            const float x = DT::to_float(xn[j]);
            const float delta = softplus_(DT::to_float(dtn[j]) + bias, sigv[j]);
            float gy = DT::to_float(gn[j]);
            dzf[j] = 0.f;
            if (gated) {
                const float z = DT::to_float(zn[j]), s = sigmoid_(z);
                dzf[j] = gy * fma_(z * s, 1.f - s, s);
                gy *= z * s;
            }
            const bool in = t < te && ok;  // a step past the end leaves the state and adds nothing
            s_delta[i][lane] = in ? delta : 0.f;
            s_x[i][lane] = in ? x : 0.f;
            s_gy[i][lane] = in ? gy : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kShare; ++j) reinterpret_cast<float *>(s_rows)[threadIdx.x + j * W * kWave] = rn[j];
        float h[S] = {hn.x, hn.y, hn.z, hn.w};
        if (!kLate && c > c0) fetch(c - 1);
        __syncthreads();

        float before[kChunk][S], decay[kChunk][S];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            const f32x4 B = s_rows[i][2 * wave], C = s_rows[i][2 * wave + 1];
            const float delta = s_delta[i][lane], dx = delta * s_x[i][lane];
            float y = 0.f;
#pragma unroll
            for (int n = 0; n < S; ++n) {
                before[i][n] = h[n];
                decay[i][n] = exp2_(delta * A2[n]);
                h[n] = fma_(decay[i][n], h[n], dx * B[n]);
                y = fma_(C[n], h[n], y);
            }
            s_part[0][wave][i][lane] = y;
        }
        FoldSteps steps;
        float sums_of[kChunk / 8];
        auto reverse = [&](auto index) {
            constexpr int i = decltype(index)::value;
            if constexpr (kLate && i == kChunk / 2) {
                if (c > c0) fetch(c - 1);
            }
            const f32x4 B = s_rows[i][2 * wave], C = s_rows[i][2 * wave + 1];
            const float delta = s_delta[i][lane], dx = delta * s_x[i][lane], gy = s_gy[i][lane];
            float inner = 0.f, rate = 0.f, sums[2 * S];
#pragma unroll
            for (int n = 0; n < S; ++n) {
                const float after = i + 1 < kChunk ? before[i + 1 < kChunk ? i + 1 : 0][n] : h[n];
                const float gn = fma_(C[n], gy, G[n]);
                sums[n] = gn * dx;
                sums[S + n] = after * gy;
                inner = fma_(gn, B[n], inner);
                G[n] = gn * decay[i][n];
                const float r = G[n] * before[i][n];
                dA[n] = fma_(r, delta, dA[n]);
                rate = fma_(r, A2[n], rate);
            }
            s_part[1][wave][i][lane] = inner;
            s_part[2][wave][i][lane] = rate;
            const float sum = steps.template take<i>(fold_values(sums, lane), lane);
            if constexpr (i % 8 == 0) sums_of[i / 8] = sum;
            // (a scheduler free to mix steps, or to put dA's additions off, wants more than the 256 registers that two waves
            // per SIMD leave)
#pragma unroll
            for (int n = 0; n < S; ++n) asm volatile("" : "+v"(dA[n]));
            __builtin_amdgcn_sched_barrier(0);
        };
        down<kChunk>(reverse);
        {
            const int k = lane >> 3, i = (lane >> 2 & 1) + (lane & 2) + (lane & 1) * 4;
#pragma unroll
            for (int j = 0; j < kChunk / 8; ++j) s_bc[8 * j + i][(k < S ? 0 : N - S) + wave * S + k] = sums_of[j];
        }
        __syncthreads();

#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int i = wave * kMine + j, t = tc + i;
            float y = 0.f, inner = 0.f, rate = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                y += s_part[0][w][i][lane];
                inner += s_part[1][w][i][lane];
                rate += s_part[2][w][i][lane];
            }
            const float delta = s_delta[i][lane], x = s_x[i][lane], gy = s_gy[i][lane];
            if (t < te && ok) {
                const float ddt = fma_(x, inner, rate * kLn2) * sigv[j];
                (dxp + (size_t)t * a.dim)[lo] = DT::from_float(fma_(delta, inner, skip * gy));
                (ddtp + (size_t)t * a.dim)[lo] = DT::from_float(ddt);
                if (dzp) (dzp + (size_t)t * a.dim)[lo] = DT::from_float(dzf[j] * fma_(skip, x, y));
                dD = fma_(gy, x, dD);
                dbias += ddt;
            }
        }
#pragma unroll
        for (int j = 0; j < kShare; ++j) {
            const int k = threadIdx.x + j * W * kWave, i = k / (2 * N);
            if (tc + i < te)
                out.BC[(((size_t)b * a.length + tc + i) * g.groups + group) * 2 * N + k % (2 * N)] = s_bc[i][k % (2 * N)];
        }
        __syncthreads();
    }

    const size_t part = (size_t)b * g.blocks + block;
    if (ok) {
#pragma unroll
        for (int n = 0; n < S; ++n) out.A[(part * a.dim + d) * N + wave * S + n] = dA[n];
        if (block == 0 && a.grad_initial) {
#pragma unroll
            for (int n = 0; n < S; ++n) a.grad_initial[((size_t)b * a.dim + d) * N + wave * S + n] = G[n];
        }
    }
    s_delta[wave][lane] = dD;
    s_x[wave][lane] = dbias;
    __syncthreads();
    if (wave < 2 && ok) {
        const float(*v)[kWave] = wave == 0 ? s_delta : s_x;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += v[w][lane];
        out.D[(part * 2 + wave) * a.dim + d] = sum;
    }
}

// dB, dC: the channel groups' shares of every step, in order; dA, dD, ddt_bias: the shares of sequences and segments.
// Workgroups [0, bc_blocks) take 1024 values of the steps each, the others 64 columns of the parameters, their 16 waves a
// range of the shares each.
template <typename DT, int N>
__global__ __launch_bounds__(1024) void scan_backward_sum_kernel(const rnntScan a, const ScanGeom g, const ScanPartials in,
                                                                 unsigned bc_blocks) {
    typedef typename DT::elem E;
    if (blockIdx.x < bc_blocks) {
        const long long i = (long long)blockIdx.x * 1024 + threadIdx.x;
        const int k = (int)(i % (2 * N));
        const long long row = i / (2 * N);
        if (row >= (long long)a.batch * a.length) return;
        const int b = (int)(row / a.length), t = (int)(row - (long long)b * a.length);
        float s = 0.f;
        if (t < clamp_len(a.lengths, b, a.length)) {
            const float *p = in.BC + (size_t)row * g.groups * 2 * N + k;
#pragma unroll 8
            for (int j = 0; j < g.groups; ++j) s += p[(size_t)j * 2 * N];
        }
        E *o = static_cast<E *>(k < N ? a.grad_B : a.grad_C);
        o[(size_t)row * N + (k < N ? k : k - N)] = DT::from_float(s);
        return;
    }
    __shared__ float s_sum[16][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const long long i = (long long)(blockIdx.x - bc_blocks) * kWave + lane;
    const long long rates = (long long)a.dim * N, columns = rates + 2 * a.dim;
    const int parts = a.batch * g.blocks, per = (parts + 15) / 16;
    const int p0 = wave * per, p1 = p0 + per < parts ? p0 + per : parts;
    float s = 0.f;
    if (i < columns) {
        const float *p = i < rates ? in.A + i : in.D + (i - rates);
        const size_t step = i < rates ? (size_t)rates : (size_t)2 * a.dim;
#pragma unroll 8
        for (int q = p0; q < p1; ++q) s += p[(size_t)q * step];
    }
    s_sum[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || i >= columns) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += s_sum[w][lane];
    if (i < rates) {
        a.grad_A[i] = s;
    } else {
        const long long k = i - rates;
        float *o = k < a.dim ? a.grad_D : a.grad_dt_bias;
        if (o) o[k < a.dim ? k : k - a.dim] = s;
    }
}

// One token per sequence: a lane owns 4 states of a channel (16 bytes of the state, read and written once), N / 4
// neighbouring lanes the channel.  256 sequences of 2048 x 16 states: 14 us, 5.1 TB/s of the state's 67 MB; one of
// 1024 x 16: 3 us.
template <typename DT, int N>
__global__ __launch_bounds__(256) void scan_step_kernel(const rnntScan a) {
    typedef typename DT::elem E;
    constexpr int Q = N / 4;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int q = (int)(i % Q);
    const long long r = i / Q;
    if (r >= (long long)a.batch * a.dim) return;  // (whole groups of Q lanes)
    const int b = (int)(r / a.dim), d = (int)(r - (long long)b * a.dim);
    float sig;
    const float x = DT::to_float(static_cast<const E *>(a.x)[b * a.x_batch + d]);
    const float delta = softplus_(DT::to_float(static_cast<const E *>(a.dt)[b * a.dt_batch + d]) + (a.dt_bias ? a.dt_bias[d] : 0.f), sig);
    const float dx = delta * x;
    const E *B = static_cast<const E *>(a.B) + b * a.B_batch + q * 4;
    const E *C = static_cast<const E *>(a.C) + b * a.C_batch + q * 4;
    const size_t at = (size_t)r * N + q * 4;
    float y = 0.f, h[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        h[n] = fma_(exp2_(delta * (a.A[(size_t)d * N + q * 4 + n] * kLog2e)), a.initial_state[at + n], dx * DT::to_float(B[n]));
        y = fma_(DT::to_float(C[n]), h[n], y);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) a.final_state[at + n] = h[n];
    if (Q >= 2) y += dpp_<kQuadXor1>(y);
    if (Q >= 4) y += dpp_<kQuadXor2>(y);
    if (Q >= 8) y += dpp_<kHalfMirror>(y);
    if (q == 0) {
        y = fma_(a.D ? a.D[d] : 0.f, x, y);
        if (a.z) {
            const float z = DT::to_float(static_cast<const E *>(a.z)[b * a.z_batch + d]);
            y *= z * sigmoid_(z);
        }
        static_cast<E *>(a.y)[r] = DT::from_float(y);
    }
}

// ---------------------------------------------------------------------------------------------
// causal convolution
// ---------------------------------------------------------------------------------------------
// A wave takes 64 channels of a run of steps; the waves of a workgroup take neighbouring runs of the same channels.
constexpr int kRunForward = 32, kRunBackward = 64;
constexpr int kConvAhead = 8;  // steps loaded at once
constexpr int kConvWaves = 4;

// row t of xe - (W - 1) rows: x for t >= 0, the initial state (zeros) before
template <typename DT, int W>
__device__ __forceinline__ float conv_in(const rnntConv &c, int b, long long t, int d) {
    typedef typename DT::elem E;
    if (t >= 0) return DT::to_float(static_cast<const E *>(c.x)[b * c.x_batch + t * c.x_time + d]);
    return c.initial_state ? DT::to_float(static_cast<const E *>(c.initial_state)[((size_t)b * (W - 1) + (W - 1 + t)) * c.dim + d]) : 0.f;
}

// Bound by memory: 16 x 1500 x 1024 fp16 (62 % of the steps live) 16.5 us, 80 MB at 4.8 TB/s (20 us with a test per step: whole
// blocks and the activation as a constant leave none).
template <typename DT, int W, bool SILU>
__global__ __launch_bounds__(kConvWaves *kWave) void conv_forward_kernel(const rnntConv c, int runs, int groups) {
    typedef typename DT::elem E;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int d = (int)(blockIdx.x % groups) * kWave + lane;
    const long long item = (long long)(blockIdx.x / groups) * kConvWaves + wave;
    const unsigned lo = d;
    const int run = (int)(item % runs);
    const long long b = item / runs;
    if (b >= c.batch || d >= c.dim) return;
    const int len = clamp_len(c.lengths, (int)b, c.length);
    const int t0 = run * kRunForward, t1 = t0 + kRunForward < c.length ? t0 + kRunForward : c.length;
    const int te = len < t1 ? (len > t0 ? len : t0) : t1;
    float w[W], win[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = c.weight[(size_t)d * W + k];
    const float bias = c.bias ? c.bias[d] : 0.f;
    const E *x = static_cast<const E *>(c.x) + b * c.x_batch;
    E *y = static_cast<E *>(c.y) + (size_t)b * c.length * c.dim;
    if (te > t0) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) win[k + 1] = conv_in<DT, W>(c, (int)b, (long long)t0 - (W - 1) + k, d);
    }
    auto block = [&](int tb, auto whole) {  // steps [tb, tb + kConvAhead), or up to te
        constexpr bool kWhole = decltype(whole)::value;
        E in[kConvAhead];
        const E *px = x + (long long)tb * c.x_time;
        E *py = y + (size_t)tb * c.dim;
#pragma unroll
        for (int j = 0; j < kConvAhead; ++j) {
            in[j] = px[lo];
            if (kWhole || tb + j + 1 < te) px += c.x_time;
        }
#pragma unroll
        for (int j = 0; j < kConvAhead; ++j) {
            if (!kWhole && tb + j >= te) break;
#pragma unroll
            for (int k = 0; k < W - 1; ++k) win[k] = win[k + 1];
            win[W - 1] = DT::to_float(in[j]);
            float p = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) p = fma_(w[k], win[k], p);
            py[lo] = DT::from_float(SILU ? p * sigmoid_(p) : p);
            py += c.dim;
        }
    };
    int tb = t0;
    for (; tb + kConvAhead <= te; tb += kConvAhead) block(tb, Index<1>());
    if (tb < te) block(tb, Index<0>());
    for (int t = te; t < t1; ++t) (y + (size_t)t * c.dim)[lo] = DT::from_float(0.f);
    if (run == 0 && c.final_state) {
        float fin[W - 1];  // (all read before any is written: final_state may be the buffer of initial_state)
#pragma unroll
        for (int k = 0; k < W - 1; ++k) fin[k] = conv_in<DT, W>(c, (int)b, (long long)len - (W - 1) + k, d);
        E *f = static_cast<E *>(c.final_state) + (size_t)b * (W - 1) * c.dim + d;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) f[(size_t)k * c.dim] = DT::from_float(fin[k]);
    }
}

// dxe[e] = sum_k w[k] gp[e - k] + grad_final, dw[k] = sum_t gp[t] xe[t + k], db = sum gp, with gp = grad_y silu'(p):
// p is formed again from the W rows that the window holds: 27 us at that shape (111 MB at 4.1 TB/s).  Every step that waits for its
// own load, or whose row is zero anyway, costs as much as a block: steps past the end left out 43 -> 29.5 us, the last steps of a run
// loaded together 29.5 -> 27.  Runs of 128 steps leave too few waves (33 us), of 32 more ends to repeat (28 us); fetching the next
// block's rows meanwhile, or a second copy of the block for a run's first rows, costs registers, so waves (48 against 42 us
// then).  partial: [workgroups of one channel group][W + 1][dim].
template <typename DT, int W, bool SILU>
__global__ __launch_bounds__(kConvWaves *kWave) void conv_backward_kernel(const rnntConv c, int runs, int groups, float *partial) {
    typedef typename DT::elem E;
    __shared__ float s_sum[kConvWaves][W + 1][kWave];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int d0 = (int)(blockIdx.x % groups) * kWave + lane;
    const bool ok = d0 < c.dim;
    const int d = ok ? d0 : c.dim - 1;
    const long long item = (long long)(blockIdx.x / groups) * kConvWaves + wave;
    const unsigned lo = d;
    const int run = (int)(item % runs);
    const long long b = item / runs;
    float dw[W], db = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k] = 0.f;
    if (b < c.batch && ok) {
        const int len = clamp_len(c.lengths, (int)b, c.length);
        const int t0 = run * kRunBackward, t1 = t0 + kRunBackward < c.length ? t0 + kRunBackward : c.length;
        float w[W], win[W], gp[W];
#pragma unroll
        for (int k = 0; k < W; ++k) {
            w[k] = c.weight[(size_t)d * W + k];
            gp[k] = 0.f;
            win[k] = 0.f;
        }
        const float bias = c.bias ? c.bias[d] : 0.f;
        const E *x = static_cast<const E *>(c.x) + b * c.x_batch;
        const E *gy = static_cast<const E *>(c.grad_y) + b * c.grad_y_batch;
        E *dx = static_cast<E *>(c.grad_x) + (size_t)b * c.length * c.dim;
        E *di = c.grad_initial ? static_cast<E *>(c.grad_initial) + (size_t)b * (W - 1) * c.dim : nullptr;
        const E *gf = c.grad_final ? static_cast<const E *>(c.grad_final) + (size_t)b * (W - 1) * c.dim + d : nullptr;
        // Step s is newest in the window, gp[k] belongs to step s - (W - 1) + k; row t = s - (W - 1) of dx is then complete.
        auto step = [&](float xs, float gs, bool own) {
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                win[k] = win[k + 1];
                gp[k] = gp[k + 1];
            }
            win[W - 1] = xs;
            float p = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) p = fma_(w[k], win[k], p);
            float v = gs;
            if (SILU) {
                const float sg = sigmoid_(p);
                v *= fma_(p * sg, 1.f - sg, sg);
            }
            gp[W - 1] = v;
            if (own) {  // (steps past t1 belong to the next run)
                db += v;
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k] = fma_(v, win[k], dw[k]);
            }
        };
        auto gradient = [&]() {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) v = fma_(w[W - 1 - k], gp[k], v);
            return v;
        };
        auto finish = [&](int t) {  // row t < len of dx, or of the initial state's gradient
            float v = gradient();
            if (gf && t >= len - (W - 1)) v += DT::to_float(gf[(size_t)(t - (len - (W - 1))) * c.dim]);
            if (t >= 0)
                (dx + (size_t)t * c.dim)[lo] = DT::from_float(v);
            else if (di)
                (di + (size_t)(t + W - 1) * c.dim)[lo] = DT::from_float(v);
        };
        // rows of dxe that this run writes: its own steps' x rows t0 .. t1-1 and, run 0, the W - 1 rows of the initial state
        const int first = run == 0 ? -(W - 1) : t0;
        // (rows past the sequence's end are zero, and steps past it give nothing to any row)
        const int end = len < t1 ? len : t1;
        if (first < len) {
#pragma unroll
            for (int k = 0; k < W - 1; ++k)
                win[k + 1] = first - (W - 1) + k >= -(W - 1) ? conv_in<DT, W>(c, (int)b, (long long)first - (W - 1) + k, d) : 0.f;
            int s = first;
            for (; s < 0; ++s) {  // the initial state's rows enter the window
                step(conv_in<DT, W>(c, (int)b, s, d), 0.f, false);
                gp[W - 1] = 0.f;  // (0 times an infinite derivative)
            }
            // Whole blocks of the sequence and the run (no part of the final state: t < len - (W - 1)): loads first, no tests.  The
            // first begins with rows of the initial state, or of the run before, which are put where row t0 comes next.
            for (; s + kConvAhead <= end; s += kConvAhead) {
                E xin[kConvAhead], gin[kConvAhead];
                const E *px = x + (long long)s * c.x_time, *pg = gy + (long long)s * c.grad_y_time;
#pragma unroll
                for (int j = 0; j < kConvAhead; ++j) {
                    xin[j] = px[lo];
                    gin[j] = pg[lo];
                    px += c.x_time;
                    pg += c.grad_y_time;
                }
                E *pd = dx + (long long)(s - (W - 1)) * c.dim;
                E *begins = run == 0 && di ? di : dx + (long long)t0 * c.dim;
                const long long begins_row = run == 0 && di ? c.dim : 0;
#pragma unroll
                for (int j = 0; j < kConvAhead; ++j) {
                    step(DT::to_float(xin[j]), DT::to_float(gin[j]), true);
                    E *p = j < W - 1 && s == t0 ? begins : pd;
                    p[lo] = DT::from_float(gradient());
                    pd += c.dim;
                    begins += begins_row;
                }
            }
            // what is left, and the W - 1 steps of the next run that these rows take part in
            const int stop = end + W - 1;
            for (; s < stop; s += kConvAhead) {
                E xin[kConvAhead], gin[kConvAhead];
#pragma unroll
                for (int j = 0; j < kConvAhead; ++j) {
                    const long long row = s + j < len ? s + j : (len > 0 ? len - 1 : 0);
                    xin[j] = (x + row * c.x_time)[lo];
                    gin[j] = (gy + row * c.grad_y_time)[lo];
                }
#pragma unroll
                for (int j = 0; j < kConvAhead; ++j) {
                    if (s + j >= stop) break;
                    const bool live = s + j < len;
                    step(live ? DT::to_float(xin[j]) : 0.f, live ? DT::to_float(gin[j]) : 0.f, live && s + j < t1);
                    if (!live) gp[W - 1] = 0.f;
                    if (s + j - (W - 1) >= first) finish(s + j - (W - 1));
                }
            }
        }
        for (int t = len > t0 ? len : t0; t < t1; ++t) (dx + (size_t)t * c.dim)[lo] = DT::from_float(0.f);
    }
#pragma unroll
    for (int k = 0; k < W; ++k) s_sum[wave][k][lane] = dw[k];
    s_sum[wave][W][lane] = db;
    __syncthreads();
    for (int k = wave; k <= W; k += kConvWaves) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kConvWaves; ++q) v += s_sum[q][k][lane];
        if (ok) partial[((size_t)(blockIdx.x / groups) * (W + 1) + k) * c.dim + d] = v;
    }
}

// 64 columns of the partial sums per workgroup, its 16 waves a range of the parts each
template <int W>
__global__ __launch_bounds__(1024) void conv_backward_sum_kernel(const rnntConv c, const float *partial, int parts) {
    __shared__ float s_sum[16][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int i = blockIdx.x * kWave + lane, columns = (W + 1) * c.dim;
    const int per = (parts + 15) / 16, p0 = wave * per, p1 = p0 + per < parts ? p0 + per : parts;
    float s = 0.f;
    if (i < columns) {
#pragma unroll 8
        for (int p = p0; p < p1; ++p) s += partial[(size_t)p * columns + i];
    }
    s_sum[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || i >= columns) return;
    s = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) s += s_sum[q][lane];
    const int k = i / c.dim, d = i - k * c.dim;
    if (k < W)
        c.grad_weight[(size_t)d * W + k] = s;
    else if (c.grad_bias)
        c.grad_bias[d] = s;
}

template <typename DT, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(const rnntConv c) {
    typedef typename DT::elem E;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)c.batch * c.dim) return;
    const int b = (int)(i / c.dim), d = (int)(i - (long long)b * c.dim);
    const E *state = static_cast<const E *>(c.initial_state) + (size_t)b * (W - 1) * c.dim + d;
    E *out = static_cast<E *>(c.final_state) + (size_t)b * (W - 1) * c.dim + d;
    E win[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) win[k] = state[(size_t)k * c.dim];
    win[W - 1] = static_cast<const E *>(c.x)[b * c.x_batch + d];
    float p = c.bias ? c.bias[d] : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) p = fma_(c.weight[(size_t)d * W + k], DT::to_float(win[k]), p);
    static_cast<E *>(c.y)[i] = DT::from_float(c.silu ? p * sigmoid_(p) : p);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) out[(size_t)k * c.dim] = win[k + 1];
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
inline rnntStatus_t launched() { return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED; }

inline size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

inline int groups_of(int dim) { return (dim + kWave - 1) / kWave; }

// (A launch has less than 2^32 threads: 16 a state and group of channels in the backward proper, one a value of B and C, and 16 a
// value of the parameters beside those in the sums.)
inline bool scan_shape_ok(int batch, int length, int dim, int state) {
    if (batch < 1 || length < 1 || dim < 1 || (state != 8 && state != 16 && state != 32) || length > (1 << 30)) return false;
    const long long chunks = (length + kChunk - 1) / kChunk, waves = (long long)batch * groups_of(dim);
    return (long long)batch * chunks < (1ll << 27) && (long long)batch * dim * state < (1ll << 31) && waves * state < (1ll << 28) &&
           waves * chunks < (1ll << 31) &&
           (batch * chunks * kChunk + 1) * 2 * state + ((long long)dim * (state + 2) + 4 * kWave) * 16 < (1ll << 32);
}

// Segments: none while the (sequence, 64 channels) pairs, a wave each, fill the chip; otherwise so many that about 10240 waves walk.
// Both sides of each choice, in us, the kernels of a forward call / of a training pass (1024 channels, 16 states, bf16, all steps live):
//   one segment from 2048 waves on   128 x 500 steps: whole 431 / 1319, cut 498 / 1856; 64 x 500 (1024 waves): 323 / 783 and 258 / 824 (a
//                                    training pass would already rather be whole: 1020 and 1253 with 96 x 500)
//   one segment up to 64 steps       32 x 41: whole 30 / 61, cut 31 / 82; 64 x 64: 43 / 117 and 55 / 152; it costs single sequences
//                                    (1 x 41: 29 / 50 and 23 / 43); 1 x 96, above it: whole 54 / 93, cut 23 / 44
//   10240 waves                      16 x 1500: 198 / 645, with 5120 212 / 674, with 2560 258 / 745, with 20480 199 / 640
//   at least 16 steps, or 32 where   1 x 500 (512 waves of 16): 27 / 57 and, with 32, 39 / 76; 4 x 1500 (6016): 72 / 209 and 72 / 210;
//   16 would give over 2048 waves    1 x 4095 x 1536 channels fp32 (6144): 82 / 236 and 75 / 221; 64 steps are slower in all (60 / 115, 90 / 233, 90 / 236)
//   segments joined from 4096 work-  16 x 1500 (8192): one each 656, two 645, four 642; 32 x 1500: 1222, 1232, 1248.  It bounds the partial sums
//   groups of the backward on        of dA, dD and ddt_bias, which each of them leaves, not the time
inline ScanGeom scan_geometry(int batch, int length, int dim) {
    ScanGeom g = {};
    g.groups = groups_of(dim);
    g.padded = (length + kChunk - 1) / kChunk * kChunk;
    const long long waves = (long long)batch * g.groups;
    const long long want = waves >= 2048 || length <= 64 ? 1 : (10240 + waves - 1) / waves;
    int len = (int)((length + want - 1) / want);
    const int least = waves * ((length + 15) / 16) <= 2048 ? 16 : 32;
    if (len < least) len = least;
    g.seg_len = (len + 15) / 16 * 16;
    g.segments = (length + g.seg_len - 1) / g.seg_len;
    const long long wgs = waves * g.segments;
    g.joined = (int)(wgs > 4096 ? (wgs + 4095) / 4096 : 1);
    if (g.joined > g.segments) g.joined = g.segments;
    g.blocks = (g.segments + g.joined - 1) / g.joined;
    return g;
}

inline size_t rows_bytes(const ScanGeom &g, int batch, int state) {
    return ((size_t)batch * g.padded + 1) * 2 * state * sizeof(float);
}
inline size_t chunk_bytes(const ScanGeom &g, int batch, int dim, int state) {
    return (size_t)batch * (g.padded / kChunk) * dim * state * sizeof(float);
}

// The workspace of a forward call without chunk_states begins with the rows of B and C; with chunk_states they stand behind
// the states there, where the backward call finds them.
struct ScanSpace {
    size_t rows, seg_state, seg_delta, BC, A, D, total;
};
inline ScanSpace scan_space(const ScanGeom &g, int batch, int length, int dim, int state, bool backward) {
    ScanSpace s = {};
    size_t at = 0;
    auto take = [&at](size_t floats) {
        const size_t here = at;
        at += round16(floats * sizeof(float));
        return here;
    };
    if (!backward) s.rows = take(rows_bytes(g, batch, state) / sizeof(float));
    if (g.segments > 1) {
        s.seg_state = take((size_t)batch * g.segments * state * dim);
        s.seg_delta = take((size_t)batch * g.segments * dim);
    }
    if (backward) {
        s.BC = take((size_t)batch * length * g.groups * 2 * state);
        s.A = take((size_t)batch * g.blocks * dim * state);
        s.D = take((size_t)batch * g.blocks * 2 * dim);
    }
    s.total = at;
    return s;
}

inline bool scan_args_ok(const rnntScan *a) {
    return a != nullptr && a->x && a->dt && a->A && a->B && a->C && scan_shape_ok(a->batch, a->length, a->dim, a->state);
}

template <int N, bool BACKWARD>
void launch_join(const rnntScan &a, const ScanGeom &g, hipStream_t st) {
    const long long n = (long long)a.batch * a.dim * (N / 4);
    const dim3 grid((unsigned)((n + kWave - 1) / kWave));
    if (g.segments <= kJoinAhead)
        hipLaunchKernelGGL((scan_join_kernel<N, BACKWARD, 1>), grid, dim3(kWave), 0, st, a, g);
    else
        hipLaunchKernelGGL((scan_join_kernel<N, BACKWARD, kJoinWaves>), grid, dim3(kJoinWaves * kWave), 0, st, a, g);
}

template <typename DT, int N>
rnntStatus_t scan_forward(const rnntScan &a, hipStream_t st) {
    ScanGeom g = scan_geometry(a.batch, a.length, a.dim);
    const unsigned grid = (unsigned)((long long)a.batch * g.segments * g.groups);
    const ScanSpace s = scan_space(g, a.batch, a.length, a.dim, N, false);
    char *ws = static_cast<char *>(a.workspace);
    g.rows = a.chunk_states ? a.chunk_states + chunk_bytes(g, a.batch, a.dim, N) / sizeof(float) : reinterpret_cast<float *>(ws + s.rows);
    const long long values = ((long long)a.batch * g.padded + 1) * 2 * N;
    hipLaunchKernelGGL((scan_rows_kernel<DT, N>), dim3((unsigned)((values + 255) / 256)), dim3(256), 0, st, a, g);
    if (g.segments > 1) {
        g.seg_state = reinterpret_cast<float *>(ws + s.seg_state);
        g.seg_delta = reinterpret_cast<float *>(ws + s.seg_delta);
        hipLaunchKernelGGL((scan_forward_kernel<DT, N, true>), dim3(grid), dim3(64), 0, st, a, g);
        launch_join<N, false>(a, g, st);
    }
    hipLaunchKernelGGL((scan_forward_kernel<DT, N, false>), dim3(grid), dim3(64), 0, st, a, g);
    return launched();
}

template <typename DT, int N>
rnntStatus_t scan_backward(const rnntScan &a, hipStream_t st) {
    ScanGeom g = scan_geometry(a.batch, a.length, a.dim);
    const ScanSpace s = scan_space(g, a.batch, a.length, a.dim, N, true);
    char *ws = static_cast<char *>(a.workspace);
    g.rows = const_cast<float *>(a.chunk_states) + chunk_bytes(g, a.batch, a.dim, N) / sizeof(float);
    const unsigned grid = (unsigned)((long long)a.batch * g.segments * g.groups);
    if (g.segments > 1) {
        g.seg_state = reinterpret_cast<float *>(ws + s.seg_state);
        g.seg_delta = reinterpret_cast<float *>(ws + s.seg_delta);
        hipLaunchKernelGGL((scan_backward_local_kernel<DT, N>), dim3(grid), dim3(64), 0, st, a, g);
        launch_join<N, true>(a, g, st);
    }
    const ScanPartials p = {reinterpret_cast<float *>(ws + s.BC), reinterpret_cast<float *>(ws + s.A),
                            reinterpret_cast<float *>(ws + s.D)};
    hipLaunchKernelGGL((scan_backward_kernel<DT, N>), dim3((unsigned)((long long)a.batch * g.blocks * g.groups)), dim3(N * 16), 0, st, a, g, p);
    const unsigned bc = (unsigned)(((long long)a.batch * a.length * 2 * N + 1023) / 1024);
    const unsigned pa = (unsigned)(((long long)a.dim * (N + 2) + kWave - 1) / kWave);
    hipLaunchKernelGGL((scan_backward_sum_kernel<DT, N>), dim3(bc + pa), dim3(1024), 0, st, a, g, p, bc);
    return launched();
}

template <typename DT, int N>
rnntStatus_t scan_step(const rnntScan &a, hipStream_t st) {
    const long long n = (long long)a.batch * a.dim * (N / 4);
    hipLaunchKernelGGL((scan_step_kernel<DT, N>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    return launched();
}

#define SCAN_BY_STATE(FN, DT)                          \
    switch (a.state) {                                 \
        case 8: return FN<DT, 8>(a, st);               \
        case 16: return FN<DT, 16>(a, st);             \
        case 32: return FN<DT, 32>(a, st);             \
        default: return RNNT_STATUS_INVALID_VALUE;     \
    }
#define SCAN_DISPATCH(FN)                                                      \
    do {                                                                       \
        const rnntScan &a = *scan;                                             \
        hipStream_t st = static_cast<hipStream_t>(scan->stream);               \
        switch (a.dtype) {                                                     \
            case RNNT_DTYPE_F32: SCAN_BY_STATE(FN, F32)                        \
            case RNNT_DTYPE_BF16: SCAN_BY_STATE(FN, BF16)                      \
            case RNNT_DTYPE_F16: SCAN_BY_STATE(FN, F16)                        \
            default: return RNNT_STATUS_INVALID_VALUE;                         \
        }                                                                      \
    } while (0)

inline int runs_of(int length, int run) { return (length + run - 1) / run; }
inline long long conv_items(int batch, int length, int run) {  // workgroups per channel group
    return ((long long)batch * runs_of(length, run) + kConvWaves - 1) / kConvWaves;
}

inline bool conv_shape_ok(int batch, int length, int dim, int width) {
    return batch >= 1 && length >= 1 && dim >= 1 && width >= 2 && width <= 4 && length <= (1 << 30) &&
           (long long)batch * length < (1ll << 31) && (long long)batch * dim < (1ll << 31) &&
           dim < (1 << 25) && conv_items(batch, length, kRunForward) * groups_of(dim) < (1ll << 24);  // (less than 2^32 threads)
}

template <typename DT, int W>
rnntStatus_t conv_forward(const rnntConv &c, hipStream_t st) {
    const unsigned grid = (unsigned)(conv_items(c.batch, c.length, kRunForward) * groups_of(c.dim));
    hipLaunchKernelGGL((c.silu ? conv_forward_kernel<DT, W, true> : conv_forward_kernel<DT, W, false>), dim3(grid), dim3(kConvWaves * kWave), 0, st, c, runs_of(c.length, kRunForward),
                       groups_of(c.dim));
    return launched();
}
template <typename DT, int W>
rnntStatus_t conv_backward(const rnntConv &c, hipStream_t st) {
    const int parts = (int)conv_items(c.batch, c.length, kRunBackward);
    float *partial = static_cast<float *>(c.workspace);
    hipLaunchKernelGGL((c.silu ? conv_backward_kernel<DT, W, true> : conv_backward_kernel<DT, W, false>), dim3((unsigned)((long long)parts * groups_of(c.dim))), dim3(kConvWaves * kWave), 0,
                       st, c, runs_of(c.length, kRunBackward), groups_of(c.dim), partial);
    hipLaunchKernelGGL((conv_backward_sum_kernel<W>), dim3((unsigned)(((long long)(W + 1) * c.dim + kWave - 1) / kWave)), dim3(1024), 0,
                       st, c, static_cast<const float *>(partial), parts);
    return launched();
}
template <typename DT, int W>
rnntStatus_t conv_step(const rnntConv &c, hipStream_t st) {
    const long long n = (long long)c.batch * c.dim;
    hipLaunchKernelGGL((conv_step_kernel<DT, W>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, c);
    return launched();
}

#define CONV_BY_WIDTH(FN, DT)                          \
    switch (c.width) {                                 \
        case 2: return FN<DT, 2>(c, st);               \
        case 3: return FN<DT, 3>(c, st);               \
        case 4: return FN<DT, 4>(c, st);               \
        default: return RNNT_STATUS_INVALID_VALUE;     \
    }
#define CONV_DISPATCH(FN)                                                      \
    do {                                                                       \
        const rnntConv &c = *conv;                                             \
        hipStream_t st = static_cast<hipStream_t>(conv->stream);               \
        switch (c.dtype) {                                                     \
            case RNNT_DTYPE_F32: CONV_BY_WIDTH(FN, F32)                        \
            case RNNT_DTYPE_BF16: CONV_BY_WIDTH(FN, BF16)                      \
            case RNNT_DTYPE_F16: CONV_BY_WIDTH(FN, F16)                        \
            default: return RNNT_STATUS_INVALID_VALUE;                         \
        }                                                                      \
    } while (0)

}  // namespace

extern "C" {

rnntStatus_t rnnt_selective_scan_states_size(int batch, int length, int dim, int state, size_t *size_bytes) {
    if (size_bytes == nullptr || !scan_shape_ok(batch, length, dim, state)) return RNNT_STATUS_INVALID_VALUE;
    const ScanGeom g = scan_geometry(batch, length, dim);
    *size_bytes = chunk_bytes(g, batch, dim, state) + rows_bytes(g, batch, state);
    return RNNT_STATUS_SUCCESS;
}

rnntStatus_t rnnt_selective_scan_workspace_size(int batch, int length, int dim, int state, int backward, size_t *size_bytes) {
    if (size_bytes == nullptr || !scan_shape_ok(batch, length, dim, state)) return RNNT_STATUS_INVALID_VALUE;
    *size_bytes = scan_space(scan_geometry(batch, length, dim), batch, length, dim, state, backward != 0).total;
    return RNNT_STATUS_SUCCESS;
}

rnntStatus_t rnnt_selective_scan_forward(const rnntScan *scan) {
    if (!scan_args_ok(scan) || scan->y == nullptr || !scan->workspace || !aligned16(scan->workspace) ||
        (scan->chunk_states && !aligned16(scan->chunk_states)))
        return RNNT_STATUS_INVALID_VALUE;
    SCAN_DISPATCH(scan_forward);
}

rnntStatus_t rnnt_selective_scan_backward(const rnntScan *scan) {
    if (!scan_args_ok(scan) || !scan->grad_y || !scan->chunk_states || !aligned16(scan->chunk_states) || !scan->grad_x ||
        !scan->grad_dt || !scan->grad_A || !scan->grad_B || !scan->grad_C || (scan->z == nullptr) != (scan->grad_z == nullptr) ||
        !scan->workspace || !aligned16(scan->workspace))
        return RNNT_STATUS_INVALID_VALUE;
    SCAN_DISPATCH(scan_backward);
}

rnntStatus_t rnnt_selective_scan_step(const rnntScan *scan) {
    if (scan == nullptr || !scan->x || !scan->dt || !scan->A || !scan->B || !scan->C || !scan->y || !scan->initial_state ||
        !scan->final_state || !scan_shape_ok(scan->batch, 1, scan->dim, scan->state))
        return RNNT_STATUS_INVALID_VALUE;
    SCAN_DISPATCH(scan_step);
}

rnntStatus_t rnnt_causal_conv_workspace_size(int batch, int length, int dim, int width, size_t *size_bytes) {
    if (size_bytes == nullptr || !conv_shape_ok(batch, length, dim, width)) return RNNT_STATUS_INVALID_VALUE;
    *size_bytes = (size_t)conv_items(batch, length, kRunBackward) * (width + 1) * dim * sizeof(float);
    return RNNT_STATUS_SUCCESS;
}

rnntStatus_t rnnt_causal_conv_forward(const rnntConv *conv) {
    if (conv == nullptr || !conv->x || !conv->weight || !conv->y ||
        !conv_shape_ok(conv->batch, conv->length, conv->dim, conv->width))
        return RNNT_STATUS_INVALID_VALUE;
    CONV_DISPATCH(conv_forward);
}

rnntStatus_t rnnt_causal_conv_backward(const rnntConv *conv) {
    if (conv == nullptr || !conv->x || !conv->weight || !conv->grad_y || !conv->grad_x || !conv->grad_weight || !conv->workspace ||
        !aligned16(conv->workspace) || !conv_shape_ok(conv->batch, conv->length, conv->dim, conv->width))
        return RNNT_STATUS_INVALID_VALUE;
    CONV_DISPATCH(conv_backward);
}

rnntStatus_t rnnt_causal_conv_step(const rnntConv *conv) {
    if (conv == nullptr || !conv->x || !conv->weight || !conv->y || !conv->initial_state || !conv->final_state ||
        !conv_shape_ok(conv->batch, 1, conv->dim, conv->width))
        return RNNT_STATUS_INVALID_VALUE;
    CONV_DISPATCH(conv_step);
}

}  // extern "C"
