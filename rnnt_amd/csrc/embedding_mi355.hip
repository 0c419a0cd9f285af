// embedding_mi355.hip — token embedding of a prediction network on MI355X (gfx950): the lookup with its scale, and its
// gradient by sorted tokens.
//
// The reference's prediction network begins with nn.Embedding (src/decoder/decoder.py:9).  Forward copies one row per
// token.  Backward sums the gradient rows of each token.  Adding them with atomics would let their order, and with it the
// last bits, vary from run to run, and would serialise on the frequent tokens (a label sequence is full of them);
// instead the positions are sorted by token first (stable: position order), the sorted list is cut into equal pieces
// whatever the tokens' frequencies, each piece sums its runs of equal tokens in fp32 registers, and the runs that
// cross pieces are joined in order.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/rnnt_mi355.h"
#include "elem_types.h"

namespace {

using namespace rnnt_mi355_detail;

constexpr int kBlock = 256;
constexpr int kBatch = 8;         // gradient rows loaded at once
constexpr int kListMax = 2048;    // up to this many positions are not sorted: every workgroup lists its own rows' positions
constexpr int kListRows = 16, kListWaves = 8, kListAlone = 64;
constexpr int kRankMax = 4096;    // up to this many positions are sorted by counting smaller ones
constexpr int kRankRows = 64;     // rows of the gradient that a workgroup of the counting kernel clears
constexpr int kSortItems = 1024;  // positions per workgroup and pass of the radix sort
constexpr int kSortMany = 3 << 17;  // from so many positions on the workgroups' counts are summed by a launch of their own
constexpr int kJoinWaves = 8, kJoinAlone = 64;
constexpr int kDigits = 256;

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ long long token_at(const void *tokens, int tokens_64, long long i) {
    return tokens_64 ? static_cast<const long long *>(tokens)[i] : (long long)static_cast<const int *>(tokens)[i];
}

// sort key: the token, or `vocab` (last) for a position that adds to no row
__device__ __forceinline__ int key_at(const void *tokens, int tokens_64, long long i, int vocab, long long padding) {
    const long long t = token_at(tokens, tokens_64, i);
    return t >= 0 && t < vocab && t != padding ? (int)t : vocab;
}

// a lane's piece of a row: VEC elements
template <typename DT, int VEC>
__device__ __forceinline__ void load_piece(const typename DT::elem *p, float (&f)[VEC]) {
    if constexpr (VEC == 1)
        f[0] = DT::to_float(*p);
    else
        DT::unpack(*reinterpret_cast<const u32x4 *>(p), f);
}
template <typename DT, int VEC>
__device__ __forceinline__ void store_piece(typename DT::elem *p, const float (&f)[VEC]) {
    if constexpr (VEC == 1)
        *p = DT::from_float(f[0]);
    else
        *reinterpret_cast<u32x4 *>(p) = DT::pack(f);
}

// Rows are shared out to groups of 2^shift lanes; a group walks its row in pieces of VEC elements per lane.  Bound by
// memory: 65 408 tokens of 512 fp32 values out of 16 384 rows 36 us (168 MB: 4.6 TB/s, a large copy runs at 4.84);
// 1312 tokens of 512 bf16 values 2.6 us.
template <typename DT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_forward_kernel(const void *__restrict__ tokens, int tokens_64, long long n,
                                                               const typename DT::elem *__restrict__ weight,
                                                               long long weight_stride, int vocab, int dim, float scale,
                                                               typename DT::elem *__restrict__ out, int shift) {
    const int sub = threadIdx.x & ((1 << shift) - 1);
    const long long i = ((long long)blockIdx.x * kBlock + threadIdx.x) >> shift;
    if (i >= n) return;
    const long long t = token_at(tokens, tokens_64, i);
    const bool ok = t >= 0 && t < vocab;
    const typename DT::elem *row = weight + (ok ? t : 0) * weight_stride;
    for (int c = sub * VEC; c < dim; c += VEC << shift) {
        float f[VEC];
        load_piece<DT, VEC>(row + c, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = ok ? f[j] * scale : __builtin_nanf("");
        store_piece<DT, VEC>(out + (size_t)i * dim + c, f);
    }
}

// ---- sorting ---------------------------------------------------------------------------------------------------------
// Few positions: a position's place is the number of positions before it in the order, counted against all others:
// n^2 comparisons in one launch, nothing to wait for.  A workgroup places 64 positions (its lanes), each wave against a
// quarter of the keys, four keys to an LDS read; "equal and earlier" is decided per block of keys, not per key.
// 1312 positions and 4232 rows to clear: 8 us, bound by latency.
// The workgroups from rank_blocks on clear 64 rows of the gradient each, those whose token no position holds.
template <typename DT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_rank_kernel(const void *__restrict__ tokens, int tokens_64, int n, int vocab,
                                                            long long padding, int *__restrict__ sorted, int *__restrict__ order,
                                                            typename DT::elem *__restrict__ grad_weight, int dim, int rank_blocks) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    constexpr int kWaves = kBlock / kWave;
    __shared__ i32x4 s_key[kRankMax / 4];
    __shared__ int s_rank[kWaves][kWave];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if ((int)blockIdx.x >= rank_blocks) {
        const int v0 = ((int)blockIdx.x - rank_blocks) * kRankRows;
        int *held = &s_rank[0][0];
        if (threadIdx.x < kRankRows) held[threadIdx.x] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kBlock) {
            const int k = key_at(tokens, tokens_64, j, vocab, padding) - v0;
            if (k >= 0 && k < kRankRows) held[k] = 1;
        }
        __syncthreads();
        const float zero[VEC] = {};
        for (int r = wave; r < kRankRows && v0 + r < vocab; r += kWaves) {
            if (held[r]) continue;
            for (int c = lane * VEC; c < dim; c += kWave * VEC) store_piece<DT, VEC>(grad_weight + (size_t)(v0 + r) * dim + c, zero);
        }
        return;
    }
    int *keys = reinterpret_cast<int *>(s_key);
    const int padded = (n + 3) & ~3;
    for (int j = threadIdx.x; j < padded; j += kBlock) keys[j] = j < n ? key_at(tokens, tokens_64, j, vocab, padding) : 0x7fffffff;
    __syncthreads();
    const int i0 = blockIdx.x * kWave, i = i0 + lane;
    const int key = i < n ? keys[i] : 0x7fffffff;
    const int quads = padded / 4, per = (quads + kWaves - 1) / kWaves;
    const int q0 = wave * per, q1 = q0 + per < quads ? q0 + per : quads;
    // quads [q0, qa): before this block of positions, equal keys count; [qa, qb): inside; [qb, q1): after, they do not
    const int qa = min(max(i0 / 4, q0), q1), qb = min(max((i0 + kWave) / 4, q0), q1);
    int rank = 0;
#pragma unroll 8
    for (int q = q0; q < qa; ++q) {
        const i32x4 k = s_key[q];
        rank += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key);
    }
    for (int q = qa; q < qb; ++q) {
        const i32x4 k = s_key[q];
        const int j = q * 4;
        rank += (k.x < key || (k.x == key && j < i)) + (k.y < key || (k.y == key && j + 1 < i)) +
                (k.z < key || (k.z == key && j + 2 < i)) + (k.w < key || (k.w == key && j + 3 < i));
    }
#pragma unroll 8
    for (int q = max(qb, q0); q < q1; ++q) {
        const i32x4 k = s_key[q];
        rank += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
    }
    s_rank[wave][lane] = rank;
    __syncthreads();
    if (wave != 0 || i >= n) return;
    rank = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) rank += s_rank[w][lane];
    sorted[rank] = key;
    order[rank] = i;
}

// Many positions: radix sort from the lowest digit, 8 bits per pass, two launches per pass (65 408 positions: 4 + 7 us the
// first pass, 4 + 8 us the second; bound by the launches' latencies, not by their 0.5 MB).  A workgroup's wave w owns
// its w-th quarter; lanes with the same digit find each other with 8 ballots, so that ranks follow the position.
// A workgroup adds up the counts of those before it itself, which is quadratic in their number: from kSortMany positions
// on a launch between the two forms the sums (MANY).  Whole backward passes of 64 fp32 columns, without and with it: 262 144
// positions 56 and 64 us, 524 288 82 and 70, 4 194 304 1477 and 458.
template <bool FIRST>
__device__ __forceinline__ int sort_key(const void *src, int tokens_64, long long i, int vocab, long long padding) {
    return FIRST ? key_at(src, tokens_64, i, vocab, padding) : static_cast<const int *>(src)[i];
}

template <bool FIRST>
__global__ __launch_bounds__(kBlock) void embed_digit_kernel(const void *__restrict__ src, int tokens_64, int n, int vocab,
                                                             long long padding, int bit, int *__restrict__ counts) {
    __shared__ int s_count[kDigits];
    s_count[threadIdx.x] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * kSortItems;
    for (int k = threadIdx.x; k < kSortItems; k += kBlock)
        if (base + k < n) atomicAdd(&s_count[(sort_key<FIRST>(src, tokens_64, base + k, vocab, padding) >> bit) & (kDigits - 1)], 1);
    __syncthreads();
    counts[(size_t)blockIdx.x * kDigits + threadIdx.x] = s_count[threadIdx.x];
}

// counts[w][digit] <- the sum over the workgroups before w, counts[parts][digit] <- over all; a workgroup per digit, its
// threads a range each.
__global__ __launch_bounds__(kBlock) void embed_prefix_kernel(int *__restrict__ counts, int parts) {
    __shared__ int s_sum[kBlock];
    const int per = (parts + kBlock - 1) / kBlock;
    const int w0 = (int)threadIdx.x * per < parts ? (int)threadIdx.x * per : parts, w1 = w0 + per < parts ? w0 + per : parts;
    int *column = counts + blockIdx.x;
    int sum = 0;
#pragma unroll 8
    for (int w = w0; w < w1; ++w) sum += column[(size_t)w * kDigits];
    s_sum[threadIdx.x] = sum;
    __syncthreads();
    for (int step = 1; step < kBlock; step <<= 1) {
        const int v = (int)threadIdx.x >= step ? s_sum[threadIdx.x - step] : 0;
        __syncthreads();
        s_sum[threadIdx.x] += v;
        __syncthreads();
    }
    int before = s_sum[threadIdx.x] - sum;
    for (int w = w0; w < w1; ++w) {
        const int c = column[(size_t)w * kDigits];
        column[(size_t)w * kDigits] = before;
        before += c;
    }
    if (threadIdx.x == kBlock - 1) column[(size_t)parts * kDigits] = before;
}

__device__ __forceinline__ unsigned long long same_digit(int digit, bool live) {
    unsigned long long peers = __ballot(live);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
        const unsigned long long set = __ballot((digit >> bit) & 1);
        peers &= (digit >> bit) & 1 ? set : ~set;
    }
    return peers;
}

template <bool FIRST, bool MANY>
__global__ __launch_bounds__(kBlock) void embed_place_kernel(const void *__restrict__ src, int tokens_64, int n, int vocab,
                                                             long long padding, int bit, const int *__restrict__ counts,
                                                             const int *__restrict__ order_in, int *__restrict__ sorted,
                                                             int *__restrict__ order) {
    constexpr int kWaves = kBlock / kWave, kRounds = kSortItems / kBlock;
    __shared__ int s_base[kWaves][kDigits];
    __shared__ int s_total[kDigits];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const long long base = (long long)blockIdx.x * kSortItems + wave * (kSortItems / kWaves);
    int before = 0, total = 0;  // of digit threadIdx.x: in the workgroups before this one, in all
    if constexpr (MANY) {
        before = counts[(size_t)blockIdx.x * kDigits + threadIdx.x];
        total = counts[(size_t)gridDim.x * kDigits + threadIdx.x];
    } else {
#pragma unroll 16
        for (int w = 0; w < (int)gridDim.x; ++w) {
            const int c = counts[(size_t)w * kDigits + threadIdx.x];
            before += w < (int)blockIdx.x ? c : 0;
            total += c;
        }
    }
    s_total[threadIdx.x] = total;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s_base[w][threadIdx.x] = 0;
    __syncthreads();
    for (int step = 1; step < kDigits; step <<= 1) {  // inclusive sums over the digits
        const int v = (int)threadIdx.x >= step ? s_total[threadIdx.x - step] : 0;
        __syncthreads();
        s_total[threadIdx.x] += v;
        __syncthreads();
    }
    int key[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const long long i = base + r * kWave + lane;
        key[r] = i < n ? sort_key<FIRST>(src, tokens_64, i, vocab, padding) : -1;
        if (i < n) atomicAdd(&s_base[wave][(key[r] >> bit) & (kDigits - 1)], 1);
    }
    __syncthreads();
    {
        int at = s_total[threadIdx.x] - total + before;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int c = s_base[w][threadIdx.x];
            s_base[w][threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const long long i = base + r * kWave + lane;
        const bool live = i < n;
        const int digit = (key[r] >> bit) & (kDigits - 1);
        const unsigned long long peers = same_digit(digit, live);
        const int ahead = __popcll(peers & ((1ull << lane) - 1));
        int at = 0;
        if (live) at = s_base[wave][digit] + ahead;
        // (a wave's LDS accesses stay in order: all lanes have read before the first of each digit moves its base on)
        __builtin_amdgcn_wave_barrier();
        if (live && ahead == 0) s_base[wave][digit] += __popcll(peers);
        __builtin_amdgcn_wave_barrier();
        if (live) {
            sorted[at] = key[r];
            order[at] = FIRST ? (int)i : order_in[i];
        }
    }
}

// ---- sums ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int lower_bound(const int *sorted, int n, int key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sorted[mid] < key)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

// Groups of 2^shift lanes.  [0, pieces * slices): a slice of the columns of a piece of sorted positions each.  A run of
// equal tokens inside the piece is written out; the part of a run that began in an earlier piece goes to
// partial[piece][0], the part of one that begins here and goes on to partial[piece][1].  Rows are loaded kBatch at a
// time: a piece is a chain of dependent additions, but its loads are not.
// The waves behind them (16 rows each) clear the rows that no position holds: a lane searches for each.
// Bound by memory: 65 408 rows of 512 fp32 values 24 us (167 MB: 7 TB/s, part of the rows still in the last-level cache).
template <typename DT, int VEC>
__global__ __launch_bounds__(kBlock) void embed_sum_kernel(const int *__restrict__ sorted, const int *__restrict__ order, int n,
                                                           const typename DT::elem *__restrict__ grad, long long grad_stride,
                                                           int vocab, int dim, float scale,
                                                           typename DT::elem *__restrict__ grad_weight,
                                                           float *__restrict__ partial, int piece, int pieces, int slices, int shift,
                                                           unsigned sum_blocks) {
    if (blockIdx.x >= sum_blocks) {
        const int lane = threadIdx.x & (kWave - 1);
        const long long wave = (long long)(blockIdx.x - sum_blocks) * (kBlock / kWave) + threadIdx.x / kWave;
        const long long v0 = wave * 16;
        const int v = (int)(v0 + (lane & 15) < vocab ? v0 + (lane & 15) : vocab - 1);
        const int at = lower_bound(sorted, n, v);
        const unsigned long long held = __ballot(at < n && sorted[at] == v);
        const float zero[VEC] = {};
        for (int r = 0; r < 16 && v0 + r < vocab; ++r) {
            if (held >> r & 1) continue;
            for (int c = lane * VEC; c < dim; c += kWave * VEC) store_piece<DT, VEC>(grad_weight + (size_t)(v0 + r) * dim + c, zero);
        }
        return;
    }
    const int sub = threadIdx.x & ((1 << shift) - 1);
    const long long group = ((long long)blockIdx.x * kBlock + threadIdx.x) >> shift;
    const long long p = group / slices;
    if (p >= pieces) return;
    const int c = ((int)(group - p * slices) << shift) * VEC + sub * VEC;
    if (c >= dim) return;
    const int begin = (int)p * piece, end = begin + piece < n ? begin + piece : n;
    const int prev = begin > 0 ? sorted[begin - 1] : -1, next = end < n ? sorted[end] : -1;
    float acc[VEC] = {};
    int cur = sorted[begin];
    bool from_before = cur == prev;
    auto close = [&](bool goes_on) {
        if (cur == vocab) return;
        if (from_before || goes_on) {
            float *o = partial + ((size_t)p * 2 + (from_before ? 0 : 1)) * dim + c;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = acc[j];
        } else {
            float f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = acc[j] * scale;
            store_piece<DT, VEC>(grad_weight + (size_t)cur * dim + c, f);
        }
    };
    for (int k0 = begin; k0 < end && cur != vocab; k0 += kBatch) {
        int tok[kBatch];
        float f[kBatch][VEC];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int at = k0 + k < end ? k0 + k : end - 1;
            tok[k] = sorted[at];
            load_piece<DT, VEC>(grad + (size_t)order[at] * grad_stride + c, f[k]);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (k0 + k >= end || cur == vocab) break;
            if (tok[k] != cur) {
                close(false);
                cur = tok[k];
                from_before = false;
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += f[k][j];
        }
    }
    close(cur == next);
}

// The runs that cross pieces, joined by the wave of the piece a run begins in, in order; a run of more than kJoinAlone
// pieces (a token that is a tenth of all positions) by the whole workgroup, each wave a range of its pieces in order, then
// the waves' sums in order.  grid.y: slices of 64 VEC columns.  8 us there: a chain of searching and two loads; a workgroup
// per piece took 17.
template <typename DT, int VEC>
__global__ __launch_bounds__(kJoinWaves *kWave) void embed_join_kernel(const int *__restrict__ sorted, int n, int vocab, int dim,
                                                                       float scale, typename DT::elem *__restrict__ grad_weight,
                                                                       const float *__restrict__ partial, int piece, int pieces) {
    __shared__ float s_acc[kJoinWaves][kWave * VEC];
    __shared__ int s_last[kJoinWaves], s_tok[kJoinWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int p = blockIdx.x * kJoinWaves + wave, begin = p * piece, end = begin + piece;
    const int c = (int)blockIdx.y * kWave * VEC + lane * VEC;
    auto add_parts = [&](int p0, int p1, float (&acc)[VEC]) {  // the parts [p0, p1) of a run that began earlier
#pragma unroll 8
        for (int q = p0; q < p1; ++q) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += partial[(size_t)q * 2 * dim + c + j];
        }
    };
    auto first_part = [&](int q, float (&acc)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = partial[((size_t)q * 2 + 1) * dim + c + j];
    };
    int last = -1, tok = vocab;  // pieces p + 1 .. last hold parts of the run that begins in piece p and goes on
    if (p < pieces && end < n) {
        tok = sorted[end - 1];
        const bool goes_on = tok != vocab && sorted[end] == tok;
        if (goes_on && !(sorted[begin] == tok && begin > 0 && sorted[begin - 1] == tok)) {
            last = p + 1;
            while (last < p + 4 && (last + 1) * (long long)piece < n && sorted[(last + 1) * piece] == tok) ++last;
            if (last == p + 4) last = (lower_bound(sorted, n, tok + 1) - 1) / piece;
        }
    }
    const bool alone = last >= 0 && last - p <= kJoinAlone;
    if (alone && c < dim) {
        float acc[VEC];
        first_part(p, acc);
        add_parts(p + 1, last + 1, acc);
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] *= scale;
        store_piece<DT, VEC>(grad_weight + (size_t)tok * dim + c, acc);
    }
    if (lane == 0) {
        s_last[wave] = alone ? -1 : last;
        s_tok[wave] = tok;
    }
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
        if (s_last[w] < 0) continue;  // (the same for the whole workgroup)
        const int from = blockIdx.x * kJoinWaves + w, to = s_last[w];
        const int per = (to - from + kJoinWaves - 1) / kJoinWaves;
        const int p0 = from + 1 + wave * per, p1 = p0 + per < to + 1 ? p0 + per : to + 1;
        float acc[VEC] = {};
        if (c < dim) {
            if (wave == 0) first_part(from, acc);
            add_parts(p0, p1, acc);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) s_acc[wave][lane * VEC + j] = acc[j];
        __syncthreads();
        if (wave == 0 && c < dim) {
            float f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float s = 0.f;
#pragma unroll
                for (int q = 0; q < kJoinWaves; ++q) s += s_acc[q][lane * VEC + j];
                f[j] = s * scale;
            }
            store_piece<DT, VEC>(grad_weight + (size_t)s_tok[w] * dim + c, f);
        }
        __syncthreads();
    }
}

// Few positions and few to a token: one launch, no sorting.  A workgroup has 16 rows of the gradient: it goes through all
// tokens, lists in LDS the positions of its rows (each wave an eighth of the positions, so that the list is in order),
// and sums them, a wave to a row; a row of more than kListAlone positions is shared by the waves, a range each, and their
// sums are added in order.  1312 tokens, 4232 rows of 512 bf16 values: 8.9 us in one launch; counting, summing and joining
// took 16 in three.
template <typename DT, int VEC>
__global__ __launch_bounds__(kListWaves *kWave) void embed_list_kernel(const void *__restrict__ tokens, int tokens_64, int n, int vocab,
                                                                       long long padding, const typename DT::elem *__restrict__ grad,
                                                                       long long grad_stride, int dim, float scale,
                                                                       typename DT::elem *__restrict__ grad_weight) {
    constexpr int kPart = kListMax / kListWaves;
    __shared__ int s_found[kListWaves][kPart], s_count[kListWaves], s_list[kListMax];
    __shared__ int s_many[kListRows];
    __shared__ float s_acc[kListWaves][kWave * VEC];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int v0 = blockIdx.x * kListRows;
    const int c = (int)blockIdx.y * kWave * VEC + lane * VEC;
    {
        const int per = (n + kListWaves - 1) / kListWaves, i0 = wave * per, i1 = i0 + per < n ? i0 + per : n;
        int count = 0, key[kPart / kWave];
#pragma unroll
        for (int u = 0; u < kPart / kWave; ++u) {
            const int i = i0 + u * kWave + lane;
            key[u] = i < i1 ? key_at(tokens, tokens_64, i, vocab, padding) : -1;
        }
#pragma unroll
        for (int u = 0; u < kPart / kWave; ++u) {
            const int i = i0 + u * kWave + lane, k = key[u] < 0 ? -1 : key[u] - v0;
            const bool mine = k >= 0 && k < kListRows && v0 + k < vocab;  // (the key of a position without a row is vocab)
            const unsigned long long found = __ballot(mine);
            if (mine) s_found[wave][count + __popcll(found & ((1ull << lane) - 1))] = i * kListRows + k;
            count += __popcll(found);
        }
        if (lane == 0) s_count[wave] = count;
        if (threadIdx.x < kListRows) s_many[threadIdx.x] = 0;
    }
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kListWaves; ++w) {
        const int k = s_count[w];
        before += w < wave ? k : 0;
        total += k;
    }
    for (int k = lane; k < s_count[wave]; k += kWave) s_list[before + k] = s_found[wave][k];
    __syncthreads();

    auto matches = [&](int r, int b, int &entry) {
        entry = b + lane < total ? s_list[b + lane] : -1;
        return __ballot(entry >= 0 && entry % kListRows == r);
    };
    // the sum of row r's positions [from, to) in order
    auto sum = [&](int r, int from, int to, float (&acc)[VEC]) {
        int seen = 0;
        for (int b = 0; b < total && seen < to; b += kWave) {
            int entry;
            unsigned long long found = matches(r, b, entry);
            const int here = __popcll(found);
            if (seen + here > from) {
                for (int skip = seen; skip < from; ++skip) found &= found - 1;
                int left = (seen + here < to ? seen + here : to) - (seen > from ? seen : from);
                while (left > 0) {
                    float f[kBatch][VEC];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        if (k < left) {
                            const int at = __builtin_amdgcn_readlane(entry, __builtin_ctzll(found)) / kListRows;
                            found &= found - 1;
                            if (c < dim) load_piece<DT, VEC>(grad + (size_t)at * grad_stride + c, f[k]);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        if (k < left) {
#pragma unroll
                            for (int j = 0; j < VEC; ++j) acc[j] += f[k][j];
                        }
                    }
                    left -= kBatch;
                }
            }
            seen += here;
        }
    };
    auto store = [&](int r, float (&acc)[VEC]) {
        if (c >= dim) return;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] *= scale;
        store_piece<DT, VEC>(grad_weight + (size_t)(v0 + r) * dim + c, acc);
    };
    for (int r = wave; r < kListRows && v0 + r < vocab; r += kListWaves) {
        int many = 0, entry;
        for (int b = 0; b < total; b += kWave) many += __popcll(matches(r, b, entry));
        if (many > kListAlone) {
            if (lane == 0) s_many[r] = many;
            continue;
        }
        float acc[VEC] = {};
        sum(r, 0, many, acc);
        store(r, acc);
    }
    __syncthreads();
    for (int r = 0; r < kListRows; ++r) {
        const int many = s_many[r];
        if (many == 0) continue;  // (the same for the whole workgroup)
        const int per = (many + kListWaves - 1) / kListWaves, from = wave * per, to = from + per < many ? from + per : many;
        float acc[VEC] = {};
        if (from < to) sum(r, from, to, acc);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s_acc[wave][lane * VEC + j] = acc[j];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                acc[j] = 0.f;
#pragma unroll
                for (int w = 0; w < kListWaves; ++w) acc[j] += s_acc[w][lane * VEC + j];
            }
            store(r, acc);
        }
        __syncthreads();
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
struct EmbedSpace {
    size_t sorted[2], order[2], counts, partial, total;
};
// Positions per piece: short pieces while there are few, so that they fill the chip; longer ones keep the joining short.
inline int piece_of(long long n) {
    int piece = kBatch;
    while (piece < 64 && n / piece > 4096) piece *= 2;
    return piece;
}
inline int pieces_of(long long n) { return (int)((n + piece_of(n) - 1) / piece_of(n)); }
inline int sort_blocks(long long n) { return (int)((n + kSortItems - 1) / kSortItems); }
// At most 16 positions to a row on average: a workgroup's 16 rows then have few enough to be summed by its waves.
// (Both sides at 1312 tokens and 4232 rows: 8.9 against 16 us; where a workgroup's list is long the sorted sums, which are
// cut evenly, take over.)
inline bool listed(long long n, int vocab) { return n <= kListMax && n <= 16ll * vocab; }
inline EmbedSpace embed_space(long long n, int vocab, int dim) {
    EmbedSpace s = {};
    size_t at = 0;
    auto take = [&at](size_t bytes) {
        const size_t here = at;
        at += (bytes + 15) & ~(size_t)15;
        return here;
    };
    if (listed(n, vocab)) return s;
    const int copies = n > kRankMax ? 2 : 1;
    for (int i = 0; i < copies; ++i) {
        s.sorted[i] = take((size_t)n * 4);
        s.order[i] = take((size_t)n * 4);
    }
    if (n > kRankMax) s.counts = take((size_t)(sort_blocks(n) + 1) * kDigits * 4);
    s.partial = take((size_t)pieces_of(n) * 2 * dim * 4);
    s.total = at;
    return s;
}

// (positions are added in 32 bits, and a launch has less than 2^32 threads: 32 to a row of the vocabulary at most)
inline bool embed_shape_ok(long long n, int vocab, int dim) {
    return n >= 1 && n <= (1ll << 30) && vocab >= 1 && vocab <= (1 << 26) && dim >= 1 && dim <= (1 << 21);
}

// lanes that share a row: a power of two that covers the row's pieces, at most a wave
inline int row_shift(int dim, int vec) {
    int shift = 0;
    while ((vec << shift) < dim && shift < 6) ++shift;
    return shift;
}

template <typename DT>
rnntStatus_t embed_forward(const void *tokens, int tokens_64, long long n, const void *weight, long long weight_stride, int vocab,
                           int dim, float scale, void *out, hipStream_t st) {
    typedef typename DT::elem E;
    constexpr long long kForwardRows = 1ll << 25;  // rows of one launch, of at most 64 threads each
    const bool vec = dim % DT::EPC == 0 && weight_stride % DT::EPC == 0 && aligned16(weight) && aligned16(out);
    const int shift = row_shift(dim, vec ? DT::EPC : 1);
    for (long long at = 0; at < n; at += kForwardRows) {
        const long long rows = n - at < kForwardRows ? n - at : kForwardRows;
        const dim3 blocks((unsigned)(((rows << shift) + kBlock - 1) / kBlock));
        const void *tok = static_cast<const char *>(tokens) + at * (tokens_64 ? 8 : 4);
        E *o = static_cast<E *>(out) + at * dim;
        if (vec)
            hipLaunchKernelGGL((embed_forward_kernel<DT, DT::EPC>), blocks, dim3(kBlock), 0, st, tok, tokens_64, rows,
                               static_cast<const E *>(weight), weight_stride, vocab, dim, scale, o, shift);
        else
            hipLaunchKernelGGL((embed_forward_kernel<DT, 1>), blocks, dim3(kBlock), 0, st, tok, tokens_64, rows,
                               static_cast<const E *>(weight), weight_stride, vocab, dim, scale, o, shift);
    }
    return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED;
}

// gives which of the two buffers holds the result
template <bool MANY>
int radix_sort(const void *tokens, int tokens_64, int n, int vocab, long long padding, int *counts, int *const *sorted, int *const *order,
               hipStream_t st) {
    const int parts = sort_blocks(n);
    int at = 0;
    for (int bit = 0; bit == 0 || (bit < 31 && (vocab >> bit) != 0); bit += 8) {
        const void *src = bit == 0 ? tokens : sorted[at];
        const int to = bit == 0 ? 0 : 1 - at;
        hipLaunchKernelGGL((bit == 0 ? embed_digit_kernel<true> : embed_digit_kernel<false>), dim3(parts), dim3(kBlock), 0, st,
                           src, tokens_64, n, vocab, padding, bit, counts);
        if (MANY) hipLaunchKernelGGL(embed_prefix_kernel, dim3(kDigits), dim3(kBlock), 0, st, counts, parts);
        hipLaunchKernelGGL((bit == 0 ? embed_place_kernel<true, MANY> : embed_place_kernel<false, MANY>), dim3(parts), dim3(kBlock), 0, st,
                           src, tokens_64, n, vocab, padding, bit, static_cast<const int *>(counts),
                           static_cast<const int *>(order[at]), sorted[to], order[to]);
        at = to;
    }
    return at;
}

template <typename DT, int VEC>
rnntStatus_t embed_backward_with(const void *tokens, int tokens_64, int n, const typename DT::elem *grad, long long grad_stride,
                                 int vocab, int dim, float scale, long long padding, typename DT::elem *grad_weight, void *workspace,
                                 hipStream_t st) {
    if (listed(n, vocab)) {
        hipLaunchKernelGGL((embed_list_kernel<DT, VEC>),
                           dim3((unsigned)((vocab - 1) / kListRows + 1), (unsigned)((dim + kWave * VEC - 1) / (kWave * VEC))),
                           dim3(kListWaves * kWave), 0, st, tokens, tokens_64, n, vocab, padding, grad, grad_stride, dim, scale,
                           grad_weight);
        return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED;
    }
    const EmbedSpace sp = embed_space(n, vocab, dim);
    char *ws = static_cast<char *>(workspace);
    int *sorted[2], *order[2];
    for (int i = 0; i < 2; ++i) {
        sorted[i] = reinterpret_cast<int *>(ws + sp.sorted[i]);
        order[i] = reinterpret_cast<int *>(ws + sp.order[i]);
    }
    float *partial = reinterpret_cast<float *>(ws + sp.partial);
    int at = 0;
    if (n <= kRankMax) {
        const int blocks = (n + kWave - 1) / kWave;
        hipLaunchKernelGGL((embed_rank_kernel<DT, VEC>), dim3(blocks + (vocab - 1) / kRankRows + 1), dim3(kBlock), 0, st, tokens, tokens_64,
                           n, vocab, padding, sorted[0], order[0], grad_weight, dim, blocks);
    } else {
        int *counts = reinterpret_cast<int *>(ws + sp.counts);
        at = (n >= kSortMany ? radix_sort<true> : radix_sort<false>)(tokens, tokens_64, n, vocab, padding, counts, sorted, order, st);
    }
    const int shift = row_shift(dim, VEC), piece = piece_of(n), pieces = pieces_of(n);
    const int slices = (dim + (VEC << shift) - 1) / (VEC << shift);
    const long long blocks = ((((long long)pieces * slices) << shift) + kBlock - 1) / kBlock;
    const long long zero_blocks = n <= kRankMax ? 0 : ((vocab - 1) / 16 / (kBlock / kWave)) + 1;
    if ((blocks + zero_blocks) * kBlock >= 1ll << 32) return RNNT_STATUS_INVALID_VALUE;
    hipLaunchKernelGGL((embed_sum_kernel<DT, VEC>), dim3((unsigned)(blocks + zero_blocks)), dim3(kBlock), 0, st,
                       static_cast<const int *>(sorted[at]), static_cast<const int *>(order[at]), n, grad, grad_stride, vocab, dim, scale,
                       grad_weight, partial, piece, pieces, slices, shift, (unsigned)blocks);
    if (pieces > 1)
        hipLaunchKernelGGL((embed_join_kernel<DT, VEC>), dim3((unsigned)((pieces + kJoinWaves - 1) / kJoinWaves), (unsigned)((dim + kWave * VEC - 1) / (kWave * VEC))),
                           dim3(kJoinWaves * kWave), 0, st, static_cast<const int *>(sorted[at]), n, vocab, dim, scale, grad_weight,
                           static_cast<const float *>(partial), piece, pieces);
    return hipGetLastError() == hipSuccess ? RNNT_STATUS_SUCCESS : RNNT_STATUS_EXECUTION_FAILED;
}

template <typename DT>
rnntStatus_t embed_backward(const void *tokens, int tokens_64, long long n, const void *grad, long long grad_stride, int vocab,
                            int dim, float scale, long long padding, void *grad_weight, void *workspace, hipStream_t st) {
    typedef typename DT::elem E;
    const bool vec = dim % DT::EPC == 0 && grad_stride % DT::EPC == 0 && aligned16(grad) && aligned16(grad_weight);
    return (vec ? embed_backward_with<DT, DT::EPC> : embed_backward_with<DT, 1>)(tokens, tokens_64, (int)n, static_cast<const E *>(grad),
                                                                               grad_stride, vocab, dim, scale, padding,
                                                                               static_cast<E *>(grad_weight), workspace, st);
}

}  // namespace

extern "C" {

rnntStatus_t rnnt_token_embedding_forward(const void *tokens, int tokens_64, long long n, const void *weight,
                                          long long weight_stride, int vocab, int dim, float scale, rnntDtype_t dtype, void *out,
                                          void *stream) {
    if (tokens == nullptr || weight == nullptr || out == nullptr || !embed_shape_ok(n, vocab, dim) || weight_stride < dim)
        return RNNT_STATUS_INVALID_VALUE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RNNT_DTYPE_F32: return embed_forward<F32>(tokens, tokens_64, n, weight, weight_stride, vocab, dim, scale, out, st);
        case RNNT_DTYPE_BF16: return embed_forward<BF16>(tokens, tokens_64, n, weight, weight_stride, vocab, dim, scale, out, st);
        case RNNT_DTYPE_F16: return embed_forward<F16>(tokens, tokens_64, n, weight, weight_stride, vocab, dim, scale, out, st);
        default: return RNNT_STATUS_INVALID_VALUE;
    }
}

rnntStatus_t rnnt_token_embedding_workspace_size(long long n, int vocab, int dim, size_t *size_bytes) {
    if (size_bytes == nullptr || !embed_shape_ok(n, vocab, dim)) return RNNT_STATUS_INVALID_VALUE;
    *size_bytes = embed_space(n, vocab, dim).total;
    return RNNT_STATUS_SUCCESS;
}

rnntStatus_t rnnt_token_embedding_backward(const void *tokens, int tokens_64, long long n, const void *grad_out,
                                           long long grad_stride, int vocab, int dim, float scale, long long padding_idx,
                                           rnntDtype_t dtype, void *grad_weight, void *workspace, void *stream) {
    if (tokens == nullptr || grad_out == nullptr || grad_weight == nullptr || !embed_shape_ok(n, vocab, dim) || grad_stride < 0 ||
        (embed_space(n, vocab, dim).total > 0 && (workspace == nullptr || !aligned16(workspace))))
        return RNNT_STATUS_INVALID_VALUE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RNNT_DTYPE_F32:
            return embed_backward<F32>(tokens, tokens_64, n, grad_out, grad_stride, vocab, dim, scale, padding_idx, grad_weight,
                                       workspace, st);
        case RNNT_DTYPE_BF16:
            return embed_backward<BF16>(tokens, tokens_64, n, grad_out, grad_stride, vocab, dim, scale, padding_idx, grad_weight,
                                        workspace, st);
        case RNNT_DTYPE_F16:
            return embed_backward<F16>(tokens, tokens_64, n, grad_out, grad_stride, vocab, dim, scale, padding_idx, grad_weight,
                                       workspace, st);
        default: return RNNT_STATUS_INVALID_VALUE;
    }
}

}  // extern "C"
