// embedding.cu — rows of a 16-bit table by token id, scaled, and the gradient of the table.
//
// The lookup is a copy, bound by memory.  The gradient adds up the rows of equal tokens in the
// order of the tokens, so that the same inputs give the same bits.  Few tokens look each other
// up, in one launch.  More are sorted first (stable), blocks of the sorted order are summed in
// fp32, and runs that cross blocks are joined from the blocks' parts in order.  Most of a large
// table's rows are zeros, whose writing bounds the whole; the sort's launches, a few CTAs each,
// write zeros to a part of the table besides, as many as go out in the time they take anyhow.
//
// Sorting: radix passes of up to 9 bits over chunks of tokens; ranks within a chunk come from
// matching lanes and per-warp counts, never from atomics' order.  A launch counts the first
// digits by chunk; each pass counts the next ones as it puts the tokens into their new chunks.
//
// Measured: lookup of 8191 x 4104 fp16, scaled, 19 us (the output stays in L2 in part), of 16 rows
// 3.1.  Gradient of 16384 tokens, 131072 x 4096, 220 us (5.5 TB/s of a copy's 6.55): the zeros,
// and what the sums read and join; of 65533 tokens, 32000 x 2048, 107: 40 of them the sort.
#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace embedding {

constexpr int kMaxRows = INT_MAX - 1023;
constexpr int kMaxCols = 1 << 30;  // of the gradient, whose columns and a slab more are 32-bit numbers

// ------------------------------------------------------------------------- lookup
constexpr int kLookupThreads = 256;

struct LookupParams {
    const void *tokens, *table;
    void *y;
    int64_t ld;  // elements
    float scale;
    int V, vecs;  // 16-byte vectors of a row
    int64_t n;    // vectors of the output
};

// U vectors a thread, all in flight together: one where the output is small and latency counts,
// four otherwise.  N: of the vectors' numbers.
template <typename T, typename I, typename N, int U, bool SCALE>
__global__ void __launch_bounds__(kLookupThreads) embedding_kernel(const LookupParams p) {
    const N first = (N)blockIdx.x * (kLookupThreads * U) + threadIdx.x;
    uint4 v[U];
    bool live[U] = {};
#pragma unroll
    for (int u = 0; u < U; u++) {
        const N i = first + u * kLookupThreads;
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (i < (N)p.n) {
            const N t = i / (N)p.vecs, c = i - t * (N)p.vecs;
            const int64_t token = static_cast<const I *>(p.tokens)[t];
            live[u] = token >= 0 && token < p.V;
            if (live[u])
                v[u] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.table) + token * p.ld) + c);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const N i = first + u * kLookupThreads;
        if (SCALE && live[u]) {
            float f[8];
            unpack8<T>(v[u], f);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] *= p.scale;
            v[u] = pack8<T>(f);
        }
        if (i < (N)p.n) static_cast<uint4 *>(p.y)[i] = v[u];
    }
}

// ------------------------------------------------------------------------- sorting
constexpr int kSortThreads = 1024;
constexpr int kMaxBits = 9;              // of a pass
constexpr int kMaxDigits = 1 << kMaxBits;
constexpr int kMaxChunks = 256;
constexpr int kMaxPasses = 4;            // of 31 bits

struct SortParams {
    const void *tokens;          // first pass
    int wide;                    // they are 64-bit
    const int *keys_in, *at_in;  // later passes
    int *keys, *at;              // sorted tokens (V for those outside the table) and their positions
    int *counts;                 // [digits][chunks], by pass
    int *next;                   // the next pass's, or null; a count sets n_next of them to zero
    int64_t n_next;
    int next_shift, next_bits;
    int T, V, chunk, chunks;
    int shift, bits;
    uint4 *zero;                 // written by the CTAs past the sort's own
    int64_t zeros;
    int sort_ctas;
};

// CTAs past the sort's own, kZeroVectors of the table each.
constexpr int kZeroVectors = 16 * kSortThreads;
__device__ __forceinline__ bool write_zeros(const SortParams &p) {
    if ((int)blockIdx.x < p.sort_ctas) return false;
    const int64_t i0 = (int64_t)((int)blockIdx.x - p.sort_ctas) * kZeroVectors + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kZeroVectors / kSortThreads; u++)
        if (i0 + u * kSortThreads < p.zeros) p.zero[i0 + u * kSortThreads] = make_uint4(0u, 0u, 0u, 0u);
    return true;
}

__device__ __forceinline__ int key_of(const SortParams &p, int64_t t) {
    const int64_t token = p.wide ? static_cast<const int64_t *>(p.tokens)[t] : static_cast<const int *>(p.tokens)[t];
    return token >= 0 && token < p.V ? (int)token : p.V;
}

__device__ __forceinline__ int load_key(const SortParams &p, int64_t t) { return p.keys_in ? p.keys_in[t] : key_of(p, t); }

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortParams p) {
    __shared__ int count[kMaxDigits];
    if (write_zeros(p)) return;
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * p.chunk, t1 = min((int64_t)p.T, t0 + p.chunk);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += kSortThreads)
        atomicAdd(&count[(load_key(p, t) >> p.shift) & (digits - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) p.counts[(int64_t)d * p.chunks + blockIdx.x] = count[d];
    for (int64_t i = (int64_t)blockIdx.x * kSortThreads + threadIdx.x; i < p.n_next; i += (int64_t)p.sort_ctas * kSortThreads)
        p.next[i] = 0;
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const SortParams p) {
    constexpr int kWarps = kSortThreads / 32;
    __shared__ int base[kMaxDigits];
    __shared__ uint16_t in_warp[kWarps][kMaxDigits];
    __shared__ int totals[kWarps];
    if (write_zeros(p)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int digits = 1 << p.bits;
    const int64_t t0 = (int64_t)blockIdx.x * p.chunk, t1 = min((int64_t)p.T, t0 + p.chunk);
    int64_t t = t0 + threadIdx.x;  // its token comes while the counts are added up
    int key = t < t1 ? load_key(p, t) : 0, at = t < t1 ? (p.at_in ? p.at_in[t] : (int)t) : 0;
    // where this chunk's part of each digit starts: all counts of smaller digits, and the
    // digit's in earlier chunks
    const int threads_per_digit = kSortThreads / digits;  // at least two
    const int d = threadIdx.x / threads_per_digit, q = threadIdx.x % threads_per_digit;
    int all = 0, before = 0;
#pragma unroll 8
    for (int c = q; c < p.chunks; c += threads_per_digit) {
        const int n = p.counts[(int64_t)d * p.chunks + c];
        all += n;
        if (c < (int)blockIdx.x) before += n;
    }
    // threads_per_digit is a power of two; digits of fewer than 32 give it whole warps and more
    for (int o = min(threads_per_digit, 32) >> 1; o; o >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    __shared__ int digit_all[kMaxDigits], digit_before[kMaxDigits];
    for (int i = threadIdx.x; i < digits; i += kSortThreads) digit_all[i] = digit_before[i] = 0;
    __syncthreads();
    if (q % 32 == 0) {
        atomicAdd(&digit_all[d], all);
        atomicAdd(&digit_before[d], before);
    }
    __syncthreads();
    const int mine = (int)threadIdx.x < digits ? digit_all[threadIdx.x] : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
    }
    if (lane == 31) totals[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int w = totals[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        totals[lane] = w;
    }
    __syncthreads();
    if (warp) sum += totals[warp - 1];
    if ((int)threadIdx.x < digits) base[threadIdx.x] = sum - mine + digit_before[threadIdx.x];

    for (int64_t tile = t0; tile < t1; tile += kSortThreads) {
        for (int i = lane; i < digits; i += 32) in_warp[warp][i] = 0;
        __syncwarp();
        const bool live = t < t1;
        const int digit = live ? (key >> p.shift) & (digits - 1) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (live && rank == 0) in_warp[warp][digit] = (uint16_t)__popc(same);
        __syncthreads();
        if ((int)threadIdx.x < digits) {
            int run = base[threadIdx.x];
            int first[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; w++) first[w] = in_warp[w][threadIdx.x];
            int within = 0;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                in_warp[w][threadIdx.x] = (uint16_t)within;  // at most 1024 - 32
                within += first[w];
            }
            digit_before[threadIdx.x] = run;
            base[threadIdx.x] = run + within;
        }
        __syncthreads();
        if (live) {
            const int to = digit_before[digit] + in_warp[warp][digit] + rank;
            p.keys[to] = key;
            p.at[to] = at;
            if (p.next) atomicAdd(&p.next[(int64_t)((key >> p.next_shift) & ((1 << p.next_bits) - 1)) * p.chunks + to / p.chunk], 1);
        }
        t += kSortThreads;
        if (t < t1) {
            key = load_key(p, t);
            at = p.at_in ? p.at_in[t] : (int)t;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------- zeros
// Zeros for those of n rows of `vecs` vectors whose bit is not set, by THREADS threads.
template <typename T, int THREADS>
__device__ __forceinline__ void zero_rows(T *d, const uint32_t *named, int n, int vecs) {
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 *to = reinterpret_cast<uint4 *>(d);
    if (vecs >= THREADS) {
        for (int r = 0; r < n; r++, to += vecs)
            if (!((named[r >> 5] >> (r & 31)) & 1u))
                for (int c = threadIdx.x; c < vecs; c += THREADS) to[c] = zero;
    } else {  // threads over the rows too
        for (int i = threadIdx.x; i < n * vecs; i += THREADS) {
            const int r = i / vecs;
            if (!((named[r >> 5] >> (r & 31)) & 1u)) to[i] = zero;
        }
    }
}

// ------------------------------------------------------------------------- few tokens
// One launch: every CTA has all tokens in shared memory, and a warp looks for the places of its
// token.  The first of a short run sums its rows.  A long run's columns go to every eighth of its
// tokens in turn, whose CTA cuts the rows between its warps.  CTAs between them write zeros to
// the rows that no token names.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewTokens = 4096;
constexpr int kLongRun = 16;
constexpr int kFewCols = 32 * 8;     // columns of a warp at a time
constexpr int kFewAhead = 8;         // rows on their way
constexpr int kFewFill = 2048;       // most rows of a CTA that writes zeros

struct FewParams {
    const void *dy, *tokens;
    int64_t ld;
    void *d;
    float scale;
    int T, V, K, cols, slabs;  // columns of a CTA; CTAs for a token
    int sum_ctas, fill_ctas, fill_rows;
};

template <typename T, typename I>
__global__ void __launch_bounds__(kFewThreads) embedding_few_kernel(const FewParams p) {
    extern __shared__ int4 key4[];  // [padded tokens / 4], and then each warp's places
    int *key = reinterpret_cast<int *>(key4);
    const int padded = (p.T + 127) & ~127, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < padded; i += kFewThreads) {
        const int64_t token = i < p.T ? (int64_t)static_cast<const I *>(p.tokens)[i] : -1;
        key[i] = token >= 0 && token < p.V ? (int)token : -1;
    }
    __syncthreads();
    // CTA i of sum_ctas + fill_ctas: how many of the first i are sums, and whether this one is
    const int64_t all = (int64_t)p.sum_ctas + p.fill_ctas;
    const int sums = (int)((int64_t)blockIdx.x * p.sum_ctas / all);
    if ((int)(((int64_t)blockIdx.x + 1) * p.sum_ctas / all) == sums) {
        __shared__ uint32_t named[kFewFill / 32];  // a bit a row
        const int64_t v0 = (int64_t)((int)blockIdx.x - sums) * p.fill_rows;
        const int n = (int)min((int64_t)p.fill_rows, p.V - v0);
        if (threadIdx.x < kFewFill / 32) named[threadIdx.x] = 0u;
        __syncthreads();
        for (int i = threadIdx.x; i < p.T; i += kFewThreads) {
            const int64_t at = key[i] - v0;
            if (at >= 0 && at < n) atomicOr(&named[at >> 5], 1u << (at & 31));
        }
        __syncthreads();
        zero_rows<T, kFewThreads>(static_cast<T *>(p.d) + v0 * p.K, named, n, p.K / 8);
        return;
    }
    __shared__ int runs[kFewWarps], leads[kFewWarps];  // a run's length if this CTA sums of it, and its part
    __shared__ float part[kFewWarps][kFewCols];
    const int group = sums / p.slabs, slab = sums - group * p.slabs, t = group * kFewWarps + warp;
    uint16_t *places = reinterpret_cast<uint16_t *>(key + padded), *mine = places + warp * padded;
    const int token = t < p.T ? key[t] : -1;
    int n = 0, before = 0;  // places, and those before this one
    if (token >= 0)
        for (int j = 0; j < padded; j += 128) {
            const int4 k = key4[j / 4 + lane];
            const int hits = (k.x == token) | (k.y == token) << 1 | (k.z == token) << 2 | (k.w == token) << 3;
            const uint32_t any = __ballot_sync(0xffffffffu, hits != 0);
            if (!any) continue;
            const int here = j + 4 * lane;
            int upto = __popc(hits);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += u;
            }
            int at = n + upto - __popc(hits);
#pragma unroll
            for (int b = 0; b < 4; b++)
                if (hits >> b & 1) {
                    before += here + b < t;
                    mine[at++] = (uint16_t)(here + b);
                }
            n += __shfl_sync(0xffffffffu, upto, 31);
        }
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) {
        runs[warp] = n > kLongRun && before % 8 == 0 ? n : 0;
        leads[warp] = before / 8;
    }
    __syncthreads();
    const T *dy = static_cast<const T *>(p.dy);
    const int c0 = slab * p.cols, c1 = min(p.K, c0 + p.cols);
    // rows list[i0] to list[i1 - 1], eight columns from c on, in order
    auto add_rows = [&](const uint16_t *list, int i0, int i1, int c, float (&sum)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) sum[e] = 0.0f;
        for (int i = i0; i < i1; i += kFewAhead) {
            uint4 row[kFewAhead];
#pragma unroll
            for (int j = 0; j < kFewAhead; j++)
                if (i + j < i1) row[j] = __ldg(reinterpret_cast<const uint4 *>(dy + list[i + j] * p.ld + c));
#pragma unroll
            for (int j = 0; j < kFewAhead; j++)
                if (i + j < i1) {
                    float f[8];
                    unpack8<T>(row[j], f);
#pragma unroll
                    for (int e = 0; e < 8; e++) sum[e] += f[e];
                }
        }
    };
    if (n > 0 && n <= kLongRun && before == 0)
        for (int c = c0 + lane * 8; c < c1; c += kFewCols) {
            float sum[8];
            add_rows(mine, 0, n, c, sum);
#pragma unroll
            for (int e = 0; e < 8; e++) sum[e] *= p.scale;
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.d) + (int64_t)token * p.K + c) = pack8<T>(sum);
        }
    for (int w = 0; w < kFewWarps; w++) {
        const int run = runs[w];
        if (!run) continue;  // the same for all
        T *to = static_cast<T *>(p.d) + (int64_t)key[group * kFewWarps + w] * p.K;
        for (int base = c0 + leads[w] * kFewCols; base < c1; base += (run + 7) / 8 * kFewCols) {
            const int c = base + lane * 8;
            if (c < c1) {
                float sum[8];
                add_rows(places + w * padded, run * warp / kFewWarps, run * (warp + 1) / kFewWarps, c, sum);
#pragma unroll
                for (int e = 0; e < 8; e++) part[warp][lane * 8 + e] = sum[e];
            }
            __syncthreads();
            if (base + (int)threadIdx.x < c1) {
                float sum = part[0][threadIdx.x];
#pragma unroll
                for (int i = 1; i < kFewWarps; i++) sum += part[i][threadIdx.x];
                to[base + threadIdx.x] = Type16<T>::round(sum * p.scale);
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------- sums
constexpr int kSumThreads = 256;
constexpr int kSumCols = kSumThreads * 8;  // columns of a CTA, for narrow rows several blocks' in one
constexpr int kAhead = 4;                  // rows of a thread in flight, as many as are added up
constexpr int kMaxBlock = 128;             // sorted tokens of a block
constexpr int kJoinCols = 32 * 4;          // columns of a warp that joins
constexpr int kJoinBlocks = 8;             // blocks of a CTA that joins, a warp each: most have nothing to join
constexpr int kJoinThreads = 32 * kJoinBlocks;

struct SumParams {
    const void *dy;
    int64_t ld;
    void *d;
    float *parts;          // [blocks][2][K]: a block's end of a run that began before it, and
                           // its start of a run that goes on after it
    const int *keys, *at;  // sorted
    float scale;
    int T, V, K, block, blocks, slabs;
    int lanes, per_cta;    // threads of a block in a CTA, blocks of a CTA
    int sum_ctas, fill_ctas, join_ctas;
    int fill_rows, join_rows; // rows of a CTA that writes zeros, beside the sums and the joins
    int fill_from, fill_end;  // rows that the sums' launch fills: the sort has filled those before,
                              // the joins' fills those after
};

template <typename T>
__device__ __forceinline__ void put_row(const SumParams &p, int64_t v, int c, const float (&sum)[8]) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = sum[i] * p.scale;
    *reinterpret_cast<uint4 *>(static_cast<T *>(p.d) + v * p.K + c) = pack8<T>(f);
}

__device__ __forceinline__ void put_part(const SumParams &p, int block, int which, int c, const float (&sum)[8]) {
    float4 *to = reinterpret_cast<float4 *>(p.parts + ((int64_t)block * 2 + which) * p.K + c);
    to[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    to[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
}

// The first of the sorted tokens that is not below v, by a warp: 32 places at a time.
__device__ __forceinline__ int lower_bound(const int *keys, int n, int v, int lane) {
    int lo = 0;  // all before it are below
    for (int64_t stride = (int64_t)1 << 30; stride; stride >>= 5) {
        const int64_t i = lo + (lane + 1) * stride - 1;
        const bool below = i < n && keys[i] < v;
        lo += (int)(__popc(__ballot_sync(0xffffffffu, below)) * stride);
    }
    return lo;
}

// Zeros for those of `rows` rows (at most 256) from v0 on that no token names, by THREADS threads.
template <typename T, int THREADS>
__device__ __forceinline__ void fill(const SumParams &p, int64_t v0, int64_t end, int rows) {
    __shared__ uint32_t named[8];  // a bit a row
    const int n = (int)min((int64_t)rows, end - v0);
    if (threadIdx.x < 8) named[threadIdx.x] = 0u;
    __syncthreads();
    if (threadIdx.x < 32) {
        int i = lower_bound(p.keys, p.T, (int)v0, (int)threadIdx.x) + (int)threadIdx.x;
        for (;; i += 32) {
            const int key = i < p.T ? p.keys[i] : INT_MAX;
            const bool mine = key - v0 < n;
            if (mine) atomicOr(&named[(key - v0) >> 5], 1u << ((key - v0) & 31));
            if (!__all_sync(0xffffffffu, mine)) break;
        }
    }
    __syncthreads();
    zero_rows<T, THREADS>(static_cast<T *>(p.d) + v0 * p.K, named, n, p.K / 8);
}

// Sums, and CTAs that write zeros between them, so that both are on every SM: the sums wait for
// rows that lie anywhere, the zeros for nothing.
template <typename T>
__global__ void __launch_bounds__(kSumThreads, 4) embedding_sum_kernel(const SumParams p) {
    // CTA i of sum_ctas + fill_ctas: how many of the first i are sums, and whether this one is
    const int64_t all = (int64_t)p.sum_ctas + p.fill_ctas;
    const int sums = (int)((int64_t)blockIdx.x * p.sum_ctas / all);
    if ((int)(((int64_t)blockIdx.x + 1) * p.sum_ctas / all) == sums) {
        fill<T, kSumThreads>(p, p.fill_from + (int64_t)((int)blockIdx.x - sums) * p.fill_rows, p.fill_end, p.fill_rows);
        return;
    }
    // of the CTA's blocks: their keys and those on both sides, and where the rows are
    __shared__ int block_keys[kSumThreads / 32][kMaxBlock + 2], block_at[kSumThreads / 32][kMaxBlock];
    const int group = sums / p.slabs, slab = sums - group * p.slabs;
    const int in_cta = threadIdx.x / p.lanes, x = threadIdx.x - in_cta * p.lanes;
    const int block = group * p.per_cta + in_cta;
    const int c = slab * kSumCols + x * 8;
    const int64_t i0 = (int64_t)block * p.block;
    const int n = in_cta < p.per_cta ? (int)max((int64_t)0, min((int64_t)p.block, p.T - i0)) : 0;
    int *keys = block_keys[in_cta], *at = block_at[in_cta];
    for (int j = x; n > 0 && j < n + 2; j += p.lanes) {
        const int64_t i = i0 - 1 + j;
        keys[j] = i >= 0 && i < p.T ? p.keys[i] : -1;
        if (j < n) at[j] = p.at[i0 + j];
    }
    __syncthreads();
    if (n <= 0 || c >= p.K) return;
    const T *dy = static_cast<const T *>(p.dy) + c;
    int run = keys[1];
    if (run >= p.V) return;          // tokens outside the table sort last
    bool began = run != keys[0];     // the current run starts in this block
    float sum[8] = {};
    auto fetch = [&](int i, uint4 (&row)[kAhead]) {
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (i + j < n && keys[1 + i + j] < p.V)
                row[j] = __ldg(reinterpret_cast<const uint4 *>(dy + (int64_t)at[i + j] * p.ld));
    };
    uint4 row[kAhead], next[kAhead];
    fetch(0, row);
    for (int i = 0; i < n; i += kAhead) {
        fetch(i + kAhead, next);
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (i + j >= n) break;
            const int key = keys[1 + i + j];
            if (key != run) {  // the run ends inside the block
                if (began) put_row<T>(p, run, c, sum);
                else put_part(p, block, 0, c, sum);
                if (key >= p.V) return;
                run = key;
                began = true;
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] = 0.0f;
            }
            float f[8];
            unpack8<T>(row[j], f);
#pragma unroll
            for (int e = 0; e < 8; e++) sum[e] += f[e];
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) row[j] = next[j];
    }
    if (!began) put_part(p, block, 0, c, sum);        // ends here, or goes on: the join knows
    else if (run == keys[1 + n]) put_part(p, block, 1, c, sum);
    else put_row<T>(p, run, c, sum);
}

// volatile: the loads of a batch are issued before the first is waited for
__device__ __forceinline__ float4 load_part(const float *from) {
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(from));
    return v;
}

// Runs of several blocks: the start in the block where the run begins, then the following
// blocks' ends, in order.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads, 4) embedding_join_kernel(const SumParams p) {
    if ((int)blockIdx.x >= p.join_ctas) {
        fill<T, kJoinThreads>(p, p.fill_end + (int64_t)((int)blockIdx.x - p.join_ctas) * p.join_rows, p.V, p.join_rows);
        return;
    }
    const int slabs = (p.K + kJoinCols - 1) / kJoinCols, lane = threadIdx.x & 31;
    const int eight = blockIdx.x / slabs, slab = blockIdx.x - eight * slabs;
    const int64_t b = (int64_t)eight * kJoinBlocks + (threadIdx.x >> 5), i0 = b * p.block, i1 = i0 + p.block;
    if (i1 >= p.T) return;
    const int block = (int)b;
    const int run = p.keys[i1 - 1], after = p.keys[i1], first = p.keys[i0], before = i0 ? p.keys[i0 - 1] : -1;
    if (run >= p.V || after != run) return;       // does not go on
    if (first == run && before == run) return;    // began in an earlier block
    // The last block whose first token is the run's: the steps of 32 that still are.
    int last = block + 1;
    for (int64_t stride = (int64_t)1 << 25; stride; stride >>= 5) {
        const int64_t q = last + (lane + 1) * stride;
        const bool same = q < p.blocks && p.keys[q * p.block] == run;
        last += (int)(__popc(__ballot_sync(0xffffffffu, same)) * stride);
    }
    const int c = slab * kJoinCols + lane * 4;
    if (c >= p.K) return;
    const float *start = p.parts + ((int64_t)block * 2 + 1) * p.K + c;
    float4 sum = *reinterpret_cast<const float4 *>(start);
    constexpr int kAtOnce = 8;  // parts on their way
    for (int q0 = block + 1; q0 <= last; q0 += kAtOnce) {
        float4 a[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; j++)
            a[j] = load_part(p.parts + (int64_t)min(q0 + j, last) * 2 * p.K + c);
#pragma unroll
        for (int j = 0; j < kAtOnce; j++) {
            const bool in = q0 + j <= last;
            sum.x += in ? a[j].x : 0.0f;
            sum.y += in ? a[j].y : 0.0f;
            sum.z += in ? a[j].z : 0.0f;
            sum.w += in ? a[j].w : 0.0f;
        }
    }
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.d) + (int64_t)run * p.K + c) =
        make_uint2(Type16<T>::pack(sum.x * p.scale, sum.y * p.scale), Type16<T>::pack(sum.z * p.scale, sum.w * p.scale));
}

// ------------------------------------------------------------------------- host side
// Sorted tokens of a block of sums: the blocks' ends of crossing runs are written and read in
// fp32, so longer blocks for more tokens of long rows.  Short ones have few warps, which wait for
// one row after another.  us, by blocks of 32, 64 and 128: 65000 tokens of 2048 121, 112, 104, of
// 1024 74, 68, 75, 60000 of 512 45, 46, 56, 45000 of 72 33, 37, 49.
static int block_tokens(int T, int K) {
    if (T <= 16384 || K <= 512) return 32;
    return T <= 32768 || K <= 1024 ? 64 : kMaxBlock;
}

// Radix chunks: one tile a CTA while there are no more than kMaxChunks.
static int chunk_tokens(int T) {
    const int64_t per = ((int64_t)T + kMaxChunks - 1) / kMaxChunks;
    return (int)std::max<int64_t>(kSortThreads, (per + kSortThreads - 1) / kSortThreads * kSortThreads);
}

struct Layout {
    size_t keys[2], at[2], counts, parts, bytes;
    int chunk, chunks, block, blocks;
};
static Layout layout(int T, int K) {
    Layout l;
    size_t n = 0;
    auto take = [&](size_t bytes) {
        const size_t at = n;
        n += (bytes + 255) & ~(size_t)255;
        return at;
    };
    l.chunk = chunk_tokens(T);
    l.chunks = (int)(((int64_t)T + l.chunk - 1) / l.chunk);
    l.block = block_tokens(T, K);
    l.blocks = (int)(((int64_t)T + l.block - 1) / l.block);
    for (int i = 0; i < 2; i++) {
        l.keys[i] = take((size_t)T * 4);
        l.at[i] = take((size_t)T * 4);
    }
    l.counts = take((size_t)kMaxPasses * kMaxDigits * l.chunks * 4);
    l.parts = take((size_t)l.blocks * 2 * K * 4);
    l.bytes = n;
    return l;
}

// Whether tokens are few enough to be looked up by each other.  us, in one launch and sorted: 1000
// tokens of 5000 x 512 10 and 21, 2000 of x 4096 18 and 30, 4000 of x 512 16 and 27, of x 4096 37
// and 30; all the same, the longest run there can be, 2000 32 and 20.
static bool unsorted(int T, int K) { return T <= kFewTokens / 2 || (T <= kFewTokens && K <= 1024); }

template <typename T, typename I>
static int few(const FewParams &p, const DeviceInfo &di, cudaStream_t s) {
    const int padded = (p.T + 127) & ~127;
    static std::atomic<bool> configured[64] = {};
    if (!configured[di.device]) {
        if (cudaFuncSetAttribute(embedding_few_kernel<T, I>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kFewTokens * (4 + 2 * kFewWarps)) != cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device] = true;
    }
    embedding_few_kernel<T, I><<<(unsigned)(p.sum_ctas + p.fill_ctas), kFewThreads, padded * (4 + 2 * kFewWarps), s>>>(p);
    count_launch();
    return cuda_status(cudaGetLastError());
}

template <typename T>
static int sum(const SumParams &p, cudaStream_t s) {
    embedding_sum_kernel<T><<<(unsigned)(p.sum_ctas + p.fill_ctas), kSumThreads, 0, s>>>(p);
    count_launch();
    if (p.blocks > 1) {
        const int ctas = (p.V - p.fill_end + p.join_rows - 1) / p.join_rows;
        embedding_join_kernel<T><<<(unsigned)(p.join_ctas + ctas), kJoinThreads, 0, s>>>(p);
        count_launch();
    }
    return cuda_status(cudaGetLastError());
}

// Bytes of zeros that go out while a launch of the sort or the joins runs, about: a count takes
// 3.5 us, a scatter 7, the joins 8.
constexpr int64_t kCountZeros = 32 << 20, kScatterZeros = 56 << 20, kJoinZeros = 40 << 20;

// Sorts the tokens; l.keys[0] and l.at[0] hold the result, or [1] if it returns 1 in *which.
// The first *zero_rows rows of the table are zeros afterwards.
static int sort(const void *tokens, int wide, int T, int V, int K, void *table, uint8_t *ws, const Layout &l, int *which,
                int *zero_rows, cudaStream_t s) {
    SortParams p = {};
    p.tokens = tokens;
    p.wide = wide;
    p.T = T;
    p.V = V;
    p.chunk = l.chunk;
    p.chunks = l.chunks;
    p.counts = reinterpret_cast<int *>(ws + l.counts);
    *which = 0;
    *zero_rows = 0;
    const int64_t row = (int64_t)K * 2;
    // the launch's share of zeros; the CTAs of all
    auto zeros = [&](int64_t bytes, int sort_ctas) {
        const int rows = (int)std::min<int64_t>(V - *zero_rows, bytes / row);
        p.zero = static_cast<uint4 *>(table) + (int64_t)*zero_rows * K / 8;
        p.zeros = (int64_t)rows * K / 8;
        p.sort_ctas = sort_ctas;
        *zero_rows += rows;
        return (unsigned)(sort_ctas + (p.zeros + kZeroVectors - 1) / kZeroVectors);
    };
    int bits = 1;  // of the largest key, V
    while (bits < 31 && (V >> bits) != 0) bits++;
    const int passes = (bits + kMaxBits - 1) / kMaxBits;
    const int64_t counts = (int64_t)kMaxDigits * l.chunks;  // of a pass
    auto bits_of = [&](int pass) { return bits / passes + (pass < bits % passes ? 1 : 0); };
    for (int i = 0; i < passes; i++) {
        p.bits = bits_of(i);
        p.next_shift = p.shift + p.bits;
        p.next_bits = i + 1 < passes ? bits_of(i + 1) : 0;
        p.next = i + 1 < passes ? p.counts + counts : nullptr;
        if (i == 0) {
            p.n_next = counts * (passes - 1);
            const unsigned ctas = zeros(kCountZeros, l.chunks);
            sort_count_kernel<<<ctas, kSortThreads, 0, s>>>(p);
            count_launch();
        }
        p.keys_in = i ? reinterpret_cast<int *>(ws + l.keys[*which]) : nullptr;
        p.at_in = i ? reinterpret_cast<int *>(ws + l.at[*which]) : nullptr;
        if (i) *which ^= 1;
        p.keys = reinterpret_cast<int *>(ws + l.keys[*which]);
        p.at = reinterpret_cast<int *>(ws + l.at[*which]);
        const unsigned ctas = zeros(kScatterZeros, l.chunks);
        sort_scatter_kernel<<<ctas, kSortThreads, 0, s>>>(p);
        count_launch();
        p.shift += p.bits;
        p.counts += counts;
    }
    return cuda_status(cudaGetLastError());
}

static bool misaligned(const void *p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// What both directions check.
static int check_sizes(const void *tokens, int token_bytes, int64_t ld, int T, int V, int K, int dtype) {
    if (dtype != NVFP4_BF16 && dtype != NVFP4_F16) return NVFP4_ERR_INVALID;
    if (token_bytes != 4 && token_bytes != 8) return NVFP4_ERR_INVALID;
    if (T < 0 || V < 1 || K < 8 || K % 8 || T > kMaxRows || V > kMaxRows || K > kMaxRows) return NVFP4_ERR_SHAPE;
    if (ld < K || ld % 8) return NVFP4_ERR_SHAPE;
    if (T && !tokens) return NVFP4_ERR_INVALID;
    return misaligned(tokens, token_bytes) ? NVFP4_ERR_ALIGN : NVFP4_OK;
}

template <typename T, typename I, typename N, int U>
static void lookup_u(const LookupParams &p, cudaStream_t s) {
    const unsigned grid = (unsigned)((p.n + U * kLookupThreads - 1) / (U * kLookupThreads));
    if (p.scale == 1.0f) embedding_kernel<T, I, N, U, false><<<grid, kLookupThreads, 0, s>>>(p);
    else embedding_kernel<T, I, N, U, true><<<grid, kLookupThreads, 0, s>>>(p);
}
// One vector a thread as long as that makes no more CTAs than run at once, eight an SM.
template <typename T, typename I>
static void lookup_i(const LookupParams &p, int sm_count, cudaStream_t s) {
    if (p.n <= (int64_t)sm_count * 8 * kLookupThreads) lookup_u<T, I, uint32_t, 1>(p, s);
    else if (p.n < ((int64_t)1 << 31)) lookup_u<T, I, uint32_t, 4>(p, s);
    else lookup_u<T, I, uint64_t, 4>(p, s);
}
template <typename T>
static void lookup(const LookupParams &p, int token_bytes, int sm_count, cudaStream_t s) {
    if (token_bytes == 8) lookup_i<T, int64_t>(p, sm_count, s);
    else lookup_i<T, int>(p, sm_count, s);
}

}  // namespace embedding
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

int nvfp4_embedding(const void *tokens, int token_bytes, const void *table, int64_t ld, float scale, void *Y, int T,
                    int V, int K, int dtype, void *stream) {
    int st = embedding::check_sizes(tokens, token_bytes, ld, T, V, K, dtype);
    if (st) return st;
    if (!table || (T && !Y)) return NVFP4_ERR_INVALID;
    if (!aligned16(table) || !aligned16(Y)) return NVFP4_ERR_ALIGN;
    embedding::LookupParams p = {};
    p.tokens = tokens;
    p.table = table;
    p.y = Y;
    p.ld = ld;
    p.scale = scale;
    p.V = V;
    p.vecs = K / 8;
    p.n = (int64_t)T * p.vecs;
    if (p.n / (4 * embedding::kLookupThreads) >= INT_MAX) return NVFP4_ERR_SHAPE;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) embedding::lookup<__nv_bfloat16>(p, token_bytes, di.sm_count, s);
    else embedding::lookup<__half>(p, token_bytes, di.sm_count, s);
    count_launch();
    return cuda_status(cudaGetLastError());
}

size_t nvfp4_embedding_backward_workspace_size(int T, int V, int K) {
    if (T < 1 || V < 1 || K < 8 || T > embedding::kMaxRows || V > embedding::kMaxRows || K > embedding::kMaxCols)
        return 0;
    return embedding::unsorted(T, K) ? 0 : embedding::layout(T, K).bytes;
}

int nvfp4_embedding_backward(const void *dY, int64_t ldy, const void *tokens, int token_bytes, float scale,
                             void *dTable, int T, int V, int K, int dtype, void *workspace, size_t workspace_bytes,
                             void *stream) {
    int st = embedding::check_sizes(tokens, token_bytes, ldy, T, V, K, dtype);
    if (st) return st;
    if (K > embedding::kMaxCols) return NVFP4_ERR_SHAPE;
    if (!dTable || (T && !dY)) return NVFP4_ERR_INVALID;
    if (!aligned16(dY) || !aligned16(dTable) || !aligned16(workspace)) return NVFP4_ERR_ALIGN;
    const size_t need = nvfp4_embedding_backward_workspace_size(T, V, K);
    if (need && (!workspace || workspace_bytes < need)) return NVFP4_ERR_WORKSPACE;
    const int slabs = (K + embedding::kSumCols - 1) / embedding::kSumCols;
    const embedding::Layout l = embedding::layout(T, K);
    if ((int64_t)l.blocks * std::max(slabs, (K + embedding::kJoinCols - 1) / embedding::kJoinCols) > INT_MAX)
        return NVFP4_ERR_SHAPE;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (T == 0)  // no token: the gradient is zero
        return cuda_status(cudaMemsetAsync(dTable, 0, (size_t)V * K * 2, s));
    // rows of zeros: about 256 KB a CTA, and 64 KB beside the joins
    const int fill_rows = (int)std::max<int64_t>(1, (256 << 10) / ((int64_t)K * 2));
    if (embedding::unsorted(T, K)) {
        embedding::FewParams p = {};
        p.dy = dY;
        p.tokens = tokens;
        p.ld = ldy;
        p.d = dTable;
        p.scale = scale;
        p.T = T;
        p.V = V;
        p.K = K;
        // the narrowest CTAs, for latency, that still run all at once
        const int64_t groups = (T + embedding::kFewWarps - 1) / embedding::kFewWarps;
        p.cols = embedding::kFewCols;
        while (groups * ((K + p.cols - 1) / p.cols) > 4 * di.sm_count && p.cols < K) p.cols *= 2;
        p.slabs = (K + p.cols - 1) / p.cols;
        p.fill_rows = std::min(embedding::kFewFill, fill_rows);
        p.fill_ctas = (int)(((int64_t)V + p.fill_rows - 1) / p.fill_rows);
        if (groups * p.slabs + p.fill_ctas > INT_MAX) return NVFP4_ERR_SHAPE;
        p.sum_ctas = (int)(groups * p.slabs);
        if (dtype == NVFP4_BF16)
            return token_bytes == 8 ? embedding::few<__nv_bfloat16, int64_t>(p, di, s)
                                    : embedding::few<__nv_bfloat16, int>(p, di, s);
        return token_bytes == 8 ? embedding::few<__half, int64_t>(p, di, s) : embedding::few<__half, int>(p, di, s);
    }
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    int which = 0, zero_rows = 0;
    if ((st = embedding::sort(tokens, token_bytes == 8, T, V, K, dTable, ws, l, &which, &zero_rows, s))) return st;
    embedding::SumParams p = {};
    p.dy = dY;
    p.ld = ldy;
    p.d = dTable;
    p.parts = reinterpret_cast<float *>(ws + l.parts);
    p.keys = reinterpret_cast<const int *>(ws + l.keys[which]);
    p.at = reinterpret_cast<const int *>(ws + l.at[which]);
    p.scale = scale;
    p.T = T;
    p.V = V;
    p.K = K;
    p.block = l.block;
    p.blocks = l.blocks;
    p.slabs = slabs;
    p.lanes = std::min(embedding::kSumThreads, (K / 8 + 31) / 32 * 32);
    p.per_cta = embedding::kSumThreads / p.lanes;
    p.sum_ctas = (l.blocks + p.per_cta - 1) / p.per_cta * slabs;
    p.join_ctas = (l.blocks + embedding::kJoinBlocks - 1) / embedding::kJoinBlocks *
                  ((K + embedding::kJoinCols - 1) / embedding::kJoinCols);
    p.fill_rows = std::min(256, fill_rows);
    p.join_rows = (p.fill_rows + 3) / 4;
    p.fill_from = zero_rows;
    p.fill_end = V;
    if (l.blocks > 1)  // the joins follow
        p.fill_end -= (int)std::min<int64_t>(V - zero_rows, embedding::kJoinZeros / ((int64_t)K * 2));
    p.fill_ctas = (p.fill_end - p.fill_from + p.fill_rows - 1) / p.fill_rows;
    if ((int64_t)p.sum_ctas + p.fill_ctas > INT_MAX || (int64_t)p.join_ctas + V / p.join_rows >= INT_MAX)
        return NVFP4_ERR_SHAPE;
    return dtype == NVFP4_BF16 ? embedding::sum<__nv_bfloat16>(p, s) : embedding::sum<__half>(p, s);
}

}  // extern "C"
