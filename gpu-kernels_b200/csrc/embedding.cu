// embedding.cu — rows of a 16-bit table by token id, scaled, and the gradient of the table.
//
// The lookup is a copy: 16 bytes a thread, bound by memory.  The gradient adds up the rows of
// equal tokens in the order of the tokens, so that the same inputs give the same bits: the
// tokens are sorted first (stable), blocks of the sorted order are summed in fp32, and runs
// that cross blocks are joined from the blocks' parts in order.  Each row of the gradient is
// written once; most of a large table's rows are zeros, whose writing bounds the whole.
//
// Sorting: up to kSmallTokens tokens in one CTA (64-bit keys: token, then position).  More
// take radix passes of up to 9 bits, each a count and a scatter over chunks of tokens; ranks
// within a chunk come from matching lanes and per-warp counts, never from atomics' order.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace embedding {

constexpr int kMaxRows = INT_MAX - 1023;

// ------------------------------------------------------------------------- lookup
constexpr int kLookupThreads = 256;

struct LookupParams {
    const void *tokens, *table;
    void *y;
    int64_t ld;  // elements
    float scale;
    int T, V, vecs;       // 16-byte vectors of a row
    int lanes, per_cta;   // threads of a row, rows of a CTA
    int slabs;            // CTAs of a row
};

template <typename T, typename I, bool SCALE>
__global__ void __launch_bounds__(kLookupThreads) embedding_kernel(const LookupParams p) {
    const int block = blockIdx.x / p.slabs, slab = blockIdx.x - block * p.slabs;
    const int in_cta = threadIdx.x / p.lanes;
    const int64_t t = (int64_t)block * p.per_cta + in_cta;
    const int c = slab * p.lanes + threadIdx.x - in_cta * p.lanes;
    if (in_cta >= p.per_cta || t >= p.T || c >= p.vecs) return;
    const int64_t token = static_cast<const I *>(p.tokens)[t];
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (token >= 0 && token < p.V) {
        v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.table) + token * p.ld) + c);
        if constexpr (SCALE) {
            float f[8];
            unpack8<T>(v, f);
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] *= p.scale;
            v = pack8<T>(f);
        }
    }
    static_cast<uint4 *>(p.y)[t * p.vecs + c] = v;
}

// ------------------------------------------------------------------------- sorting
constexpr int kSortThreads = 1024;
constexpr int kSmallTokens = 4096;
constexpr int kMaxBits = 9;              // of a pass
constexpr int kMaxDigits = 1 << kMaxBits;
constexpr int kMaxChunks = 256;

struct SortParams {
    const void *tokens;          // first pass
    int wide;                    // they are 64-bit
    const int *keys_in, *at_in;  // later passes
    int *keys, *at;              // sorted tokens (V for those outside the table) and their positions
    int *counts;                 // [digits][chunks]
    int T, V, chunk, chunks;
    int shift, bits;
};

__device__ __forceinline__ int key_of(const SortParams &p, int64_t t) {
    const int64_t token = p.wide ? static_cast<const int64_t *>(p.tokens)[t] : static_cast<const int *>(p.tokens)[t];
    return token >= 0 && token < p.V ? (int)token : p.V;
}

// Bitonic sort of n (a power of two) keys that are all different, so it is stable.
__global__ void __launch_bounds__(kSortThreads) sort_small_kernel(const SortParams p, int n) {
    extern __shared__ uint64_t key[];
    for (int i = threadIdx.x; i < n; i += kSortThreads)
        key[i] = i < p.T ? (uint64_t)(uint32_t)key_of(p, i) << 32 | (uint32_t)i : ~0ull;
    __syncthreads();
    for (int size = 2; size <= n; size <<= 1)
        for (int o = size >> 1; o; o >>= 1) {
            for (int i = threadIdx.x; i < n / 2; i += kSortThreads) {
                const int a = 2 * i - (i & (o - 1)), b = a + o;
                const uint64_t x = key[a], y = key[b];
                if ((x > y) == ((a & size) == 0)) {
                    key[a] = y;
                    key[b] = x;
                }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < p.T; i += kSortThreads) {
        p.keys[i] = (int)(key[i] >> 32);
        p.at[i] = (int)(uint32_t)key[i];
    }
}

__device__ __forceinline__ int load_key(const SortParams &p, int64_t t) { return p.keys_in ? p.keys_in[t] : key_of(p, t); }

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortParams p) {
    __shared__ int count[kMaxDigits];
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * p.chunk, t1 = min((int64_t)p.T, t0 + p.chunk);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += kSortThreads)
        atomicAdd(&count[(load_key(p, t) >> p.shift) & (digits - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) p.counts[(int64_t)d * p.chunks + blockIdx.x] = count[d];
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const SortParams p) {
    constexpr int kWarps = kSortThreads / 32;
    __shared__ int base[kMaxDigits];
    __shared__ uint16_t in_warp[kWarps][kMaxDigits];
    __shared__ int totals[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int digits = 1 << p.bits;
    // where this chunk's part of each digit starts: all counts of smaller digits, and the
    // digit's in earlier chunks
    const int threads_per_digit = kSortThreads / digits;  // at least two
    const int d = threadIdx.x / threads_per_digit, q = threadIdx.x % threads_per_digit;
    int all = 0, before = 0;
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
    for (int w = 0; w < warp; w++) sum += totals[w];
    if ((int)threadIdx.x < digits) base[threadIdx.x] = sum - mine + digit_before[threadIdx.x];

    const int64_t t0 = (int64_t)blockIdx.x * p.chunk, t1 = min((int64_t)p.T, t0 + p.chunk);
    for (int64_t tile = t0; tile < t1; tile += kSortThreads) {
        for (int i = lane; i < digits; i += 32) in_warp[warp][i] = 0;
        __syncwarp();
        const int64_t t = tile + threadIdx.x;
        const bool live = t < t1;
        const int key = live ? load_key(p, t) : 0;
        const int at = live ? (p.at_in ? p.at_in[t] : (int)t) : 0;
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
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------- sums
constexpr int kSumThreads = 256;
constexpr int kSumCols = kSumThreads * 8;  // columns of a CTA
constexpr int kAhead = 8;                  // rows of a thread in flight

struct SumParams {
    const void *dy;
    int64_t ld;
    void *d;
    float *parts;          // [blocks][2][K]: a block's end of a run that began before it, and
                           // its start of a run that goes on after it
    const int *keys, *at;  // sorted
    float scale;
    int T, V, K, block, blocks, slabs;
    int sum_ctas;
    int fill_rows;         // rows of a CTA that writes zeros
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

// The first of the sorted tokens that is not below v.
__device__ __forceinline__ int lower_bound(const int *keys, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(kSumThreads) embedding_sum_kernel(const SumParams p) {
    if ((int)blockIdx.x >= p.sum_ctas) {
        // rows that no token names
        __shared__ uint32_t named[8];  // a bit a row
        const int64_t v0 = (int64_t)(blockIdx.x - p.sum_ctas) * p.fill_rows;
        const int n = (int)min((int64_t)p.fill_rows, p.V - v0);
        if (threadIdx.x < 8) named[threadIdx.x] = 0u;
        __syncthreads();
        if (threadIdx.x < 32) {
            int i = 0;
            if (threadIdx.x == 0) i = lower_bound(p.keys, p.T, (int)v0);
            i = __shfl_sync(0xffffffffu, i, 0) + (int)threadIdx.x;
            for (;; i += 32) {
                const int key = i < p.T ? p.keys[i] : INT_MAX;
                const bool mine = key - v0 < n;
                if (mine) atomicOr(&named[(key - v0) >> 5], 1u << ((key - v0) & 31));
                if (!__all_sync(0xffffffffu, mine)) break;
            }
        }
        __syncthreads();
        const int vecs = p.K / 8;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        for (int r = 0; r < n; r++) {
            if ((named[r >> 5] >> (r & 31)) & 1u) continue;
            uint4 *to = reinterpret_cast<uint4 *>(static_cast<T *>(p.d) + (v0 + r) * p.K);
            for (int c = threadIdx.x; c < vecs; c += kSumThreads) to[c] = zero;
        }
        return;
    }
    const int block = blockIdx.x / p.slabs, slab = blockIdx.x - block * p.slabs;
    const int c = slab * kSumCols + (int)threadIdx.x * 8;
    if (c >= p.K) return;
    const int64_t i0 = (int64_t)block * p.block, i1 = min((int64_t)p.T, i0 + p.block);
    const T *dy = static_cast<const T *>(p.dy);
    const int before = i0 ? p.keys[i0 - 1] : -1;
    const int after = i1 < p.T ? p.keys[i1] : -1;
    float sum[8] = {};
    int run = p.keys[i0];
    bool began = run != before;  // the current run starts in this block
    if (run >= p.V) return;      // tokens outside the table sort last
    for (int64_t i = i0; i < i1; i += kAhead) {
        int key[kAhead];
        uint4 row[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            key[j] = i + j < i1 ? p.keys[i + j] : INT_MAX;
            if (key[j] < p.V) row[j] = __ldg(reinterpret_cast<const uint4 *>(dy + (int64_t)p.at[i + j] * p.ld + c));
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (i + j >= i1) break;
            if (key[j] != run) {  // the run ends inside the block
                if (began) put_row<T>(p, run, c, sum);
                else put_part(p, block, 0, c, sum);
                if (key[j] >= p.V) return;
                run = key[j];
                began = true;
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] = 0.0f;
            }
            float f[8];
            unpack8<T>(row[j], f);
#pragma unroll
            for (int e = 0; e < 8; e++) sum[e] += f[e];
        }
    }
    if (!began) put_part(p, block, 0, c, sum);        // ends here, or goes on: the join knows
    else if (run == after) put_part(p, block, 1, c, sum);
    else put_row<T>(p, run, c, sum);
}

// Runs of several blocks: the start in the block where the run begins, then the following
// blocks' ends, in order.
template <typename T>
__global__ void __launch_bounds__(kSumThreads) embedding_join_kernel(const SumParams p) {
    const int block = blockIdx.x / p.slabs, slab = blockIdx.x - block * p.slabs;
    const int c = slab * kSumCols + (int)threadIdx.x * 8;
    const int64_t i0 = (int64_t)block * p.block, i1 = i0 + p.block;
    if (i1 >= p.T) return;
    const int run = p.keys[i1 - 1];
    if (run >= p.V || p.keys[i1] != run) return;        // does not go on
    if (p.keys[i0] == run && i0 && p.keys[i0 - 1] == run) return;  // began in an earlier block
    if (c >= p.K) return;
    const int last = (lower_bound(p.keys, p.T, run + 1) - 1) / p.block;
    const float *from = p.parts + ((int64_t)block * 2 + 1) * p.K + c;
    float sum[8];
    {
        const float4 a = reinterpret_cast<const float4 *>(from)[0], b = reinterpret_cast<const float4 *>(from)[1];
        sum[0] = a.x, sum[1] = a.y, sum[2] = a.z, sum[3] = a.w;
        sum[4] = b.x, sum[5] = b.y, sum[6] = b.z, sum[7] = b.w;
    }
#pragma unroll 4
    for (int q = block + 1; q <= last; q++) {
        const float4 *f = reinterpret_cast<const float4 *>(p.parts + (int64_t)q * 2 * p.K + c);
        const float4 a = f[0], b = f[1];
        sum[0] += a.x, sum[1] += a.y, sum[2] += a.z, sum[3] += a.w;
        sum[4] += b.x, sum[5] += b.y, sum[6] += b.z, sum[7] += b.w;
    }
    put_row<T>(p, run, c, sum);
}

// ------------------------------------------------------------------------- host side
// Sorted tokens of a block of sums: the blocks' ends of crossing runs are written and read in
// fp32, so longer blocks for more tokens.
static int block_tokens(int T) { return T <= 32768 ? 32 : T <= 131072 ? 64 : 128; }

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
    l.block = block_tokens(T);
    l.blocks = (int)(((int64_t)T + l.block - 1) / l.block);
    for (int i = 0; i < 2; i++) {
        l.keys[i] = take((size_t)T * 4);
        l.at[i] = take((size_t)T * 4);
    }
    l.counts = take((size_t)kMaxDigits * l.chunks * 4);
    l.parts = take((size_t)l.blocks * 2 * K * 4);
    l.bytes = n;
    return l;
}

template <typename T>
static int sum(const SumParams &p, int64_t fill_ctas, cudaStream_t s) {
    if (p.sum_ctas + fill_ctas > INT_MAX) return NVFP4_ERR_SHAPE;
    embedding_sum_kernel<T><<<(unsigned)(p.sum_ctas + fill_ctas), kSumThreads, 0, s>>>(p);
    count_launch();
    if (p.blocks > 1) {
        embedding_join_kernel<T><<<(unsigned)p.sum_ctas, kSumThreads, 0, s>>>(p);
        count_launch();
    }
    return cuda_status(cudaGetLastError());
}

// Sorts the tokens; l.keys[0] and l.at[0] hold the result, or [1] if it returns 1 in *which.
static int sort(const void *tokens, int wide, int T, int V, uint8_t *ws, const Layout &l, int *which, cudaStream_t s) {
    SortParams p = {};
    p.tokens = tokens;
    p.wide = wide;
    p.T = T;
    p.V = V;
    p.chunk = l.chunk;
    p.chunks = l.chunks;
    p.counts = reinterpret_cast<int *>(ws + l.counts);
    *which = 0;
    if (T <= kSmallTokens) {
        int n = 1;
        while (n < T) n *= 2;
        p.keys = reinterpret_cast<int *>(ws + l.keys[0]);
        p.at = reinterpret_cast<int *>(ws + l.at[0]);
        sort_small_kernel<<<1, kSortThreads, n * sizeof(uint64_t), s>>>(p, n);
        count_launch();
        return cuda_status(cudaGetLastError());
    }
    int bits = 1;  // of the largest key, V
    while (bits < 31 && (V >> bits) != 0) bits++;
    const int passes = (bits + kMaxBits - 1) / kMaxBits;
    for (int i = 0, done = 0; i < passes; i++) {
        p.shift = done;
        p.bits = (bits - done + passes - i - 1) / (passes - i);
        done += p.bits;
        p.keys_in = i ? reinterpret_cast<int *>(ws + l.keys[*which]) : nullptr;
        p.at_in = i ? reinterpret_cast<int *>(ws + l.at[*which]) : nullptr;
        if (i) *which ^= 1;
        p.keys = reinterpret_cast<int *>(ws + l.keys[*which]);
        p.at = reinterpret_cast<int *>(ws + l.at[*which]);
        sort_count_kernel<<<l.chunks, kSortThreads, 0, s>>>(p);
        sort_scatter_kernel<<<l.chunks, kSortThreads, 0, s>>>(p);
        count_launch();
        count_launch();
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

template <typename T>
static void lookup(const LookupParams &p, int token_bytes, unsigned grid, cudaStream_t s) {
    if (p.scale == 1.0f) {
        if (token_bytes == 8) embedding_kernel<T, int64_t, false><<<grid, kLookupThreads, 0, s>>>(p);
        else embedding_kernel<T, int, false><<<grid, kLookupThreads, 0, s>>>(p);
    } else {
        if (token_bytes == 8) embedding_kernel<T, int64_t, true><<<grid, kLookupThreads, 0, s>>>(p);
        else embedding_kernel<T, int, true><<<grid, kLookupThreads, 0, s>>>(p);
    }
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
    p.T = T;
    p.V = V;
    p.vecs = K / 8;
    p.lanes = std::min(embedding::kLookupThreads, (p.vecs + 31) / 32 * 32);
    p.per_cta = embedding::kLookupThreads / p.lanes;
    p.slabs = (p.vecs + p.lanes - 1) / p.lanes;
    const int64_t grid = ((int64_t)T + p.per_cta - 1) / p.per_cta * p.slabs;
    if (grid > INT_MAX) return NVFP4_ERR_SHAPE;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) embedding::lookup<__nv_bfloat16>(p, token_bytes, (unsigned)grid, s);
    else embedding::lookup<__half>(p, token_bytes, (unsigned)grid, s);
    count_launch();
    return cuda_status(cudaGetLastError());
}

size_t nvfp4_embedding_backward_workspace_size(int T, int V, int K) {
    if (T < 1 || V < 1 || K < 8 || T > embedding::kMaxRows || V > embedding::kMaxRows || K > embedding::kMaxRows)
        return 0;
    return embedding::layout(T, K).bytes;
}

int nvfp4_embedding_backward(const void *dY, int64_t ldy, const void *tokens, int token_bytes, float scale,
                             void *dTable, int T, int V, int K, int dtype, void *workspace, size_t workspace_bytes,
                             void *stream) {
    int st = embedding::check_sizes(tokens, token_bytes, ldy, T, V, K, dtype);
    if (st) return st;
    if (!dTable || (T && !dY)) return NVFP4_ERR_INVALID;
    if (!aligned16(dY) || !aligned16(dTable) || !aligned16(workspace)) return NVFP4_ERR_ALIGN;
    if (T && (!workspace || workspace_bytes < nvfp4_embedding_backward_workspace_size(T, V, K)))
        return NVFP4_ERR_WORKSPACE;
    const int slabs = (K + embedding::kSumCols - 1) / embedding::kSumCols;
    const embedding::Layout l = embedding::layout(T, K);
    if ((int64_t)l.blocks * slabs > INT_MAX) return NVFP4_ERR_SHAPE;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (T == 0)  // no token: the gradient is zero
        return cuda_status(cudaMemsetAsync(dTable, 0, (size_t)V * K * 2, s));
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    int which = 0;
    if ((st = embedding::sort(tokens, token_bytes == 8, T, V, ws, l, &which, s))) return st;
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
    p.sum_ctas = l.blocks * slabs;
    p.fill_rows = 64;
    const int64_t fill = ((int64_t)V + p.fill_rows - 1) / p.fill_rows;
    return dtype == NVFP4_BF16 ? embedding::sum<__nv_bfloat16>(p, fill, s) : embedding::sum<__half>(p, fill, s);
}

}  // extern "C"
