// logprobs.cu — log probabilities of given tokens from rows of logits, with the entropy and
// the most probable alternatives, and the gradient of the logits.
//
// One pass over a row.  With c = log2(e) / temperature and m the maximum so far, a thread keeps
//   S0 = sum 2^(c (x - m)),  S1 = sum c (x - m) 2^(c (x - m))
// and rescales both when its maximum moves, once for a batch of vectors at most.  Parts are
// joined the same way; then log p = (x - m) / temperature - ln S0 and the entropy is
// ln S0 - ln2 S1 / S0: nothing is subtracted that is large beside the result.
//
// At 8 instructions an element the pass was bound by their issue (2.8 TB/s).  So the exponents
// come from one fused multiply-add on pairs, c x - r with r = c m rounded (what the rounding
// leaves, c m - r, is known exactly and taken out of the sums at the end), and values far
// below the maximum, -inf and NaN among them, are first raised to a finite one, in pairs of
// 16-bit values, whose power of two is zero all the same.  Where that does not hold (nothing
// but masked logits so far, or a maximum near the type's lowest value), or c m is so large that
// its rounding is no small part of an exponent (past 2^24: masks of -1e9 and the like, in the
// parts of a row that hold nothing else), the exponents are taken one by one from the difference.
//
// A warp of its own copies the rows through a ring in shared memory, in bulk copies of 16 or 32 KB,
// and runs on into the next row while the others finish this one.
//
// Alternatives: a row's k-th highest value cannot be below the k-th highest of 32 disjoint
// parts' maxima, which the pass has at hand; only quarters of a thread's vectors whose maximum
// reaches that bound can hold a candidate, so a percent of the row is read again, and the
// candidates are ranked by counting.  The rare row with more candidates than are kept (long
// runs of equal logits) takes rounds of "highest value, lowest tokens first".
//
// A row is one CTA's, or is cut between the CTAs of a cluster when there are few rows (the parts
// meet in distributed shared memory), or a warp's when rows are short and many: a CTA's
// barriers and its last steps take 2.5 us a row, 5 with alternatives.  Every sum has a fixed
// order.
//
// Measured: 4096 rows of 131072 bf16, statistics 173 us (6.2 TB/s of a copy's 6.55), with the
// entropy 179, and 8 alternatives 221 (their second reading and the ranking, 5 us a row of a
// CTA; 238 where the logits are others in every call), 32 263; the gradient 329 (6.5 TB/s).  16000
// rows of 8000 52 us (4.9 TB/s).  Without
// alternatives the pass is bound by memory and nearly by issue (61 % of cycles; the unit of
// powers of two is 66 % busy).  One row of 50257 fp32 with 5 alternatives 9.1 us: launch, a pass of
// 3 us, the join of a cluster and the ranking.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int kResident = 3;       // CTAs an SM
constexpr int kRingBytes = 64 * 1024;  // a CTA's: chunks of a batch for each thread
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kCandidates = kThreads;  // one a thread when they are ranked
constexpr int kMaxCluster = 8;
constexpr int kRowWarps = 8, kRowResident = 4, kRowBatch = 4;  // of the kernel of short rows
constexpr int kQuarters = 4;         // of a thread's vectors, each with its maximum
constexpr float kCoolest = 1e-30f, kHottest = 1e30f;  // temperatures: c stays a normal number
// Vectors of a thread that are added up together: what a batch costs beside its elements (the
// wait, the maximum, the branches) is 2 instructions an element with 4, 4096 rows of 131072 in
// 191 us, and 180 with 8; with alternatives, 8 do not fit into the registers (218 us and 498).
template <bool TOP>
constexpr int kBatchOf = TOP ? 4 : 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -200.0f;    // 2^-200 is zero in fp32: where the exponents of masked logits are put

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Pairs of fp32 values.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The words of a vector.  floor: the finite value that -inf and NaN are raised to.
template <typename T>
struct Word {  // two 16-bit values
    static constexpr float kFloor = std::is_same<T, __half>::value ? -65504.0f : -1e20f;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 r = __hmax2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
            return *reinterpret_cast<const uint32_t *>(&r);
        } else {
            const __nv_bfloat162 r =
                __hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
            return *reinterpret_cast<const uint32_t *>(&r);
        }
    }
    // the maximum of a vector's values, NaN only if all are
    static __device__ __forceinline__ uint32_t top(const uint4 &v) { return max2(max2(v.x, v.y), max2(v.z, v.w)); }
    static __device__ __forceinline__ float top_value(uint32_t t) {
        const float2 f = Type16<T>::unpack(t);
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ void raised(const uint4 &v, uint64_t (&p)[4]) {
        const uint32_t floor = Type16<T>::pack(kFloor, kFloor), w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = Type16<T>::unpack(max2(w[i], floor));
            p[i] = pair(f.x, f.y);
        }
    }
    static constexpr int kPairs = 4;
    static constexpr uint32_t kMasked = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max2(a, b); }
};
template <>
struct Word<float> {
    static constexpr float kFloor = -1e20f;
    static __device__ __forceinline__ uint32_t top(const uint4 &v) {
        return __float_as_uint(fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                                     fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
    }
    static __device__ __forceinline__ float top_value(uint32_t t) { return __uint_as_float(t); }
    static __device__ __forceinline__ void raised(const uint4 &v, uint64_t (&p)[2]) {
        p[0] = pair(fmaxf(__uint_as_float(v.x), kFloor), fmaxf(__uint_as_float(v.y), kFloor));
        p[1] = pair(fmaxf(__uint_as_float(v.z), kFloor), fmaxf(__uint_as_float(v.w), kFloor));
    }
    static constexpr int kPairs = 2;
    static constexpr uint32_t kMasked = 0xff800000u;
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
};

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ float to_float(T v) {
    return Type16<T>::load(&v);
}
template <>
__device__ __forceinline__ float to_float<float>(float v) {
    return v;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &v, float (&f)[kVec<T>]) {
    if constexpr (sizeof(T) == 4) {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    } else {
        unpack8<T>(v, f);
    }
}

// c m up to which the exponents are c x - r: what r's rounding leaves of c m is then half a unit
// at most.  It is a factor of all sums until they are handed on, which 2^128 and more would end.
constexpr float kMostPaired = 0x1p24f;

// Whether a value raised to `floor` has the power of two zero, and a finite exponent.
__device__ __forceinline__ bool raises(float floor, float c, float r) {
    return c < 1e6f && fmaf(floor, c, -r) < -150.0f;
}

// The same the other way.
template <typename T>
__device__ __forceinline__ T value_of(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return Type16<T>::round(v);
}
template <typename T>
__device__ __forceinline__ uint4 vector_of(const float (&f)[kVec<T>]) {
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    else
        return pack8<T>(f);
}

// A row as 16-byte vectors at 16-byte addresses; the first and the last may reach past it.
template <typename T>
struct Row {
    const T *x;   // first element
    int shift;    // elements of the first vector before it
    int n;        // elements
    __device__ __forceinline__ Row(const T *p, int len)
        : x(p), shift((int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T))), n(len) {}
    __device__ __forceinline__ int vectors() const { return (int)(((int64_t)n + shift + kVec<T> - 1) / kVec<T>); }
    __device__ __forceinline__ int first(int v) const { return v * kVec<T> - shift; }  // may be negative
    // vectors [whole0(), whole1()) lie within the row
    __device__ __forceinline__ int whole0() const { return shift ? 1 : 0; }
    __device__ __forceinline__ int whole1() const { return (int)(((int64_t)n + shift) / kVec<T>); }
    __device__ __forceinline__ uint4 whole(int v) const {
        return __ldg(reinterpret_cast<const uint4 *>(x + first(v)));
    }
    // -inf past the row's ends; its elements alone are read
    __device__ __forceinline__ uint4 any(int v) const {
        if (v >= whole0() && v < whole1()) return whole(v);
        uint32_t w[4] = {Word<T>::kMasked, Word<T>::kMasked, Word<T>::kMasked, Word<T>::kMasked};
        const int e = first(v);
#pragma unroll
        for (int i = 0; i < kVec<T>; i++)
            if (e + i >= 0 && e + i < n) {
                if constexpr (sizeof(T) == 4) {
                    w[i] = __float_as_uint(x[e + i]);
                } else {
                    const uint32_t bits = reinterpret_cast<const uint16_t *>(x)[e + i];
                    w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | bits << 16 : (w[i / 2] & 0xffff0000u) | bits;
                }
            }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void load(int v, float (&f)[kVec<T>]) const { unpack<T>(any(v), f); }
};

struct Params {
    const void *logits, *targets;
    int64_t ld;
    int target8;       // targets are 64-bit
    int T, V, k;
    float temperature, c;  // c = log2(e) / temperature
    float *logprobs, *entropy, *top_logprobs, *lse;
    int *top_tokens;
    KernelCtl ctl;
};

__device__ __forceinline__ int64_t target_of(const void *targets, int wide, int64_t t) {
    return wide ? static_cast<const int64_t *>(targets)[t] : static_cast<const int *>(targets)[t];
}

// A number whose signed order is the floats' order, both zeros alike.
__device__ __forceinline__ int order_key(float v) {
    const int u = __float_as_int(v + 0.0f);
    return u ^ ((u >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float key_value(int key) { return __int_as_float(key ^ ((key >> 31) & 0x7fffffff)); }
// Unsigned order of (value, lowest token first).
__device__ __forceinline__ uint64_t pair_key(float v, int token) {
    return ((uint64_t)((uint32_t)order_key(v) ^ 0x80000000u) << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float pair_value(uint64_t k) { return key_value((int)((uint32_t)(k >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ int pair_token(uint64_t k) { return (int)~(uint32_t)k; }

struct Stats {
    float m, s0, s1;  // maximum (of the logits themselves), and the sums relative to it
};
// fmaxf takes the bound where the difference is NaN: of two infinities, or of a masked NaN.
__device__ __forceinline__ Stats join(const Stats &a, const Stats &b, float c) {
    Stats r;
    r.m = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - r.m) * c, kFar), db = fmaxf((b.m - r.m) * c, kFar);
    const float fa = ex2(da), fb = ex2(db);
    r.s0 = a.s0 * fa + b.s0 * fb;
    r.s1 = fmaf(a.s0, da, a.s1) * fa + fmaf(b.s0, db, b.s1) * fb;
    return r;
}
__device__ __forceinline__ Stats shuffle(const Stats &a, int o) {
    return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s0, o),
            __shfl_xor_sync(0xffffffffu, a.s1, o)};
}

// The sums of a thread's part of a row so far.
template <typename T, bool ENTROPY>
struct Sums {
    float m = -INFINITY, r = 0.0f, rest = 0.0f;  // r: c m rounded, rest: what that left
    uint64_t s0[2] = {0, 0}, s1[2] = {0, 0};
    bool paired = false;

    // N vectors more; their maximum
    template <int N>
    __device__ __forceinline__ float add(const uint4 (&raw)[N], float c) {
        uint32_t top = Word<T>::top(raw[0]);
#pragma unroll
        for (int b = 1; b < N; b++) top = Word<T>::join(top, Word<T>::top(raw[b]));
        const float high = Word<T>::top_value(top);
        if (high > m) {
            const float r_next = high * c;
            const bool pairs = raises(Word<T>::kFloor, c, r_next) && fabsf(r_next) < kMostPaired;
            const float rest_next = pairs ? fmaf(high, c, -r_next) : 0.0f;
            const float d = fmaxf((m - high) * c, kFar) - rest + rest_next, scale = ex2(d);
            const uint64_t dd = pair(d, d), ss = pair(scale, scale);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (ENTROPY) s1[i] = mul2(fma2(s0[i], dd, s1[i]), ss);
                s0[i] = mul2(s0[i], ss);
            }
            m = high;
            r = r_next;
            rest = rest_next;
            paired = pairs;
        }
        if (paired) {
            const uint64_t cc = pair(c, c), rr = pair(-r, -r);
#pragma unroll
            for (int b = 0; b < N; b++) {
                uint64_t x[Word<T>::kPairs];
                Word<T>::raised(raw[b], x);
#pragma unroll
                for (int i = 0; i < Word<T>::kPairs; i++) {
                    const uint64_t d = fma2(x[i], cc, rr);
                    const float2 f = unpair(d);
                    const uint64_t e = pair(ex2(f.x), ex2(f.y));
                    s0[i & 1] = add2(s0[i & 1], e);
                    if (ENTROPY) s1[i & 1] = fma2(d, e, s1[i & 1]);
                }
            }
        } else {
            // fmaxf takes the bound where the difference is NaN, of two infinities or of a NaN
            float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
            for (int b = 0; b < N; b++) {
                float f[kVec<T>];
                unpack<T>(raw[b], f);
#pragma unroll
                for (int i = 0; i < kVec<T>; i++) {
                    const float d = fmaxf((f[i] - m) * c, kFar), e = ex2(d);
                    t0 += e;
                    if (ENTROPY) t1 = fmaf(d, e, t1);
                }
            }
            s0[0] = add2(s0[0], pair(t0, 0.0f));
            if (ENTROPY) s1[0] = add2(s1[0], pair(t1, 0.0f));
        }
        return high;
    }
    __device__ __forceinline__ Stats stats() const {
        const float2 x = unpair(add2(s0[0], s0[1])), y = unpair(add2(s1[0], s1[1]));
        const float sum0 = x.x + x.y, sum1 = y.x + y.y, back = ex2(-rest);
        return {m, sum0 * back, ENTROPY ? fmaf(-rest, sum0, sum1) * back : 0.0f};
    }
};

// Barrier of the threads that add up, without the one that copies.
__device__ __forceinline__ void sync_adders() {
    __syncwarp();  // .aligned
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
}

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}

struct Shared {
    uint64_t cand[kCandidates];
    uint64_t top[kMaxTop];        // this CTA's alternatives, highest first
    Stats part[2][kWarps];
    float best[kQuarters][kThreads];  // the maxima of quarters of the threads' vectors
    int winners[kQuarters * kThreads];
    int count[kWarps + 1];
    int n_winners, n_cand, n_top;
};

// Ranks n <= kThreads distinct keys by counting; the first k to out.
__device__ __forceinline__ void rank_keys(const uint64_t *keys, int n, int k, uint64_t *out) {
    if ((int)threadIdx.x < n) {
        const uint64_t mine = keys[threadIdx.x];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += keys[j] > mine;
        if (rank < k) out[rank] = mine;
    }
}

// The alternatives of vectors [v0, v1) where equal values are too many to keep: the highest
// value that is left, then its tokens from the lowest, until there are k.  By the threads that
// add up, whose warps' counts meet in `count`, or (WARP) by one warp.  Returns how many.
template <typename T, bool WARP>
__device__ __noinline__ int select_rounds(const Row<T> &row, int v0, int v1, int k, uint64_t *top, int *count) {
    constexpr int kTeam = WARP ? 32 : kThreads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, me = WARP ? lane : (int)threadIdx.x;
    int have = 0, last = INT_MAX;  // order_key of +inf is below INT_MAX
    while (have < k) {
        int best = INT_MIN;
#pragma unroll 4
        for (int v = v0 + me; v < v1; v += kTeam) {
            float f[kVec<T>];
            row.load(v, f);
#pragma unroll
            for (int i = 0; i < kVec<T>; i++) {
                const int key = f[i] > -INFINITY ? order_key(f[i]) : INT_MIN;
                if (key < last) best = max(best, key);
            }
        }
        best = __reduce_max_sync(0xffffffffu, best);
        if (!WARP) {
            sync_adders();
            if (lane == 0) count[warp] = best;
            sync_adders();
            for (int w = 0; w < kWarps; w++) best = max(best, count[w]);
        }
        if (best == INT_MIN) break;
        for (int base = v0; base < v1 && have < k; base += kTeam) {
            const int v = base + me;
            float f[kVec<T>];
            int n = 0;
            if (v < v1) {
                row.load(v, f);
#pragma unroll
                for (int i = 0; i < kVec<T>; i++) n += f[i] > -INFINITY && order_key(f[i]) == best;
            }
            int before = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += u;
            }
            int at = have + before - n, total = __shfl_sync(0xffffffffu, before, 31);
            if (!WARP) {
                sync_adders();  // the counts of the round before have been read
                if (lane == 31) count[warp] = before;
                sync_adders();
                total = 0;
                for (int w = 0; w < kWarps; w++) {
                    if (w < warp) at += count[w];
                    total += count[w];
                }
            }
            if (n)
#pragma unroll
                for (int i = 0; i < kVec<T>; i++)
                    if (f[i] > -INFINITY && order_key(f[i]) == best) {
                        if (at < k) top[at] = pair_key(f[i], row.first(v) + i);
                        at++;
                    }
            have = min(k, have + total);
        }
        last = best;
    }
    return have;
}

// A warp's values, the highest first.
__device__ __forceinline__ float sort_lanes(float b, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, b, o);
            const bool high = ((lane & o) == 0) == ((lane & size) == 0);  // descending overall
            b = high ? fmaxf(b, other) : fminf(b, other);
        }
    return b;
}

// What a row's statistics say, by one thread; l = ln s0.
template <bool ENTROPY>
__device__ __forceinline__ void finish_row(const Params &p, int64_t t, const Stats &all, float l, bool ignored,
                                           float target) {
    const bool empty = all.m == -INFINITY;
    const bool none = !(target > -INFINITY);
    p.lse[t] = empty ? -INFINITY : all.m / p.temperature + l;
    p.logprobs[t] = ignored ? 0.0f : empty || none ? -INFINITY : (target - all.m) / p.temperature - l;
    if (ENTROPY) {
        const float H = l - all.s1 / all.s0 * kLn2;
        p.entropy[t] = empty || H < 0.0f ? 0.0f : H;  // below zero it is rounding
    }
}
// An alternative, by a lane: the `lane`-th of n.
__device__ __forceinline__ void put_top(const Params &p, int64_t t, const Stats &all, float l, const uint64_t *top,
                                        int n, int lane) {
    if (lane >= p.k) return;
    const int64_t at = t * p.k + lane;
    const float v = lane < n ? pair_value(top[lane]) : -INFINITY;
    p.top_tokens[at] = lane < n ? pair_token(top[lane]) : -1;
    p.top_logprobs[at] = lane < n ? (v - all.m) / p.temperature - l : -INFINITY;
}

template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kThreads + 32, kResident) logprobs_kernel(const Params p) {
    constexpr int kBatch = kBatchOf<TOP>, kChunk = kBatch * kThreads;  // vectors
    constexpr int kRing = kRingBytes / (kChunk * 16);
    extern __shared__ __align__(16) uint4 ring[];  // [kRing][kChunk]
    __shared__ Shared s;
    __shared__ uint64_t bars[2 * kRing];
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = (int)cluster_size(), part = (int)cluster_ctarank();
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kRing;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; i++) {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, kWarps);
        }
        abort_word = 0;
        fence_barrier_init();
    }
    __syncthreads();
    auto row_at = [&](int64_t t) { return Row<T>(static_cast<const T *>(p.logits) + t * p.ld, p.V); };
    auto from = [&](const Row<T> &row, int part) { return (int)((int64_t)row.vectors() * part / parts); };
    const int64_t first = blockIdx.x / parts, step = gridDim.x / parts;
    int slot = 0, phase = 0;  // of the ring
    auto pass_slot = [&] {
        if (++slot == kRing) {
            slot = 0;
            phase ^= 1;
        }
    };
    if (warp == kWarps) {
        // ---- copies: the whole vectors of the rows, chunk by chunk
        if (lane == 0) {
            uint32_t issued = 0, issued_phase = 0;
            bool ok = true;
            for (int64_t t = first; ok && t < p.T; t += step) {
                const Row<T> row = row_at(t);
                const int v0 = from(row, part), v1 = from(row, part + 1);
                for (int v = v0; v < v1; v += kChunk) {
                    if (!wait_parity(bar_empty + 8 * slot, phase ^ 1, p.ctl.wait_timeout_ns, abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        ok = false;
                        break;
                    }
                    const int a = max(v, row.whole0()), b = min(min(v + kChunk, v1), row.whole1());
                    if (a < b) {
                        const uint32_t bytes = (uint32_t)(b - a) * 16;
                        mbar_arrive_expect_tx(bar_full + 8 * slot, bytes);
                        issued |= 1u << slot;
                        issued_phase = (issued_phase & ~(1u << slot)) | ((uint32_t)phase << slot);
                        bulk_load(smem_u32(ring + slot * kChunk + (a - v)), row.x + row.first(a), bytes,
                                  bar_full + 8 * slot);
                    } else {
                        mbar_arrive(bar_full + 8 * slot);
                    }
                    pass_slot();
                }
            }
            if (!ok) {  // let the copies in flight land before the memory goes
                volatile int never = 0;
                for (int i = 0; i < kRing; i++)
                    if (issued & (1u << i))
                        wait_parity(bar_full + 8 * i, (issued_phase >> i) & 1, p.ctl.drain_timeout_ns, &never);
            }
        }
        return;
    }
    // the row's target, read a row ahead: its logit is under way while the row is summed
    const bool finishes = part == 0 && threadIdx.x == 0;
    int64_t next = finishes && first < p.T ? target_of(p.targets, p.target8, first) : -1;
    int turn = 0;  // of the statistics' two places
    for (int64_t t = first; t < p.T; t += step) {
        const Row<T> row = row_at(t);
        const int v0 = from(row, part), v1 = from(row, part + 1);
        float target = -INFINITY;
        bool ignored = true;
        if (finishes) {
            ignored = next < 0 || next >= p.V;
            if (!ignored) target = to_float<T>(row.x[next]);
            if (t + step < p.T) next = target_of(p.targets, p.target8, t + step);
        }
        // ---- the pass
        Sums<T, ENTROPY> sums;
        const int quarter = max(1, ((v1 - v0 + kBatch * kThreads - 1) / (kBatch * kThreads) + kQuarters - 1) / kQuarters);
        float high_quarter = -INFINITY;
        auto add = [&](const auto &raw) {
            const float high = sums.add(raw, p.c);
            if (TOP) high_quarter = fmaxf(high_quarter, high);
        };
        {
            int left = quarter;
            float *best = &s.best[0][threadIdx.x];
            const int w0 = row.whole0(), w1 = min(v1, row.whole1());
            for (int v = v0 + (int)threadIdx.x; v - (int)threadIdx.x < v1; v += kChunk) {
                // after a wait that gave up the sums are of anything, and the status says so
                if (!wait_parity(bar_full + 8 * slot, phase, p.ctl.wait_timeout_ns, abort_flag))
                    report_timeout(abort_flag, p.ctl.status);
                const uint4 *chunk = ring + slot * kChunk + threadIdx.x;
                if (v >= w0 && v + (kBatch - 1) * kThreads < w1) {
                    uint4 raw[kBatch];
#pragma unroll
                    for (int b = 0; b < kBatch; b++) raw[b] = chunk[b * kThreads];
                    add(raw);
                } else if (v >= w0 && v + kBatch / 2 * kThreads < w1) {  // the row's end, more than half a batch
                    const uint4 masked = make_uint4(Word<T>::kMasked, Word<T>::kMasked, Word<T>::kMasked, Word<T>::kMasked);
                    uint4 raw[kBatch];
#pragma unroll
                    for (int b = 0; b < kBatch; b++) raw[b] = v + b * kThreads < w1 ? chunk[b * kThreads] : masked;
                    add(raw);
                    for (int b = kBatch / 2; b < kBatch; b++)  // the vector that the row ends in
                        if (v + b * kThreads >= w1 && v + b * kThreads < v1) {
                            uint4 last[1] = {row.any(v + b * kThreads)};
                            add(last);
                        }
                } else {  // no more than its vectors
                    for (int b = 0; b < kBatch && v + b * kThreads < v1; b++) {
                        const int at = v + b * kThreads;
                        uint4 raw[1];
                        raw[0] = at >= w0 && at < w1 ? chunk[b * kThreads] : row.any(at);
                        add(raw);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_empty + 8 * slot);
                pass_slot();
                if (TOP && (--left == 0 || v - (int)threadIdx.x + kChunk >= v1)) {
                    *best = high_quarter;
                    best += kThreads;
                    high_quarter = -INFINITY;
                    left = quarter;
                }
            }
            if (TOP)
                for (; best < &s.best[kQuarters][0]; best += kThreads) *best = -INFINITY;
        }
        // ---- statistics of the CTA
        Stats w = sums.stats();
#pragma unroll
        for (int o = 16; o; o >>= 1) w = join(w, shuffle(w, o), p.c);
        if (lane == 0) s.part[turn][warp] = w;
        if (threadIdx.x == 0) s.n_winners = s.n_cand = s.n_top = 0;
        sync_adders();
        if (TOP) {
            // ---- candidates: the lanes' columns of maxima, sorted; the k-th is the bound
            float b = -INFINITY;
#pragma unroll
            for (int i = 0; i < kQuarters; i++)
#pragma unroll
                for (int w = 0; w < kWarps; w++) b = fmaxf(b, s.best[i][w * 32 + lane]);
            b = sort_lanes(b, lane);
            float bound = __shfl_sync(0xffffffffu, b, p.k - 1), high = __shfl_sync(0xffffffffu, b, 0);
            // of many alternatives the columns' bound is loose: while more than twice as many quarters as
            // there are alternatives reach it, halve the way up to the maximum, as far as enough still do
            auto reached = [&](float v) {
                int n = 0;
#pragma unroll
                for (int j = 0; j < kQuarters; j++)
#pragma unroll
                    for (int w = 0; w < kWarps; w++) n += s.best[j][w * 32 + lane] >= v;
                return __reduce_add_sync(0xffffffffu, n);
            };
            if (bound > -INFINITY) {
                int n = p.k > 8 ? reached(bound) : 0;
                for (int i = 0; i < 6 && n > 2 * p.k; i++) {
                    const float mid = 0.5f * bound + 0.5f * high;
                    const int at = reached(mid);
                    if (at >= p.k) {
                        bound = mid;
                        n = at;
                    } else {
                        high = mid;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kQuarters; i++) {
                const float mine = s.best[i][threadIdx.x];
                if (mine > -INFINITY && mine >= bound)
                    s.winners[atomicAdd(&s.n_winners, 1)] = i * kThreads + (int)threadIdx.x;
            }
            sync_adders();
            const int per = quarter * kBatch;  // vectors of a quarter, at most
            const int all = s.n_winners * per;
            // (more candidates than are kept, long runs of equal logits, are left to the rounds below)
            for (int i = threadIdx.x; i < all && *(volatile int *)&s.n_cand <= kCandidates; i += kThreads) {
                const int w = s.winners[i / per], v = v0 + w % kThreads + (w / kThreads * per + i % per) * kThreads;
                if (v >= v1) continue;
                float f[kVec<T>];
                row.load(v, f);
#pragma unroll
                for (int e = 0; e < kVec<T>; e++)
                    if (f[e] > -INFINITY && f[e] >= bound) {
                        const int at = atomicAdd(&s.n_cand, 1);
                        if (at < kCandidates) s.cand[at] = pair_key(f[e], row.first(v) + e);
                    }
            }
            sync_adders();
            const int n = s.n_cand;
            if (n <= kCandidates) {
                rank_keys(s.cand, n, p.k, s.top);
                if (threadIdx.x == 0) s.n_top = min(n, p.k);
            } else {
                const int n = select_rounds<T, false>(row, v0, v1, p.k, s.top, s.count);
                if (threadIdx.x == 0) s.n_top = n;
            }
        }
        // ---- join the CTAs' parts, finish the row
        if (parts > 1) {
            __syncwarp();
            cluster_sync();
        } else if (TOP) {
            sync_adders();
        }
        if (part == 0) {
            Stats all = {-INFINITY, 0.0f, 0.0f};
            if (warp == 0) {
                for (int i = lane; i < parts * kWarps; i += 32) {
                    const uint32_t at = map_to_cta(smem_u32(&s.part[turn][i % kWarps]), i / kWarps);
                    all = join(all, {ld_cluster_f32(at), ld_cluster_f32(at + 4), ld_cluster_f32(at + 8)}, p.c);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) all = join(all, shuffle(all, o), p.c);
                // lane 0's for all: a join's two sides round differently
                all.m = __shfl_sync(0xffffffffu, all.m, 0);
                all.s0 = __shfl_sync(0xffffffffu, all.s0, 0);
                all.s1 = __shfl_sync(0xffffffffu, all.s1, 0);
            }
            const float l = logf(all.s0);
            if (threadIdx.x == 0) finish_row<ENTROPY>(p, t, all, l, ignored, target);
            if (TOP) {
                int n = s.n_top;  // of this CTA
                if (parts > 1) {
                    // the candidates have been ranked: their place takes the parts' lists; a key's rank is
                    // the number of keys above it in all of them
                    const int q = threadIdx.x / kMaxTop, j = threadIdx.x % kMaxTop;
                    uint64_t mine = 0;
                    if (q < parts) {
                        const int have = __float_as_int(ld_cluster_f32(map_to_cta(smem_u32(&s.n_top), q)));
                        if (j == 0) s.winners[q] = have;
                        if (j < have) s.cand[threadIdx.x] = mine = ld_cluster_u64(map_to_cta(smem_u32(&s.top[j]), q));
                    }
                    sync_adders();
                    n = 0;
                    for (int o = 0; o < parts; o++) n += s.winners[o];
                    n = min(n, p.k);
                    int above[kMaxCluster] = {};  // in each list, by halving steps, the lists side by side
                    if (mine)
#pragma unroll
                        for (int step = kMaxTop; step; step >>= 1)
#pragma unroll
                            for (int o = 0; o < kMaxCluster; o++)
                                if (o < parts && above[o] + step <= s.winners[o] &&
                                    s.cand[o * kMaxTop + above[o] + step - 1] > mine)
                                    above[o] += step;
                    int rank = 0;
#pragma unroll
                    for (int o = 0; o < kMaxCluster; o++) rank += above[o];
                    sync_adders();  // every list has been read
                    if (mine && rank < p.k) s.top[rank] = mine;
                    sync_adders();
                }
                if (warp == 0) put_top(p, t, all, l, s.top, n, lane);
            }
        }
        if (parts > 1) {
            __syncwarp();
            cluster_sync();  // the first CTA has read the others' parts
        } else if (TOP) {
            sync_adders();
        } else {  // the first warp finishes this row while the others begin the next
            turn ^= 1;
        }
    }
}

// Short rows, a warp each, in the same steps: nothing waits for a CTA.
template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(32 * kRowWarps, kRowResident) logprobs_rows_kernel(const Params p) {
    __shared__ uint64_t cands[TOP ? kRowWarps : 1][kCandidates], tops[TOP ? kRowWarps : 1][kMaxTop];
    __shared__ int counts[kRowWarps];
    __shared__ uint8_t lists[kRowWarps][32 * kRowBatch];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * kRowWarps + warp;
    if (t >= p.T) return;
    const Row<T> row(static_cast<const T *>(p.logits) + t * p.ld, p.V);
    const int nv = row.vectors(), w0 = row.whole0(), w1 = row.whole1();
    const uint4 masked = make_uint4(Word<T>::kMasked, Word<T>::kMasked, Word<T>::kMasked, Word<T>::kMasked);
    auto load = [&](int v, uint4 (&raw)[kRowBatch]) {
#pragma unroll
        for (int b = 0; b < kRowBatch; b++) raw[b] = v + b * 32 < w1 ? row.whole(v + b * 32) : masked;
    };
    uint4 next[kRowBatch];
    load(w0 + lane, next);
    const int64_t at = lane == 0 ? target_of(p.targets, p.target8, t) : -1;
    // the vectors that the row begins and ends in
    const int edge = lane == 0 && w0 ? 0 : lane == 1 && w1 < nv && nv > w0 ? nv - 1 : -1;
    uint4 ends[1] = {edge >= 0 ? row.any(edge) : masked};
    const bool ignored = at < 0 || at >= p.V;
    const float target = ignored ? -INFINITY : to_float<T>(row.x[at]);
    Sums<T, ENTROPY> sums;
    uint32_t best[kRowBatch];  // maxima of the lane's vectors, by their place in the batch
#pragma unroll
    for (int b = 0; b < kRowBatch; b++) best[b] = Word<T>::kMasked;
    for (int v = w0; v < w1; v += 32 * kRowBatch) {
        uint4 raw[kRowBatch];
#pragma unroll
        for (int b = 0; b < kRowBatch; b++) raw[b] = next[b];
        if (v + 32 * kRowBatch < w1) load(v + 32 * kRowBatch + lane, next);
        sums.add(raw, p.c);
        if (TOP)
#pragma unroll
            for (int b = 0; b < kRowBatch; b++) best[b] = Word<T>::join(best[b], Word<T>::top(raw[b]));
    }
    if (w0 || w1 < nv) sums.add(ends, p.c);
    Stats all = sums.stats();
#pragma unroll
    for (int o = 16; o; o >>= 1) all = join(all, shuffle(all, o), p.c);
    // lane 0's for all: a join's two sides round differently
    all.m = __shfl_sync(0xffffffffu, all.m, 0);
    all.s0 = __shfl_sync(0xffffffffu, all.s0, 0);
    const float l = logf(all.s0);
    if (lane == 0) finish_row<ENTROPY>(p, t, all, l, ignored, target);
    if constexpr (TOP) {
        uint64_t *cand = cands[warp], *top = tops[warp];
        int *n_cand = &counts[warp];
        uint8_t *list = lists[warp];
        // the k-th highest of the lanes' maxima, then, while more than twice as many of their four
        // parts each as there are alternatives reach it, halfway up to the highest
        float part[kRowBatch], b = -INFINITY;
#pragma unroll
        for (int i = 0; i < kRowBatch; i++) b = fmaxf(b, part[i] = Word<T>::top_value(best[i]));
        b = sort_lanes(b, lane);
        float bound = __shfl_sync(0xffffffffu, b, p.k - 1), high = __shfl_sync(0xffffffffu, b, 0);
        auto reached = [&](float v) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < kRowBatch; i++) n += part[i] >= v;
            return __reduce_add_sync(0xffffffffu, n);
        };
        if (bound > -INFINITY) {
            int n = reached(bound);
            for (int i = 0; i < 6 && n > 2 * p.k; i++) {
                const float mid = 0.5f * bound + 0.5f * high;
                const int at = reached(mid);
                if (at >= p.k) {
                    bound = mid;
                    n = at;
                } else {
                    high = mid;
                }
            }
        }
        int winners = 0;
#pragma unroll
        for (int i = 0; i < kRowBatch; i++) {
            const bool wins = part[i] > -INFINITY && part[i] >= bound;
            const uint32_t all = __ballot_sync(0xffffffffu, wins);
            if (wins) list[winners + __popc(all & ((1u << lane) - 1u))] = (uint8_t)(i * 32 + lane);
            winners += __popc(all);
        }
        if (lane == 0) *n_cand = 0;
        __syncwarp();
        auto take = [&](const uint4 &raw, int v) {
            float f[kVec<T>];
            unpack<T>(raw, f);
#pragma unroll
            for (int e = 0; e < kVec<T>; e++)
                if (f[e] > -INFINITY && f[e] >= bound) {
                    const int i = atomicAdd(n_cand, 1);
                    if (i < kCandidates) cand[i] = pair_key(f[e], row.first(v) + e);
                }
        };
        if (edge >= 0) take(ends[0], edge);
        const int per = (w1 - w0 + 32 * kRowBatch - 1) / (32 * kRowBatch), items = per * winners;
#pragma unroll 4
        for (int i = lane; i < items; i += 32) {
            const int which = i / per, v = w0 + list[which] + (i - which * per) * 32 * kRowBatch;
            if (v >= w1) continue;
            const uint4 raw = row.whole(v);
            if (Word<T>::top_value(Word<T>::top(raw)) >= bound) take(raw, v);
        }
        __syncwarp();
        int n = *(volatile int *)n_cand;
        if (n <= kCandidates) {
            for (int i = lane; i < n; i += 32) {
                const uint64_t mine = cand[i];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < n; j++) rank += cand[j] > mine;
                if (rank < p.k) top[rank] = mine;
            }
            n = min(n, p.k);
        } else {
            n = select_rounds<T, true>(row, 0, nv, p.k, top, nullptr);
        }
        __syncwarp();
        put_top(p, t, all, l, top, n, lane);
    }
}

// ------------------------------------------------------------------------- gradient
struct GradParams {
    const float *dlogprobs, *dentropy, *lse, *entropy;
    const void *logits, *targets;
    void *dlogits;
    int64_t ld, ldd;
    int target8;
    int V, W;
    int64_t n_rows;
    int chunks;  // CTAs of a row
    int wide;    // log2 of a row's threads in a CTA, which has several short rows
    float inv_temperature;
};

constexpr int kGradThreads = 256;
constexpr int kGradBatch = 4;

// |lse| up to which the probabilities come from it.  It is one rounded number, so log p is off by up
// to 4e-7 of it: 1e-4 for 16-bit results, 3e-5 for fp32.  Beyond that it says too little (past 2^29
// nothing of ln s is left in it), and the row is summed again.
template <typename T>
constexpr float kMostLse = sizeof(T) == 4 ? 64.0f : 256.0f;

// A row whose lse says too little, by one CTA, or (WARP) one warp: its maximum m and sum s once
// more, then d from 2^(c (x - m)) / s, as the log probabilities' own kernel has it.  One reader of
// the whole row, which writes behind its last read: in place too.  Not inlined and with one load in
// flight, so that the kernel's registers are those of the other rows; 4096 rows of 131072 bf16 that
// are all of this sort take 875 us where the others take 329.
template <typename T, bool WARP>
__device__ __noinline__ void far_row(const GradParams &p, int64_t t) {
    constexpr int kTeam = WARP ? 32 : kGradThreads;
    const int me = threadIdx.x & (kTeam - 1), lane = threadIdx.x & 31;
    const float c = p.inv_temperature * kLog2e;
    const T *x = static_cast<const T *>(p.logits) + t * p.ld;
    T *d = static_cast<T *>(p.dlogits) + t * p.ldd;
    const bool whole = (reinterpret_cast<uintptr_t>(x) & 15u) == 0, whole_out = (reinterpret_cast<uintptr_t>(d) & 15u) == 0;
    const uint32_t V = p.V, W = p.W;  // a place past them by a team's elements is no negative number
    // kVec elements from e on, -inf past the row's n.  Pieces count from the row's start, whatever
    // its alignment, for the same bits
    auto load = [&](uint32_t e, uint32_t n, float (&f)[kVec<T>]) {
        if (whole && e + kVec<T> <= n) {
            unpack<T>(*reinterpret_cast<const uint4 *>(x + e), f);
        } else {
#pragma unroll
            for (int i = 0; i < kVec<T>; i++) f[i] = e + i < n ? to_float<T>(x[e + i]) : -INFINITY;
        }
    };
    Stats all = {-INFINITY, 0.0f, 0.0f};
#pragma unroll 1
    for (uint32_t e = me * kVec<T>; e < V; e += kTeam * kVec<T>) {
        float f[kVec<T>], high = -INFINITY, sum = 0.0f;
        load(e, V, f);
#pragma unroll
        for (int i = 0; i < kVec<T>; i++) high = fmaxf(high, f[i]);
        if (high > all.m) {
            all.s0 *= ex2(fmaxf((all.m - high) * c, kFar));
            all.m = high;
        }
#pragma unroll
        for (int i = 0; i < kVec<T>; i++) sum += ex2(fmaxf((f[i] - all.m) * c, kFar));
        all.s0 += sum;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) all = join(all, shuffle(all, o), c);
    if constexpr (!WARP) {
        __shared__ Stats part[kGradThreads / 32];
        if (lane == 0) part[threadIdx.x >> 5] = all;
        __syncthreads();
        all = part[0];
        for (int w = 1; w < kGradThreads / 32; w++) all = join(all, part[w], c);
    } else {  // lane 0's for all: a join's two sides round differently
        all.m = __shfl_sync(0xffffffffu, all.m, 0);
        all.s0 = __shfl_sync(0xffffffffu, all.s0, 0);
    }
    const float ln_s = logf(all.s0), inv_s = 1.0f / all.s0;
    const int64_t target = target_of(p.targets, p.target8, t);
    const float g = target >= 0 && target < p.V ? p.dlogprobs[t] * p.inv_temperature : 0.0f;
    const float h = p.dentropy ? p.dentropy[t] * p.inv_temperature : 0.0f;
    const float a = p.dentropy ? fmaf(h, p.entropy[t], g) : g;
#pragma unroll 1
    for (uint32_t e = me * kVec<T>; e < W; e += kTeam * kVec<T>) {
        float f[kVec<T>];
        load(e, W, f);
#pragma unroll
        for (int i = 0; i < kVec<T>; i++) {
            float y = 0.0f;
            if (e + i < V && f[i] > -INFINITY) {
                const float off = f[i] - all.m, q = ex2(off * c) * inv_s;
                y = q == 0.0f ? 0.0f : -q * fmaf(h, fmaf(off, p.inv_temperature, -ln_s), a);
                if (e + i == target) y += g;
            }
            f[i] = y;
        }
        if (whole_out && e + kVec<T> <= W) {
            *reinterpret_cast<uint4 *>(d + e) = vector_of<T>(f);
        } else {
#pragma unroll
            for (int i = 0; i < kVec<T>; i++)
                if (e + i < W) d[e + i] = value_of<T>(f[i]);
        }
    }
}

// Elementwise, with the row's scalars in registers: bound by reading and writing the logits.
// SAME: the gradient's rows have the logits' alignment, so whole vectors go out.  SHORT: a CTA
// has several rows (16000 of 1500 50 -> 28 us; with long ones in the same code 326 -> 381).
template <typename T, bool SAME, bool SHORT>
__global__ void __launch_bounds__(kGradThreads, SHORT && SAME ? 4 : SAME ? 5 : 8)
    logprobs_grad_kernel(const __grid_constant__ GradParams p) {
    const int team = SHORT ? 1 << p.wide : kGradThreads, me = SHORT ? threadIdx.x & (team - 1) : threadIdx.x;
    int64_t t;
    int chunk = 0;
    if constexpr (SHORT) {
        t = (int64_t)blockIdx.x * (kGradThreads >> p.wide) + (threadIdx.x >> p.wide);
        if (t >= p.n_rows) return;
    } else {
        t = blockIdx.x / p.chunks;
        chunk = (int)(blockIdx.x - t * p.chunks);
    }
    const T *x = static_cast<const T *>(p.logits) + t * p.ld;
    T *d = static_cast<T *>(p.dlogits) + t * p.ldd;
    const int64_t target = target_of(p.targets, p.target8, t);
    const float g = target >= 0 && target < p.V ? p.dlogprobs[t] * p.inv_temperature : 0.0f;
    const float h = p.dentropy ? p.dentropy[t] * p.inv_temperature : 0.0f;
    const float H = p.dentropy ? p.entropy[t] : 0.0f;
    const float lse = p.lse[t];
    const bool far = !(fabsf(lse) <= kMostLse<T>);
    const float a = fmaf(h, H, g);  // d = -p (g + h H + h log p)
    // Away from the target in pairs, from log2 p = c x - c lse: -inf and NaN are raised as in the
    // forward pass, where that leaves them at zero.
    const float c = p.inv_temperature * kLog2e, lse2 = lse * kLog2e, b = -h * kLn2;
    const bool paired = raises(Word<T>::kFloor, c, lse2);
    const uint64_t cc = pair(c, c), ll = pair(-lse2, -lse2), aa = pair(-a, -a), bb = pair(b, b);
    auto grad = [&](float v, int64_t e) {  // one element, the same bits
        if (e >= p.V || !(v > -INFINITY)) return 0.0f;
        float y;
        if (paired) {
            const float l = fmaf(fmaxf(v, Word<T>::kFloor), c, -lse2);
            y = ex2(l) * fmaf(b, l, -a);
        } else {
            const float l = fmaf(v, p.inv_temperature, -lse), q = ex2(l * kLog2e);
            y = q == 0.0f ? 0.0f : -q * fmaf(h, l, a);
        }
        return e == target ? y + g : y;
    };
    if constexpr (SAME) {
        const Row<T> row(x, p.W);
        const int nv = row.vectors();
        const int64_t v0 = (int64_t)chunk * kGradBatch * kGradThreads + me;
        uint4 raw[kGradBatch];
#pragma unroll
        for (int i = 0; i < kGradBatch; i++) {
            const int64_t v = v0 + i * team;
            const int64_t e = v * kVec<T> - row.shift;
            if (v < nv && e >= 0 && e + kVec<T> <= p.W) raw[i] = *reinterpret_cast<const uint4 *>(x + e);
        }
        const int n_out = far ? 0 : nv;  // asked once the logits are on their way
#pragma unroll
        for (int i = 0; i < kGradBatch; i++) {
            const int64_t v = v0 + i * team;
            if (v >= n_out) break;
            const int64_t e = v * kVec<T> - row.shift;
            if (e >= 0 && e + kVec<T> <= p.W) {
                float f[kVec<T>];
                if (paired && e + kVec<T> <= p.V && (target < e || target >= e + kVec<T>)) {
                    uint64_t w[Word<T>::kPairs];
                    Word<T>::raised(raw[i], w);
#pragma unroll
                    for (int j = 0; j < Word<T>::kPairs; j++) {
                        const uint64_t l = fma2(w[j], cc, ll);
                        const float2 x = unpair(l);
                        const float2 y = unpair(mul2(pair(ex2(x.x), ex2(x.y)), fma2(bb, l, aa)));
                        f[2 * j] = y.x;
                        f[2 * j + 1] = y.y;
                    }
                } else {
                    unpack<T>(raw[i], f);
#pragma unroll
                    for (int j = 0; j < kVec<T>; j++) f[j] = grad(f[j], e + j);
                }
                *reinterpret_cast<uint4 *>(d + e) = vector_of<T>(f);
            } else {
                for (int j = 0; j < kVec<T>; j++)
                    if (e + j >= 0 && e + j < p.W) d[e + j] = value_of<T>(grad(to_float<T>(x[e + j]), e + j));
            }
        }
    } else {
        const int64_t e0 = (int64_t)chunk * kGradBatch * kGradThreads * kVec<T> + me;
        const int64_t n_out = far ? 0 : min((int64_t)p.W, e0 + kGradBatch * kVec<T> * team);
#pragma unroll 4
        for (int64_t e = e0; e < n_out; e += team) d[e] = value_of<T>(grad(to_float<T>(x[e]), e));
    }
    if (far && chunk == 0 && (!SHORT || me < 32)) far_row<T, SHORT>(p, t);
}

// ------------------------------------------------------------------------- host side
// CTAs that share a row: as many as keep all rows' at two an SM, while each has a vector for
// every thread, or, with alternatives, enough of them for the join of the lists (2-4 us).  us, by
// 1, 2, 4 and 8 CTAs, bf16: 16 rows of 131072 13.4, 10.8, 8.8, 8.6, with 20 alternatives 19.2,
// 15.8, 13.4, 13.2; 16 of 50257 with 5 13.0, 13.3, 12.8, 13.0, of 25600 10.8, 11.0, 10.9, 12.9; 55
// of 131072 14.7, 11.6, 10.8, 14.8 (8 would be three an SM); 300 rows 25.4, 25.4, 29.6, 42.5.
// A cluster has one row: its copies do not run on into a next one, for which its other warps
// would have to give slots back before they meet the cluster.
static int parts_of(int T, int64_t vectors, bool top, int sm_count) {
    const int64_t least = top ? 1536 : kThreads;
    int parts = 1;
    if (top && vectors < 4 * least) return parts;
    while (parts < kMaxCluster && (int64_t)T * parts <= sm_count && vectors >= parts * 2 * least) parts *= 2;
    return parts;
}

// Whether a row is a warp's: short ones of which there are many.  us, a CTA a row and a warp a
// row, bf16 with entropy: 16000 rows of 1000 90 and 15, with 8 alternatives 195 and 25; of 8000
// 136 and 52, 231 and 75; 592 rows of 4000 8.8 and 7.4, 15 and 11; 1200 of 8000 16 and 13, 23 and
// 17; 2400 of 16000 29 and 25, 46 and 35; but 256 of 8000 8.8 and 10.6, 2400 of 32000 39 and 45.
static bool short_rows(int T, int64_t bytes, int sm_count) {
    return bytes <= 32768 && T > kResident * sm_count * std::max<int64_t>(1, bytes / 8192);
}

template <typename T, bool ENTROPY, bool TOP>
static int launch(const Params &p, const DeviceInfo &di, cudaStream_t s) {
    if (short_rows(p.T, p.V * (int64_t)sizeof(T), di.sm_count)) {
        logprobs_rows_kernel<T, ENTROPY, TOP><<<(unsigned)((p.T + kRowWarps - 1) / kRowWarps), 32 * kRowWarps, 0, s>>>(p);
        count_launch();
        return cuda_status(cudaGetLastError());
    }
    const int parts = parts_of(p.T, p.V / kVec<T>, TOP, di.sm_count);
    static std::atomic<bool> configured[64] = {};
    if (!configured[di.device].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(logprobs_kernel<T, ENTROPY, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kRingBytes) !=
            cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(parts == 1 ? std::min<int64_t>(p.T, kResident * di.sm_count) : p.T * parts));
    cfg.blockDim = dim3(kThreads + 32);
    cfg.dynamicSmemBytes = kRingBytes;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, logprobs_kernel<T, ENTROPY, TOP>, p) != cudaSuccess) return NVFP4_ERR_CUDA;
    count_launch();
    return cuda_status(cudaGetLastError());
}

template <typename T>
static int forward(const Params &p, const DeviceInfo &di, cudaStream_t s) {
    if (p.entropy) return p.k ? launch<T, true, true>(p, di, s) : launch<T, true, false>(p, di, s);
    return p.k ? launch<T, false, true>(p, di, s) : launch<T, false, false>(p, di, s);
}

// CTAs of a row's gradient, at any alignment of the row.
static int grad_chunks(int W, int size) {
    const int64_t per = 16 / size, vectors = ((int64_t)W + 2 * per - 2) / per;
    return (int)((vectors + kGradBatch * kGradThreads - 1) / (kGradBatch * kGradThreads));
}

template <typename T>
static int backward(GradParams p, int64_t n_rows, cudaStream_t s) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p.logits), to = reinterpret_cast<uintptr_t>(p.dlogits);
    const bool same = ((from - to) & 15u) == 0 && ((p.ld - p.ldd) * (int64_t)sizeof(T)) % 16 == 0;
    p.chunks = grad_chunks(p.W, sizeof(T));
    // a short row's threads: as many as have four vectors each, 32 at least
    const int64_t vectors = ((int64_t)p.W + 2 * kVec<T> - 2) / kVec<T>;
    for (p.wide = 5; (kGradBatch << p.wide) < vectors && (1 << p.wide) < kGradThreads;) p.wide++;
    p.n_rows = n_rows;
    const int64_t rows = kGradThreads >> p.wide;
    const unsigned grid = (unsigned)(rows > 1 ? (n_rows + rows - 1) / rows : n_rows * p.chunks);
    if (rows > 1) {
        if (same) logprobs_grad_kernel<T, true, true><<<grid, kGradThreads, 0, s>>>(p);
        else logprobs_grad_kernel<T, false, true><<<grid, kGradThreads, 0, s>>>(p);
    } else {
        if (same) logprobs_grad_kernel<T, true, false><<<grid, kGradThreads, 0, s>>>(p);
        else logprobs_grad_kernel<T, false, false><<<grid, kGradThreads, 0, s>>>(p);
    }
    count_launch();
    return cuda_status(cudaGetLastError());
}

static bool misaligned(const void *p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// What both directions check of the logits and targets.
static int check_rows(const void *logits, int64_t ld, int dtype, const void *targets, int target_bytes, int T, int V,
                      int W, float temperature) {
    if (dtype < NVFP4_BF16 || dtype > NVFP4_F32 || (target_bytes != 4 && target_bytes != 8)) return NVFP4_ERR_INVALID;
    if (!(temperature >= kCoolest) || !(temperature <= kHottest)) return NVFP4_ERR_INVALID;
    if (T < 0 || V < 1 || V > INT_MAX - 1024 || W < V || W > INT_MAX - 1024 || ld < W) return NVFP4_ERR_SHAPE;
    if (T && (!logits || !targets)) return NVFP4_ERR_INVALID;
    if (misaligned(logits, dtype == NVFP4_F32 ? 4 : 2) || misaligned(targets, target_bytes)) return NVFP4_ERR_ALIGN;
    return NVFP4_OK;
}

}  // namespace logprobs
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

int nvfp4_token_logprobs(const void *logits, int64_t ld, int dtype, const void *targets, int target_bytes, int T,
                         int V, int top_k, float temperature, float *logprobs, float *entropy, float *top_logprobs,
                         int32_t *top_tokens, float *lse, void *stream) {
    int st = logprobs::check_rows(logits, ld, dtype, targets, target_bytes, T, V, V, temperature);
    if (st) return st;
    if (top_k < 0 || top_k > logprobs::kMaxTop) return NVFP4_ERR_SHAPE;
    if (T && (!logprobs || !lse || (top_k && (!top_logprobs || !top_tokens)))) return NVFP4_ERR_INVALID;
    if (logprobs::misaligned(logprobs, 4) || logprobs::misaligned(entropy, 4) || logprobs::misaligned(lse, 4) ||
        logprobs::misaligned(top_logprobs, 4) || logprobs::misaligned(top_tokens, 4))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    logprobs::Params p = {};
    p.logits = logits;
    p.targets = targets;
    p.ld = ld;
    p.target8 = target_bytes == 8;
    p.T = T;
    p.V = V;
    p.k = top_k;
    p.temperature = temperature;
    p.c = logprobs::kLog2e / temperature;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.top_logprobs = top_logprobs;
    p.top_tokens = top_tokens;
    p.lse = lse;
    if ((st = kernel_ctl(&p.ctl))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) return logprobs::forward<__nv_bfloat16>(p, di, s);
    if (dtype == NVFP4_F16) return logprobs::forward<__half>(p, di, s);
    return logprobs::forward<float>(p, di, s);
}

int nvfp4_token_logprobs_backward(const float *dlogprobs, const float *dentropy, const void *logits, int64_t ld,
                                  int dtype, const void *targets, int target_bytes, const float *lse,
                                  const float *entropy, int T, int V, int W, float temperature, void *dlogits,
                                  int64_t ldd, void *stream) {
    int st = logprobs::check_rows(logits, ld, dtype, targets, target_bytes, T, V, W, temperature);
    if (st) return st;
    if (ldd < W || (int64_t)T * logprobs::grad_chunks(W, dtype == NVFP4_F32 ? 4 : 2) > INT_MAX) return NVFP4_ERR_SHAPE;
    if (T && (!dlogprobs || !lse || !dlogits || (dentropy && !entropy))) return NVFP4_ERR_INVALID;
    if (logprobs::misaligned(dlogprobs, 4) || logprobs::misaligned(dentropy, 4) || logprobs::misaligned(lse, 4) ||
        logprobs::misaligned(entropy, 4) || logprobs::misaligned(dlogits, dtype == NVFP4_F32 ? 4 : 2))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    logprobs::GradParams p = {};
    p.dlogprobs = dlogprobs;
    p.dentropy = dentropy;
    p.lse = lse;
    p.entropy = entropy;
    p.logits = logits;
    p.targets = targets;
    p.dlogits = dlogits;
    p.ld = ld;
    p.ldd = ldd;
    p.target8 = target_bytes == 8;
    p.V = V;
    p.W = W;
    p.inv_temperature = 1.0f / temperature;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) return logprobs::backward<__nv_bfloat16>(p, T, s);
    if (dtype == NVFP4_F16) return logprobs::backward<__half>(p, T, s);
    return logprobs::backward<float>(p, T, s);
}

}  // extern "C"
