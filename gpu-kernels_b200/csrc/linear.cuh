// linear.cuh — what the 16-bit linear kernels share: the tcgen05 kind::f16 forms, the
// epilogue's arithmetic, row-group tables and launch parameters.
//
// All of them compute with the FEATURES of the output on the MMA's M side (the weight is
// operand A) and the TOKENS on its N side: N is a run-time field of the instruction, so a
// tile of a ragged group costs what its own rows cost (in steps of 32 on a CTA pair, of 16 on
// one CTA, up to 256), and the same orientation streams the weights for a single token.
#pragma once
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "epilogue.cuh"
#include "ptx.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace linear {

constexpr int kMaxGroups = 256;
constexpr int kMaxExtent = INT32_MAX - 1023;       // of rows and columns: rounding up to a tile stays in 32 bits
constexpr int kBlockK = 64;                        // reduction elements of a ring slot: one 128-byte swizzle row
constexpr int kTileBytes = 128 * kBlockK * 2;      // one CTA's A tile: 128 features

// Forward:  Y[t, n] = sum_k W[n, k] X[t, k]     A = W as stored, B = X as stored
// Dgrad:    dX[t, k] = sum_n W[n, k] dZ[t, n]   A = W with the reduction along its rows
// Wgrad:    dW[n, k] = sum_t dZ[t, n] X[t, k]   both with the reduction (tokens) along rows
// "Along its rows": the operand is staged as 64-element chunks of a row by 64 rows and read
// by the MMA as an M/N-major operand, so nothing is ever transposed in memory.
enum Form : int { kForward = 0, kDgrad = 1, kWgrad = 2 };

struct Params {
    void *y;               // output: [m_total, out_cols], wgrad [groups * features, out_cols]
    void *z;               // forward: pre-activation [m_total, features], or null
    const void *bias;      // [groups, features] or null
    const void *residual;  // [m_total, out_cols] or null
    const int *m_offsets;  // [groups + 1] on the device, or null: one group of m_total rows
    int groups, m_total;
    int features;          // output features: N (forward, wgrad) or K (dgrad)
    int red;               // reduction length: K (forward), N (dgrad); wgrad: the group's rows
    int out_cols;          // row length of y
    int bt;                // tokens of a tile (wgrad: output columns of a tile)
    int wide;              // 1: a tile is two of them beside each other, sharing the A tile
    int strip;             // feature tiles that sweep the tokens together (L2 reuse)
    int act;
    int splits;            // decode: CTAs that share a tile's reduction
    int stages;            // ring slots
    int ncap;              // decode: token rows of a ring slot
    KernelCtl ctl;
};

// Instruction descriptor of kind::f16 (bf16 x bf16 or f16 x f16 -> fp32): bit 4 fp32 D,
// bits 7-9 / 10-12 the A / B format (0 f16, 1 bf16), bits 15 / 16 set when A / B is
// M/N-major, bits 17-22 N >> 3, bits 24-28 M >> 4.
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, bool a_mn, bool b_mn, uint32_t m, uint32_t n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Shared-memory descriptors of a 128-byte-swizzled operand (layout 2).
// K-major: rows of 128 bytes (64 K), groups of 8 rows every 1024 bytes; 16 K = 32 bytes.
// M/N-major: chunks of 64 M/N elements by 64 K rows of 128 bytes; chunks every 8192 bytes
// (leading offset), groups of 8 K rows every 1024 bytes (stride offset); 16 K = 2048 bytes.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return MN ? smem_desc(addr, 64 * 128, 1024, 2) : smem_desc(addr, 16, 1024, 2);
}
template <bool MN>
constexpr uint32_t kStep16 = MN ? 2048 >> 4 : 32 >> 4;  // descriptor advance of 16 K

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 3-D tiled loads (weights: [group][row][column], so a tile never reads the next group).
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *tmap, uint32_t bar_cluster,
                                                 int32_t x, int32_t y, int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar_cluster)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *tmap, uint32_t bar, int32_t x, int32_t y,
                                            int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap *tmap, uint32_t src, int32_t x, int32_t y, int32_t z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                     reinterpret_cast<uint64_t>(tmap)),
                 "r"(x), "r"(y), "r"(z), "r"(src)
                 : "memory");
}

// Bounded wait by a whole warp, whose lanes are together when it returns: lane 0 polls, the
// shuffle brings the others.  What follows (tcgen05.ld, stmatrix, barrier.cluster: .aligned)
// needs all of them at once; lanes that polled each for itself would see the phase complete
// at different polls, and the compiler may leave them apart until the branch for a wait that
// gave up joins again, after the role's loop.
__device__ __forceinline__ bool warp_wait_parity(uint32_t bar, uint32_t parity, uint64_t timeout_ns,
                                                 volatile int *abort, int lane) {
    int ok = 1;
    if (lane == 0) ok = wait_parity(bar, parity, timeout_ns, abort);
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// barrier.cluster is .aligned too: bring the warp's lanes together before it.
__device__ __forceinline__ void warp_cluster_sync() {
    __syncwarp();
    cluster_sync();
}

// 16 lanes x 32 fp32 columns as matrix fragments: with l the lane, r[4i], r[4i+1] hold row
// l/4 and columns 8i + 2(l%4), +1; r[4i+2], r[4i+3] the same columns of row l/4 + 8.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// Four 8x8 16-bit matrices between fragments (register j: matrix j, row l/4, columns
// 2(l%4), +1) and shared memory holding their transposes; lane 8j + i gives the address of
// row i (16 bytes) of the transpose of matrix j.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
                 "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
                 : "r"(addr)
                 : "memory");
}

// ------------------------------------------------------------------------- activations
// In fp32 from exp and one division; the fast exponential's error grows with its argument, to
// 2^-18 of the result at y = -20 and 2^-16 at -88, where sigma is 2e-9 and 6e-39.  Outputs here
// are 16-bit (fp16 has 11 bits); the hardware tanh of the NVFP4 epilogue is coarser.
//   sigma(y) = 1 / (1 + exp(-y));  silu = y sigma(y)
//   gelu (tanh form) = y sigma(2u),  u = sqrt(2/pi) (y + 0.044715 y^3)
__device__ __forceinline__ float sigma(float y) { return __fdividef(1.0f, 1.0f + __expf(-y)); }

constexpr float kGelu0 = 0.7978845608028654f, kGelu1 = 0.044715f;

template <int ACT>
__device__ __forceinline__ float act(float y) {
    if constexpr (ACT == kActRelu) return y > 0.0f ? y : (y != y ? y : 0.0f);
    if constexpr (ACT == kActSilu) return y * sigma(y);
    if constexpr (ACT == kActGeluTanh) return y * sigma(2.0f * kGelu0 * fmaf(kGelu1 * y * y, y, y));
    return y;
}

// Derivative of act at z (not SwiGLU, which has two arguments).  Where sigma has rounded to 0
// or 1 the derivative is that: the other term's factor sigma (1 - sigma) is 0, and z or its
// square, which passes fp32 from 5e19 on, would make it NaN.
__device__ __forceinline__ float act_grad(int a, float z) {
    if (a == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    if (a == kActSilu) {
        const float s = sigma(z), d = s * (1.0f - s);
        return d == 0.0f ? s : fmaf(z, d, s);
    }
    if (a == kActGeluTanh) {
        const float s = sigma(2.0f * kGelu0 * fmaf(kGelu1 * z * z, z, z)), d = s * (1.0f - s);
        return d == 0.0f ? s : fmaf(z * d, 2.0f * kGelu0 * fmaf(3.0f * kGelu1 * z, z, 1.0f), s);
    }
    return 1.0f;
}

// ------------------------------------------------------------------------- row groups
// Rows [r0, r1) of group g: offsets clamped to [0, m_total], an end before its start empty.
__device__ __forceinline__ void group_rows(const int *m_offsets, int g, int m_total, int &r0, int &r1) {
    if (!m_offsets) {
        r0 = 0;
        r1 = m_total;
        return;
    }
    r0 = min(max(m_offsets[g], 0), m_total);
    r1 = min(max(m_offsets[g + 1], r0), m_total);
}

// One warp fills r0[g], r1[g] and t0[g] (first tile of group g, t0[G] = all tiles), a group
// of n rows having ceil(n / unit) * per_unit tiles, or per_unit when unit is 0.
__device__ __forceinline__ void build_tables(const int *m_offsets, int G, int m_total, int unit, int per_unit,
                                             int lane, int *r0, int *r1, int *t0) {
    int carry = 0;
    for (int base = 0; base < G; base += 32) {
        const int g = base + lane;
        int a = 0, z = 0, tiles = 0;
        if (g < G) {
            group_rows(m_offsets, g, m_total, a, z);
            tiles = unit ? (z - a + unit - 1) / unit * per_unit : per_unit;
        }
        int s = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        if (g < G) {
            r0[g] = a;
            r1[g] = z;
            t0[g + 1] = carry + s;
        }
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) t0[0] = 0;
}

// ------------------------------------------------------------------------- host side
template <typename T>
constexpr CUtensorMapDataType tma_type() {
    return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// [rows, cols] with a row pitch, as boxes of 64 columns (one swizzle row) by box_rows.
template <typename T>
inline int map_rows(CUtensorMap *m, const void *base, int64_t rows, int cols, int64_t pitch, int box_rows) {
    const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)pitch * 2};
    const uint32_t box[2] = {64, (uint32_t)box_rows};
    return encode_tiled(m, tma_type<T>(), 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The weight [groups, N, K].
template <typename T>
inline int map_weight(CUtensorMap *m, const void *base, int groups, int N, int K, int box_rows) {
    const uint64_t dims[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)groups};
    const uint64_t strides[2] = {(uint64_t)K * 2, (uint64_t)N * (uint64_t)K * 2};
    const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
    return encode_tiled(m, tma_type<T>(), 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The weight's gradient [groups, N, K], written in boxes of 32 rows x 32 columns.
template <typename T>
inline int map_gradient(CUtensorMap *m, const void *base, int groups, int N, int K) {
    const uint64_t dims[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)groups};
    const uint64_t strides[2] = {(uint64_t)K * 2, (uint64_t)N * (uint64_t)K * 2};
    const uint32_t box[3] = {32, 32, 1};
    return encode_tiled(m, tma_type<T>(), 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

// How a product is launched, from its sizes and the GPU's SM count alone.
struct Plan {
    int decode;        // 1: the split-reduction kernel, 0: the persistent CTA-pair kernel
    int bt, wide;      // pair: tokens of a tile part (wgrad: columns of a tile), two parts a tile
    int splits;        // decode: CTAs that share a tile's reduction
    int stages;        // ring slots
    int programmatic;  // launched as a programmatic dependent of the previous kernel
    int64_t tiles;     // pair: tiles, an upper bound for row groups; decode: CTAs
};
// linear.cu.  features: the output's (N, for the input gradient K); red: the reduction (K, for
// the input gradient N; the weight gradient's columns K).
Plan make_plan(int form, int groups, bool ragged, int m_total, int features, int red, int sm_count);

// linear_decode.cu: the forward product (B = X, red = K) or the input gradient (B = dZ, red =
// N) for at most kDecodeTokens token rows in all.
constexpr int kDecodeTokens = 128;
void plan_decode(int form, int groups, int m_total, int features, int red, int sm_count, Plan *plan);
template <typename T, int FORM>
int decode_product(const void *B, int64_t ldb, const void *W, Params p, const Plan &plan, int red, const DeviceInfo &di,
                   cudaStream_t s);

}  // namespace linear
}  // namespace nvfp4
