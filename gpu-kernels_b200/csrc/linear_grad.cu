// linear_grad.cu — gradient of the linear layers' epilogue: dZ = dY * act'(Z), and the bias
// gradient (column sums of dZ by row group), in one pass over dY and Z.
//
// dZ is rounded to the 16-bit type here, and the two products that follow take it so: their
// tensor instructions read 16-bit operands, and a dZ of 32 bits as two parts would double both
// products' instructions and the bytes of dZ.  It costs one more rounding than a 32-bit dZ
// would: the norm of dX's and dW's error grows from 0.0017 to 0.0023 of theirs in bf16.  In
// fp16 a dZ past 65504 becomes an infinity (for SwiGLU the factor is not bounded), as any fp16
// gradient does, for the loss scale to catch.  The bias gradient sums the unrounded dZ.
//
// Bound by memory: dY and Z are read once and dZ written once, 16 bytes a thread.  The
// column sums are kept in fp32: each CTA sums 64 rows of one group, and a second kernel adds
// the CTAs' sums in row order, so the result has the same bits on every call.  16387 rows of
// 2048 columns with SwiGLU and 64 groups: 33 us (5.1 TB/s), and 6.5 us for the groups' sums; 4096 x 14336
// with gelu 75 us (4.7 TB/s) and 11 us.
#include <algorithm>
#include <climits>

#include "linear.cuh"

namespace nvfp4 {
namespace linear {

constexpr int kGradRows = 64;      // rows of one CTA
constexpr int kGradLanes = 32;     // 8-column units of one CTA
constexpr int kGradRowLanes = 8;
constexpr int kGradThreads = kGradLanes * kGradRowLanes;

struct GradParams {
    const void *dy, *z;
    void *dz;        // may be null: only the column sums are wanted
    float *partial;  // [chunks][N], null: no bias gradient
    const int *m_offsets;
    int groups, m_total, N;
    int act;
};

// Tables of 64-row chunks by group, in shared memory.
struct ChunkTables {
    int r0[kMaxGroups + 1], r1[kMaxGroups + 1], c0[kMaxGroups + 1];
};

template <typename T>
__global__ void __launch_bounds__(kGradThreads) activation_backward_kernel(const GradParams p) {
    __shared__ ChunkTables tab;
    __shared__ float sums[kGradRowLanes][kGradLanes][17];  // 17: no bank conflicts between units
    if (threadIdx.x < 32) build_tables(p.m_offsets, p.groups, p.m_total, kGradRows, 1, threadIdx.x, tab.r0, tab.r1, tab.c0);
    __syncthreads();
    const int col_blocks = ((p.act == kActSwiglu ? p.N / 2 : p.N) / 8 + kGradLanes - 1) / kGradLanes;
    const int chunk = blockIdx.x / col_blocks, col_block = blockIdx.x - chunk * col_blocks;
    if (chunk >= tab.c0[p.groups]) return;
    int g = 0, hi = p.groups - 1;
    while (g < hi) {
        const int mid = (g + hi + 1) >> 1;
        if (tab.c0[mid] <= chunk) g = mid; else hi = mid - 1;
    }
    const int row0 = tab.r0[g] + (chunk - tab.c0[g]) * kGradRows, row1 = min(row0 + kGradRows, tab.r1[g]);
    const bool glu = p.act == kActSwiglu;
    const int No = glu ? p.N / 2 : p.N;
    const int unit = col_block * kGradLanes + (threadIdx.x & 31), rl = threadIdx.x >> 5;
    const int col = unit * 8;  // column of dY
    // columns of Z: the same, or the gate's (and 16 further the up's) for SwiGLU
    const int zc = glu ? (col >> 4) * 32 + (col & 15) : col;
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; i++) sum[i] = 0.0f;
    if (col < No)
#pragma unroll 2
        for (int r = row0 + rl; r < row1; r += kGradRowLanes) {
            const uint4 raw = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.dy) + (int64_t)r * No + col);
            float d[8];
            if (glu) {
                const T *zp = static_cast<const T *>(p.z) + (int64_t)r * p.N + zc;
                const uint4 zg = *reinterpret_cast<const uint4 *>(zp);
                const uint4 zu = *reinterpret_cast<const uint4 *>(zp + 16);
                float gate[8], up[8], dg[8], du[8];
                unpack8<T>(raw, d);
                unpack8<T>(zg, gate);
                unpack8<T>(zu, up);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float s = sigma(gate[i]), h = gate[i] * s;
                    dg[i] = d[i] * up[i] * fmaf(h, 1.0f - s, s);
                    du[i] = d[i] * h;
                    sum[i] += dg[i];
                    sum[8 + i] += du[i];
                }
                T *out = static_cast<T *>(p.dz) + (int64_t)r * p.N + zc;
                *reinterpret_cast<uint4 *>(out) = pack8<T>(dg);
                *reinterpret_cast<uint4 *>(out + 16) = pack8<T>(du);
            } else {
                unpack8<T>(raw, d);
                if (p.act != kActNone) {
                    const uint4 zr = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.z) + (int64_t)r * p.N + zc);
                    float z[8];
                    unpack8<T>(zr, z);
#pragma unroll
                    for (int i = 0; i < 8; i++) d[i] *= act_grad(p.act, z[i]);
                    *reinterpret_cast<uint4 *>(static_cast<T *>(p.dz) + (int64_t)r * p.N + zc) = pack8<T>(d);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) sum[i] += d[i];
            }
        }
    if (!p.partial) return;
#pragma unroll
    for (int i = 0; i < 16; i++) sums[rl][threadIdx.x & 31][i] = sum[i];
    __syncthreads();
    // one thread a column of the CTA's units: the eight row lanes in order
    const int per_unit = glu ? 16 : 8;
    for (int i = threadIdx.x; i < kGradLanes * per_unit; i += kGradThreads) {
        const int u = i / per_unit, e = i % per_unit, c = (col_block * kGradLanes + u) * 8;
        if (c >= No) continue;
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < kGradRowLanes; q++) s += sums[q][u][e];
        const int at = glu ? (c >> 4) * 32 + (c & 15) + (e >= 8 ? 8 + e : e) : c + e;
        p.partial[(int64_t)chunk * p.N + at] = s;
    }
}

// chunks: of the workspace.  Offsets that decrease, which the host cannot see, may count
// more; none is read past it.
template <typename T>
__global__ void __launch_bounds__(256) bias_sum_kernel(const float *partial, T *db, const int *m_offsets, int chunks,
                                                       int m_total, int N) {
    __shared__ int before;  // first chunk of this group
    const int g = blockIdx.y;
    if (threadIdx.x < 32) {
        int c = 0;
        for (int h = threadIdx.x; h < g; h += 32) {
            int a, z;
            group_rows(m_offsets, h, m_total, a, z);
            c += (z - a + kGradRows - 1) / kGradRows;
        }
        c = __reduce_add_sync(0xffffffffu, c);
        if (threadIdx.x == 0) before = c;
    }
    __syncthreads();
    int a, z;
    group_rows(m_offsets, g, m_total, a, z);
    const int n = max(0, min((z - a + kGradRows - 1) / kGradRows, chunks - before));
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    const float *src = partial + (int64_t)before * N + c;
    float s = 0.0f;
#pragma unroll 8
    for (int i = 0; i < n; i++) s += src[(int64_t)i * N];
    db[(int64_t)g * N + c] = Type16<T>::round(s);
}

static int64_t grad_chunks(int groups, int M) { return ((int64_t)M + kGradRows - 1) / kGradRows + (groups > 1 ? groups : 0); }

// CTAs: chunks x blocks of columns, the columns fastest.
static int64_t grad_blocks(int groups, int M, int N, int act) {
    const int No = act == kActSwiglu ? N / 2 : N;
    return grad_chunks(groups, M) * ((No / 8 + kGradLanes - 1) / kGradLanes);
}

template <typename Kernel, typename... Args>
static int launch(Kernel kern, dim3 grid, int threads, cudaStream_t stream, Args... args) {
    kern<<<grid, threads, 0, stream>>>(args...);
    count_launch();
    return cuda_status(cudaGetLastError());
}

template <typename T>
static int activation_backward(const GradParams &p, T *db, cudaStream_t s) {
    const dim3 grid((unsigned)grad_blocks(p.groups, p.m_total, p.N, p.act));
    int st = launch(activation_backward_kernel<T>, grid, kGradThreads, s, p);
    if (st || !db) return st;
    return launch(bias_sum_kernel<T>, dim3((p.N + 255) / 256, p.groups), 256, s, (const float *)p.partial, db,
                  p.m_offsets, (int)grad_chunks(p.groups, p.m_total), p.m_total, p.N);
}

}  // namespace linear
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

size_t nvfp4_activation_backward_workspace_size(int groups, int M, int N) {
    if (groups < 1 || groups > linear::kMaxGroups || M < 0 || N < 8 || N % 8) return 0;
    return (size_t)std::max<int64_t>(1, linear::grad_chunks(groups, M)) * N * sizeof(float);
}

int nvfp4_activation_backward(const void *dY, const void *Z, void *dZ, void *dbias, const int32_t *m_offsets,
                              int groups, int M, int N, int activation, int dtype, void *workspace,
                              size_t workspace_bytes, void *stream) {
    if (dtype != NVFP4_BF16 && dtype != NVFP4_F16) return NVFP4_ERR_INVALID;
    if (activation < NVFP4_ACT_NONE || activation > NVFP4_ACT_SWIGLU) return NVFP4_ERR_INVALID;
    if (groups < 1 || (groups > 1 && !m_offsets)) return NVFP4_ERR_INVALID;
    if (groups > linear::kMaxGroups || M < 0 || N < 8 || N % 8 || (activation == NVFP4_ACT_SWIGLU && N % 32))
        return NVFP4_ERR_SHAPE;
    if (M > linear::kMaxExtent || N > linear::kMaxExtent) return NVFP4_ERR_SHAPE;
    if (linear::grad_blocks(groups, M, N, activation) > INT_MAX) return NVFP4_ERR_SHAPE;
    const bool act = activation != NVFP4_ACT_NONE;
    if (M && (!dY || (act && (!Z || !dZ)))) return NVFP4_ERR_INVALID;
    if (!act && !dbias) return NVFP4_OK;  // dZ is dY
    if (!aligned16(dY) || !aligned16(Z) || !aligned16(dZ) || (reinterpret_cast<uintptr_t>(dbias) & 1u) ||
        (reinterpret_cast<uintptr_t>(m_offsets) & 3u) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
        return NVFP4_ERR_ALIGN;
    if (dbias && (!workspace || workspace_bytes < nvfp4_activation_backward_workspace_size(groups, M, N)))
        return NVFP4_ERR_WORKSPACE;
    DeviceInfo di;
    int st = device_info(&di);
    if (st) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M == 0)
        return dbias ? cuda_status(cudaMemsetAsync(dbias, 0, (size_t)groups * N * 2, s)) : NVFP4_OK;
    linear::GradParams p = {};
    p.dy = dY;
    p.z = Z;
    p.dz = act ? dZ : nullptr;
    p.partial = dbias ? static_cast<float *>(workspace) : nullptr;
    p.m_offsets = m_offsets;
    p.groups = groups;
    p.m_total = M;
    p.N = N;
    p.act = activation;
    return dtype == NVFP4_BF16
               ? linear::activation_backward<__nv_bfloat16>(p, static_cast<__nv_bfloat16 *>(dbias), s)
               : linear::activation_backward<__half>(p, static_cast<__half *>(dbias), s);
}

}  // extern "C"
