// moe_products.cuh — moe_layer for many rows an expert: two grouped products and a sum.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "common.cuh"

namespace nvfp4 {
namespace moe_products {

constexpr int kMaxTokens = 64;  // an expert's rows are the MMA's N
constexpr int kMaxParts = 5;    // that a W2 tile's reduction is cut into
constexpr int kTile = 128;      // W2 rows, columns of the output

struct Args {
    const void *x, *w13, *w2, *residual;
    void *y;
    int64_t ldx;
    const float *weights;            // [T, k], by the router
    const int *experts, *rows;       // [T, k]
    const int *m_offsets;            // [E + 1]
    void *x_rows, *h;                // workspace: [T k, K] and [T k, F] 16-bit
    float *part;                     // workspace: [kMaxParts][T k, K]
    uint8_t *parts;                  // workspace: [E][tiles of 128 columns]
    int T, E, k, K, F, dtype;
};

int run(const Args &a, const DeviceInfo &di, cudaStream_t stream);

}  // namespace moe_products
}  // namespace nvfp4
