// What the kernels of layers grouped by expert share: their arguments, the rows of the experts, tensor maps.
#pragma once
#include "tb200_common.cuh"
#include "tb200_tmap.cuh"
#include "tb200_ptx.cuh"

#include <type_traits>

namespace tb200 {

constexpr int kMaxExperts = 2048;

struct RaggedArgs {
    const int32_t* offsets;     // [experts + 1]
    const float* bias;          // [experts, cols] or NULL (rows)
    const void* residual;       // [T, cols] or NULL (rows)
    void* out;                  // [T, cols], or [experts, n, k] (weights)
    float* db;                  // [experts, n] or NULL (weights)
    float* partial;             // [pairs][2] partial tiles, NULL: tiles are never shared (weights)
    float* db_partial;          // [pairs][2][256] sums of the rows of those pieces
    int4* pieces;               // [pairs][2] what they are part of: expert (-1: nothing), first row and column of the tile, last piece?
    int32_t* status;
    int32_t experts, stages;
    int64_t T;
    int32_t cols;               // of a result row
    int32_t depth;              // contracted length (rows, row grads)
    int32_t n;                  // rows of a weight gradient
    int32_t silu;
    int32_t clear;              // rows of no expert are set to zero
};

// Where every expert's rows begin, by one warp; the offsets come from the kernel in front.  An offset outside [0, T] is moved to
// the nearer end and one that lies before an earlier one counts as that one, so that no two experts share a row.
__device__ __forceinline__ void first_rows(const RaggedArgs& g, int32_t* begin, int lane) {
    constexpr int kAhead = 4;      // loads in flight
    int32_t top = 0;
    for (int base = 0; base <= g.experts; base += 32 * kAhead) {
        int32_t v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = base + 32 * k + lane <= g.experts ? __ldcg(g.offsets + base + 32 * k + lane) : 0;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int at = base + 32 * k;
            if (at > g.experts) break;
            int32_t m = v[k] < 0 ? 0 : (v[k] > g.T ? static_cast<int32_t>(g.T) : v[k]);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t u = __shfl_up_sync(0xffffffffu, m, o);
                if (lane >= o) m = max(m, u);
            }
            m = max(m, top);
            if (at + lane <= g.experts) begin[at + lane] = m;
            top = __shfl_sync(0xffffffffu, m, 31);
        }
    }
    __syncwarp();
}
// pre[i] = sum of units(0 .. i - 1), by one warp
template <typename F>
__device__ __forceinline__ void prefix(int32_t* pre, int n, int lane, F units) {
    int32_t sum = 0;
    for (int base = 0; base < n; base += 32) {
        int32_t v = base + lane < n ? units(base + lane) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (base + lane < n) pre[base + lane + 1] = sum + v;
        sum += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) pre[0] = 0;
    __syncwarp();
}
// the last i with pre[i] <= unit: the expert whose units hold `unit`
__device__ __forceinline__ int expert_of(const int32_t* pre, int experts, int64_t unit) {
    int lo = 0, hi = experts;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}
// silu(x) = x / (1 + exp(-x))
__device__ __forceinline__ float silu(float x) { return x * __fdividef(1.0f, 1.0f + __expf(-x)); }

// a matrix or a stack of matrices of 16-bit values, boxes of box_rows x 128 bytes
inline bool make_map(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t stack, uint32_t box_rows) {
    const auto fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {2 * cols, rows, stack};
    const cuuint64_t strides[2] = {2 * cols, 2 * cols * rows};
    const cuuint32_t box[3] = {128, box_rows, 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, stack == 0 ? 2 : 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The same matrices as chunks of 64 columns, for boxes of 64 rows x two chunks, which land chunk after chunk: the 128 columns of an
// MN-major operand in one copy.  Whole chunks only: the last piece of a row would reach into the next.
inline bool make_chunk_map(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t stack) {
    const auto fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[4] = {128, rows, cols / 64, stack};
    const cuuint64_t strides[3] = {2 * cols, 128, 2 * cols * rows};
    const cuuint32_t box[4] = {128, 64, 2, 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, stack == 0 ? 3 : 4, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tb200
