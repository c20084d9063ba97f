// Activations kept in 8 bits for the backward pass, and the (gated) SiLU that keeps its input so.
//
//   keep      a = max |x| over the finite values of 128 columns of a row;  s = the smallest power of two with a / s <= 448;
//             q = e4m3(x / s).  Both divisions and q s are exact, so that what was kept is restored without a second
//             rounding (bf16 and fp32; fp16 where the value is in its range), and a kernel that computes from q sees the
//             values that any other reader of the checkpoint sees.  Infinities and NaN are kept as NaN and leave the
//             scale of their block alone, so that a gradient computed from them does not look finite.
//   silu_gate h = g sig(g) v          (gated: up = [g | v] or [v | g])      h = g sig(g)     (not gated)
//   backward  dv = dh g sig(g),  dg = dh v sig(g) (1 + g (1 - sig(g))), and h once more: the next layer's weight
//             gradient needs it, and it comes from the same 8 bits instead of 16 kept ones.
//
// Bound by HBM: each value is read and written once.  A lane works on an octet (8 columns), 16 neighbouring lanes hold a
// block of 128 columns, whose largest value is found by four shuffles; a lane has kUnroll octets of different places in
// flight.  sig(g) = 1 / (1 + exp(-g)) in fp32 on the special-function unit (exp to 2 ulp of 2^x, a reciprocal): far below the
// rounding of a 16-bit result; an fp32 result takes expf and a division.
#include "quant.cuh"
#include "tb200_common.cuh"

namespace tb200 {
void count_launch();

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;

// 16-bit results: the fast exponential and reciprocal; fp32: the accurate ones
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    if (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
    return __fdividef(1.0f, 1.0f + __expf(-g));
}

// e4m3 values and scale of the 128 columns that this lane's 16 neighbours hold; all 32 lanes call it
__device__ __forceinline__ uint2 keep(float (&x)[8], float* scale) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float m = fabsf(x[e]);
        const bool finite = m <= 3.402823466e38f;
        if (!finite) x[e] = __int_as_float(0x7FC00000);
        amax = fmaxf(amax, finite ? m : 0.f);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float2 s = exact_pow2_scale(amax);
    *scale = s.x;
    return make_uint2(pack_e4m3x4(x[0] * s.y, x[1] * s.y, x[2] * s.y, x[3] * s.y),
                      pack_e4m3x4(x[4] * s.y, x[5] * s.y, x[6] * s.y, x[7] * s.y));
}

// MODE: 0 keep and restore nothing else (x -> q, scales), 1 ungated, 2 gated; KEEP: write q and scales
template <typename T, int MODE, bool KEEP>
__global__ void __launch_bounds__(kThreads)
gate_kernel(const T* __restrict__ up, T* __restrict__ h, uint2* __restrict__ q, float* __restrict__ scales, uint32_t items, uint32_t octets,
            int32_t gate_at) {
    chain_release();
    chain_wait();
    // items: octets of the activation in all rows; octets: of one row.  gate_at: 0 = the gate is the first half, 1 the second
    const uint32_t stride = gridDim.x * kThreads;
    const uint32_t width = MODE == 2 ? 2 * octets : octets;          // octets of an input row
    // every lane of a warp walks the same number of rounds: the shuffles name all of them
    for (uint32_t base = blockIdx.x * kThreads + threadIdx.x; base - (threadIdx.x & 31) < items; base += kUnroll * stride) {
        Octet<T> rg[kUnroll], rv[kUnroll];
        uint32_t at[kUnroll];
        int64_t in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            at[u] = base + u * stride;
            rg[u].clear();
            rv[u].clear();
            in[u] = 0;
            if (at[u] < items) {
                const uint32_t row = at[u] / octets;
                in[u] = static_cast<int64_t>(row) * width + (at[u] - row * octets);
                rg[u].load(up + (in[u] + (MODE == 2 ? gate_at * octets : 0)) * 8);
                if (MODE == 2) rv[u].load(up + (in[u] + (gate_at ^ 1) * octets) * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float g[8], v[8], o[8];
            rg[u].unpack(g);
            if (MODE == 2) rv[u].unpack(v);
            if (MODE != 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] = g[e] * sigmoid<T>(g[e]);
                    if (MODE == 2) o[e] *= v[e];
                }
            }
            const bool live = at[u] < items;
            if (MODE != 0 && live) Octet<T>::store(h + static_cast<int64_t>(at[u]) * 8, o);
            if (KEEP) {
                float s;
                const int64_t og = in[u] + (MODE == 2 ? gate_at * octets : 0);
                const uint2 wg = keep(g, &s);
                if (live) {
                    q[og] = wg;
                    if ((threadIdx.x & 15) == 0) scales[og >> 4] = s;
                }
                if (MODE == 2) {
                    const int64_t ov = in[u] + (gate_at ^ 1) * octets;
                    const uint2 wv = keep(v, &s);
                    if (live) {
                        q[ov] = wv;
                        if ((threadIdx.x & 15) == 0) scales[ov >> 4] = s;
                    }
                }
            }
        }
    }
}

// MODE: 0 restore (q, scales -> x), 1 backward of the ungated form, 2 of the gated one
template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads)
gate_bwd_kernel(const uint2* __restrict__ q, const float* __restrict__ scales, const T* __restrict__ dh, T* __restrict__ dup, T* __restrict__ h,
                uint32_t items, uint32_t octets, int32_t gate_at) {
    chain_release();
    chain_wait();
    const uint32_t stride = gridDim.x * kThreads;
    const uint32_t width = MODE == 2 ? 2 * octets : octets;
    for (uint32_t base = blockIdx.x * kThreads + threadIdx.x; base < items; base += kUnroll * stride) {
        uint2 qg[kUnroll], qv[kUnroll];
        float sg[kUnroll], sv[kUnroll];
        Octet<T> rd[kUnroll];
        uint32_t at[kUnroll];
        int64_t in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            at[u] = base + u * stride;
            if (at[u] < items) {
                const uint32_t row = at[u] / octets;
                in[u] = static_cast<int64_t>(row) * width + (at[u] - row * octets);
                const int64_t ig = in[u] + (MODE == 2 ? gate_at * octets : 0), iv = in[u] + (gate_at ^ 1) * octets;
                qg[u] = __ldcs(q + ig);
                sg[u] = __ldg(scales + (ig >> 4));
                if (MODE == 2) {
                    qv[u] = __ldcs(q + iv);
                    sv[u] = __ldg(scales + (iv >> 4));
                }
                if (MODE != 0) rd[u].load(dh + static_cast<int64_t>(at[u]) * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (at[u] >= items) continue;
            float g[8], v[8], d[8], o[8], dv[8];
            unpack_e4m3x8(qg[u], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] *= sg[u];
            const int64_t ig = (in[u] + (MODE == 2 ? gate_at * octets : 0)) * 8;
            if (MODE == 0) {
                Octet<T>::store(dup + ig, g);
                continue;
            }
            if (MODE == 2) unpack_e4m3x8(qv[u], v);
            rd[u].unpack(d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float sig = sigmoid<T>(g[e]);
                const float silu = g[e] * sig;
                const float slope = sig * fmaf(g[e], 1.0f - sig, 1.0f);
                if (MODE == 2) {
                    const float val = v[e] * sv[u];
                    o[e] = silu * val;
                    dv[e] = d[e] * silu;
                    d[e] = d[e] * val * slope;
                } else {
                    o[e] = silu;
                    d[e] *= slope;
                }
            }
            Octet<T>::store(dup + ig, d);
            if (MODE == 2) Octet<T>::store(dup + (in[u] + (gate_at ^ 1) * octets) * 8, dv);
            if (h != nullptr) Octet<T>::store(h + static_cast<int64_t>(at[u]) * 8, o);
        }
    }
}

unsigned grid_of(int64_t items) {
    const int64_t ctas = (items + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    const int64_t cap = static_cast<int64_t>(device_info().sm_count) * 16;
    return static_cast<unsigned>(ctas > cap ? cap : ctas);
}

// Launches take at most this many octets of the activation, so that their numbers (and the stride past the last) stay in 32
// bits; more rows go out in several launches
constexpr int64_t kMaxItems = int64_t(1) << 30;

template <typename T, int MODE, bool KEEP>
int run_gate(const void* up, void* h, void* q, float* scales, int64_t rows, int32_t hidden, int gate_at, cudaStream_t st) {
    const int64_t octets = hidden / 8, width = octets * (MODE == 2 ? 2 : 1);
    const int64_t chunk = kMaxItems / octets;
    for (int64_t r = 0; r < rows; r += chunk) {
        const int64_t n = rows - r < chunk ? rows - r : chunk;
        launch_chained(gate_kernel<T, MODE, KEEP>, grid_of(n * octets), kThreads, 0, st, static_cast<const T*>(up) + r * width * 8,
                       h == nullptr ? nullptr : static_cast<T*>(h) + r * hidden, KEEP ? static_cast<uint2*>(q) + r * width : nullptr,
                       KEEP ? scales + r * width / 16 : nullptr, static_cast<uint32_t>(n * octets), static_cast<uint32_t>(octets), gate_at);
        count_launch();
        const int code = launch_status();
        if (code != TB200_OK) return code;
    }
    return TB200_OK;
}

template <typename T, int MODE>
int run_gate_bwd(const void* q, const float* scales, const void* dh, void* dup, void* h, int64_t rows, int32_t hidden, int gate_at,
                 cudaStream_t st) {
    const int64_t octets = hidden / 8, width = octets * (MODE == 2 ? 2 : 1);
    const int64_t chunk = kMaxItems / octets;
    for (int64_t r = 0; r < rows; r += chunk) {
        const int64_t n = rows - r < chunk ? rows - r : chunk;
        launch_chained(gate_bwd_kernel<T, MODE>, grid_of(n * octets), kThreads, 0, st, static_cast<const uint2*>(q) + r * width,
                       scales + r * width / 16, MODE == 0 ? nullptr : static_cast<const T*>(dh) + r * hidden,
                       static_cast<T*>(dup) + r * width * 8, h == nullptr ? nullptr : static_cast<T*>(h) + r * hidden,
                       static_cast<uint32_t>(n * octets), static_cast<uint32_t>(octets), gate_at);
        count_launch();
        const int code = launch_status();
        if (code != TB200_OK) return code;
    }
    return TB200_OK;
}

// 0: served; hidden is the width of one half where the input is gated
int checked(int64_t rows, int32_t hidden, int dtype) {
    if (rows < 0 || hidden < 1) return TB200_ERR_SHAPE;
    if (dtype_size(dtype) == 0) return TB200_ERR_DTYPE;
    if (hidden % 128 != 0) return TB200_ERR_SHAPE;
    return TB200_OK;
}

template <typename T>
int gate_of(const void* up, void* h, void* q, float* scales, int64_t rows, int32_t hidden, int gated, int gate_at, cudaStream_t st) {
    if (q == nullptr)
        return gated ? run_gate<T, 2, false>(up, h, q, scales, rows, hidden, gate_at, st) : run_gate<T, 1, false>(up, h, q, scales, rows, hidden, 0, st);
    return gated ? run_gate<T, 2, true>(up, h, q, scales, rows, hidden, gate_at, st) : run_gate<T, 1, true>(up, h, q, scales, rows, hidden, 0, st);
}

template <typename T>
int gate_bwd_of(const void* q, const float* scales, const void* dh, void* dup, void* h, int64_t rows, int32_t hidden, int gated, int gate_at,
                cudaStream_t st) {
    return gated ? run_gate_bwd<T, 2>(q, scales, dh, dup, h, rows, hidden, gate_at, st) : run_gate_bwd<T, 1>(q, scales, dh, dup, h, rows, hidden, 0, st);
}

}  // namespace
}  // namespace tb200

extern "C" int tb200_keep_fwd(const void* x, void* q, float* scales, int64_t rows, int32_t cols, int dtype, void* stream) {
    using namespace tb200;
    const int code = checked(rows, cols, dtype);
    if (code != TB200_OK || rows == 0) return code;
    if (x == nullptr || q == nullptr || scales == nullptr) return TB200_ERR_NULL;
    if (!aligned16(x) || !aligned16(q) || (reinterpret_cast<uintptr_t>(scales) & 3) != 0) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case TB200_F32: return run_gate<float, 0, true>(x, nullptr, q, scales, rows, cols, 0, st);
        case TB200_F16: return run_gate<__half, 0, true>(x, nullptr, q, scales, rows, cols, 0, st);
        default: return run_gate<__nv_bfloat16, 0, true>(x, nullptr, q, scales, rows, cols, 0, st);
    }
}

extern "C" int tb200_keep_restore(const void* q, const float* scales, void* x, int64_t rows, int32_t cols, int dtype, void* stream) {
    using namespace tb200;
    const int code = checked(rows, cols, dtype);
    if (code != TB200_OK || rows == 0) return code;
    if (x == nullptr || q == nullptr || scales == nullptr) return TB200_ERR_NULL;
    if (!aligned16(x) || !aligned16(q) || (reinterpret_cast<uintptr_t>(scales) & 3) != 0) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case TB200_F32: return run_gate_bwd<float, 0>(q, scales, nullptr, x, nullptr, rows, cols, 0, st);
        case TB200_F16: return run_gate_bwd<__half, 0>(q, scales, nullptr, x, nullptr, rows, cols, 0, st);
        default: return run_gate_bwd<__nv_bfloat16, 0>(q, scales, nullptr, x, nullptr, rows, cols, 0, st);
    }
}

extern "C" int tb200_silu_gate_fwd(const void* up, void* h, void* q, float* scales, int64_t rows, int32_t hidden, int32_t gated,
                                   int32_t gate_first, int dtype, void* stream) {
    using namespace tb200;
    const int code = checked(rows, hidden, dtype);
    if (code != TB200_OK || rows == 0) return code;
    if (up == nullptr || h == nullptr || (q == nullptr) != (scales == nullptr)) return TB200_ERR_NULL;
    if (!aligned16(up) || !aligned16(h) || !aligned16(q) || (reinterpret_cast<uintptr_t>(scales) & 3) != 0) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int at = gate_first ? 0 : 1;
    switch (dtype) {
        case TB200_F32: return gate_of<float>(up, h, q, scales, rows, hidden, gated, at, st);
        case TB200_F16: return gate_of<__half>(up, h, q, scales, rows, hidden, gated, at, st);
        default: return gate_of<__nv_bfloat16>(up, h, q, scales, rows, hidden, gated, at, st);
    }
}

extern "C" int tb200_silu_gate_bwd(const void* q, const float* scales, const void* dh, void* dup, void* h, int64_t rows, int32_t hidden,
                                   int32_t gated, int32_t gate_first, int dtype, void* stream) {
    using namespace tb200;
    const int code = checked(rows, hidden, dtype);
    if (code != TB200_OK || rows == 0) return code;
    if (q == nullptr || scales == nullptr || dh == nullptr || dup == nullptr) return TB200_ERR_NULL;
    if (!aligned16(q) || !aligned16(dh) || !aligned16(dup) || !aligned16(h) || (reinterpret_cast<uintptr_t>(scales) & 3) != 0) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int at = gate_first ? 0 : 1;
    switch (dtype) {
        case TB200_F32: return gate_bwd_of<float>(q, scales, dh, dup, h, rows, hidden, gated, at, st);
        case TB200_F16: return gate_bwd_of<__half>(q, scales, dh, dup, h, rows, hidden, gated, at, st);
        default: return gate_bwd_of<__nv_bfloat16>(q, scales, dh, dup, h, rows, hidden, gated, at, st);
    }
}
