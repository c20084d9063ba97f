// Activations kept in 8 bits for the backward pass, and the (gated) SiLU that keeps its input so.
//
//   keep      a = max |x| over the finite values of 128 columns of a row;  s = the smallest power of two with a / s <= 448;
//             q = e4m3(x / s).  Both divisions and q s are exact, so that what was kept is restored without a second
//             rounding (bf16 and fp32; fp16 where the value is in its range), and a kernel that computes from q sees the
//             values that any other reader of the checkpoint sees.  Infinities and NaN are kept as NaN and leave the
//             scale of their block alone, so that a gradient computed from them does not look finite.  Finite values stay
//             finite: those from 31 / 32 of the power of two behind their type's range on are kept as that power of two, and a
//             reader whose type does not hold a value takes its largest number.
//   silu_gate h = g sig(g) v          (gated: up = [g | v] or [v | g])      h = g sig(g)     (not gated)
//   backward  dv = dh g sig(g),  dg = dh v sig(g) (1 + g (1 - sig(g))), and h once more: the next layer's weight
//             gradient needs it, and it comes from the same 8 bits instead of 16 kept ones (its type's largest number where
//             the kept values' rounding took it behind that).  The same from the input itself, for a gradient that 8 bits
//             do not round.
//
// Bound by HBM: each value is read and written once.  A lane works on an octet (8 columns), 16 neighbouring lanes hold a
// block of 128 columns, whose largest value is found by four shuffles; a lane has kUnroll octets of different places in
// flight.  Instructions are what competes with the bytes: maxima of bits, packed arithmetic and places without divisions took the
// gated forward pass of 32768 x 2048 bf16 (541 MB) from 103 to 93 us; its backward pass (675 MB) takes 105.  sig(g) =
// 1 / (1 + exp(-g)) in fp32 on the special-function unit (__expf, a reciprocal to 1 ulp): far below the rounding of a 16-bit
// result; an fp32 result takes expf and a division.
#include <type_traits>

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
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-g)));
    return r;
}

// Finite numbers that a type does not hold become its largest one, two packed values at a time behind their rounding (infinity is what
// they round to there); NaN stays NaN.  The sign is the value's, the limit being positive.
template <typename T>
__device__ __forceinline__ uint32_t held(uint32_t x) {
    uint32_t y;
    if (std::is_same<T, __half>::value) asm("min.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x7BFF7BFFu));
    else if (sizeof(T) == 2) asm("min.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x7F7F7F7Fu));
    else asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x7F7FFFFFu));
    return y;
}
template <typename T>
__device__ __forceinline__ void store_held(T* p, const float2 (&f)[4]) {
    constexpr int N = Vec16<T>::N / 2;
#pragma unroll
    for (int i = 0; i < Octet<T>::P; ++i) {
        float2 g[N];
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = f[i * N + e];
        const uint4 w = Vec16<T>::pack2(g);
        *(reinterpret_cast<uint4*>(p) + i) = make_uint4(held<T>(w.x), held<T>(w.y), held<T>(w.z), held<T>(w.w));
    }
}

// The values that eight e4m3 bytes stand for.  From s = 2^120 on they may be infinite where the bytes are not: see finite.
__device__ __forceinline__ void kept_values(uint2 q, float s, float2 (&x)[4]) {
    unpack_e4m3x8(q, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __fmul2_rn(x[e], make_float2(s, s));
}
__device__ __forceinline__ bool huge_scale(float s) { return s > 0x1p119f; }
__device__ __forceinline__ void finite(float2 (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        x[e] = make_float2(__uint_as_float(held<float>(__float_as_uint(x[e].x))), __uint_as_float(held<float>(__float_as_uint(x[e].y))));
}

// ---- largest value of a block.  |x| of every type orders as its bits do, infinity and NaN on top, so the maximum is taken of
// integers: two 16-bit values at a time, and those of the gate's and the value's block in the halves of one word, which one chain
// of shuffles reduces.
template <typename T>
struct Bits {      // 16-bit types: (maximum, 0) as a word
    static constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    static __device__ uint32_t max_of(const Octet<T>& o) {
        const uint4 v = o.v[0];
        const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
        return max(m & 0xFFFFu, m >> 16);
    }
    static __device__ float value(uint32_t bits) {
        const uint16_t b = static_cast<uint16_t>(bits);
        return to_float<T>(*reinterpret_cast<const T*>(&b));
    }
};
template <>
struct Bits<float> {
    static constexpr uint32_t kInf = 0x7F800000u;
    static __device__ uint32_t max_of(const Octet<float>& o) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            m = max(m, max(max(o.v[i].x & 0x7FFFFFFFu, o.v[i].y & 0x7FFFFFFFu), max(o.v[i].z & 0x7FFFFFFFu, o.v[i].w & 0x7FFFFFFFu)));
        return m;
    }
    static __device__ float value(uint32_t bits) { return __uint_as_float(bits); }
};

// the blocks' largest bits, of gate and value, among the 16 neighbours; all 32 lanes call it
template <typename T, bool TWO>
__device__ __forceinline__ uint2 block_max(const Octet<T>& g, const Octet<T>& v) {
    uint32_t a = Bits<T>::max_of(g), b = TWO ? Bits<T>::max_of(v) : 0u;
    if constexpr (sizeof(T) == 2) {
        a |= b << 16;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, o));
        return make_uint2(a & 0xFFFFu, a >> 16);
    } else {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
            if (TWO) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
        }
        return make_uint2(a, b);
    }
}

// Infinity or NaN in the block: NaN in their place, and the largest of the others.  Rare; the lanes of a block come here together.
__device__ __forceinline__ float finite_max(float2 (&x)[4]) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (!(fabsf(x[e].x) <= 3.402823466e38f)) x[e].x = __int_as_float(0x7FC00000);
        if (!(fabsf(x[e].y) <= 3.402823466e38f)) x[e].y = __int_as_float(0x7FC00000);
        m = fmaxf(m, fmaxf(fabsf(x[e].x), fabsf(x[e].y)));
    }
    const uint32_t mask = 0xFFFFu << (threadIdx.x & 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, o));
    return m;
}

// e4m3 values and scale of a block whose largest bits are `top`
template <typename T>
__device__ __forceinline__ uint2 keep(float2 (&x)[4], uint32_t top, float* scale) {
    const float amax = top >= Bits<T>::kInf ? finite_max(x) : Bits<T>::value(top);
    const float2 s = exact_pow2_scale(amax), inv = make_float2(s.y, s.y);
    *scale = s.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __fmul2_rn(x[e], inv);
    return make_uint2(pack_e4m3x4(x[0].x, x[0].y, x[1].x, x[1].y), pack_e4m3x4(x[2].x, x[2].y, x[3].x, x[3].y));
}

// Row and octet of a flat item, and of the one a stride further without another division
struct Place {
    uint32_t row, col;
    __device__ Place(uint32_t item, uint32_t octets) : row(item / octets), col(item - row * octets) {}
    __device__ void advance(const Place& by, uint32_t octets) {
        row += by.row;
        col += by.col;
        if (col >= octets) {
            col -= octets;
            ++row;
        }
    }
};

// MODE: 0 keep and nothing else (x -> q, scales), 1 ungated, 2 gated; KEEP: write q and scales
template <typename T, int MODE, bool KEEP>
__global__ void __launch_bounds__(kThreads)
gate_kernel(const T* __restrict__ up, T* __restrict__ h, uint2* __restrict__ q, float* __restrict__ scales, uint32_t items, uint32_t octets,
            int32_t gate_at) {
    chain_release();
    chain_wait();
    // items: octets of the activation in all rows; octets: of one row.  gate_at: 0 = the gate is the first half, 1 the second
    const uint32_t stride = gridDim.x * kThreads;
    const uint32_t width = MODE == 2 ? 2 * octets : octets;          // octets of an input row
    const uint32_t to_gate = MODE == 2 ? gate_at * octets : 0, to_value = (gate_at ^ 1) * octets;
    const Place by(stride, octets);
    Place place(blockIdx.x * kThreads + threadIdx.x, octets);
    // every lane of a warp walks the same number of rounds: the shuffles name all of them
    for (uint32_t base = blockIdx.x * kThreads + threadIdx.x; base - (threadIdx.x & 31) < items; base += kUnroll * stride) {
        Octet<T> rg[kUnroll], rv[kUnroll];
        int64_t in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            rg[u].clear();
            rv[u].clear();
            in[u] = static_cast<int64_t>(place.row) * width + place.col;
            if (base + u * stride < items) {
                rg[u].load(up + (in[u] + to_gate) * 8);
                if (MODE == 2) rv[u].load(up + (in[u] + to_value) * 8);
            }
            place.advance(by, octets);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const bool live = base + u * stride < items;
            float2 g[4], v[4];
            rg[u].unpack2(g);
            if (MODE == 2) rv[u].unpack2(v);
            if (MODE != 0) {
                float2 o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] = __fmul2_rn(g[e], make_float2(sigmoid<T>(g[e].x), sigmoid<T>(g[e].y)));
                    if (MODE == 2) o[e] = __fmul2_rn(o[e], v[e]);
                }
                if (live) Octet<T>::store2(h + static_cast<int64_t>(base + u * stride) * 8, o);
            }
            if (KEEP) {
                float s;
                const uint2 top = block_max<T, MODE == 2>(rg[u], rv[u]);
                const int64_t og = in[u] + to_gate;
                const uint2 wg = keep<T>(g, top.x, &s);
                if (live) {
                    q[og] = wg;
                    if ((threadIdx.x & 15) == 0) scales[og >> 4] = s;
                }
                if (MODE == 2) {
                    const int64_t ov = in[u] + to_value;
                    const uint2 wv = keep<T>(v, top.y, &s);
                    if (live) {
                        q[ov] = wv;
                        if ((threadIdx.x & 15) == 0) scales[ov >> 4] = s;
                    }
                }
            }
        }
    }
}

// What the backward pass computes from: eight kept values with their scale, or eight of the input itself (T)
template <typename T, bool KEPT>
struct Source {
    uint2 q;
    float s;
    __device__ void load(const void* from, const float* scales, int64_t at) {
        q = __ldcs(static_cast<const uint2*>(from) + at);
        s = __ldg(scales + (at >> 4));
    }
    __device__ void values(float2 (&x)[4]) const { kept_values(q, s, x); }
};
template <typename T>
struct Source<T, false> {
    Octet<T> v;
    static constexpr float s = 1.0f;
    __device__ void load(const void* from, const float*, int64_t at) { v.load(static_cast<const T*>(from) + at * 8); }
    __device__ void values(float2 (&x)[4]) const { v.unpack2(x); }
};

// MODE: 0 restore (q, scales -> x), 1 backward of the ungated form, 2 of the gated one.  KEPT: `from` holds e4m3 values, else T.  16-bit types: four CTAs an SM (left alone the
// gated form takes 66 registers, three CTAs: 32768 x 2048 119 us a call instead of 109)
template <typename T, int MODE, bool KEPT>
__global__ void __launch_bounds__(kThreads, MODE == 2 && sizeof(T) == 2 ? 4 : 0)
gate_bwd_kernel(const void* __restrict__ from, const float* __restrict__ scales, const T* __restrict__ dh, T* __restrict__ dup, T* __restrict__ h,
                uint32_t items, uint32_t octets, int32_t gate_at) {
    chain_release();
    chain_wait();
    const uint32_t stride = gridDim.x * kThreads;
    const uint32_t width = MODE == 2 ? 2 * octets : octets;
    const uint32_t to_gate = MODE == 2 ? gate_at * octets : 0, to_value = (gate_at ^ 1) * octets;
    const Place by(stride, octets);
    Place place(blockIdx.x * kThreads + threadIdx.x, octets);
    for (uint32_t base = blockIdx.x * kThreads + threadIdx.x; base < items; base += kUnroll * stride) {
        Source<T, KEPT> sg[kUnroll], sv[kUnroll];
        Octet<T> rd[kUnroll];
        int64_t in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            in[u] = static_cast<int64_t>(place.row) * width + place.col;
            if (base + u * stride < items) {
                sg[u].load(from, scales, in[u] + to_gate);
                if (MODE == 2) sv[u].load(from, scales, in[u] + to_value);
                if (MODE != 0) rd[u].load(dh + static_cast<int64_t>(base + u * stride) * 8);
            }
            place.advance(by, octets);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + u * stride >= items) continue;
            float2 g[4], v[4], d[4], o[4];
            sg[u].values(g);
            const int64_t ig = (in[u] + to_gate) * 8;
            if (MODE == 0) {
                store_held(dup + ig, g);
                continue;
            }
            if (MODE == 2) sv[u].values(v);
            if (KEPT && huge_scale(MODE == 2 ? fmaxf(sg[u].s, sv[u].s) : sg[u].s)) {      // a branch for both: one for each takes 1 % more
                finite(g);
                if (MODE == 2) finite(v);
            }
            rd[u].unpack2(d);
            const float2 one = make_float2(1.f, 1.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 sig = make_float2(sigmoid<T>(g[e].x), sigmoid<T>(g[e].y));
                const float2 silu = __fmul2_rn(g[e], sig);
                // sig (1 + g (1 - sig)) = sig + silu (1 - sig)
                const float2 slope = __ffma2_rn(silu, __fadd2_rn(one, make_float2(-sig.x, -sig.y)), sig);
                if (MODE == 2) {
                    o[e] = __fmul2_rn(silu, v[e]);
                    v[e] = __fmul2_rn(d[e], v[e]);
                    g[e] = __fmul2_rn(d[e], silu);
                    d[e] = __fmul2_rn(v[e], slope);
                } else {
                    o[e] = silu;
                    d[e] = __fmul2_rn(d[e], slope);
                }
            }
            Octet<T>::store2(dup + ig, d);
            if (MODE == 2) Octet<T>::store2(dup + (in[u] + to_value) * 8, g);
            if (h != nullptr) {      // from the input itself it is the forward pass's, which held nothing
                T* at = h + static_cast<int64_t>(base + u * stride) * 8;
                if (KEPT) store_held(at, o);
                else Octet<T>::store2(at, o);
            }
        }
    }
}

// CTAs an SM at most: forward 16 (8: 93.4, 16: 92.7, 64: 96.1 us at 32768 x 2048, gated), backward 64 (8: 118.6, 16: 112.3, 64: 105.5)
unsigned grid_of(int64_t items, int per_sm) {
    const int64_t ctas = (items + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    const int64_t cap = static_cast<int64_t>(device_info().sm_count) * per_sm;
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
        launch_chained(gate_kernel<T, MODE, KEEP>, grid_of(n * octets, 16), kThreads, 0, st, static_cast<const T*>(up) + r * width * 8,
                       h == nullptr ? nullptr : static_cast<T*>(h) + r * hidden, KEEP ? static_cast<uint2*>(q) + r * width : nullptr,
                       KEEP ? scales + r * width / 16 : nullptr, static_cast<uint32_t>(n * octets), static_cast<uint32_t>(octets), gate_at);
        count_launch();
        const int code = launch_status();
        if (code != TB200_OK) return code;
    }
    return TB200_OK;
}

template <typename T, int MODE, bool KEPT>
int run_gate_bwd(const void* from, const float* scales, const void* dh, void* dup, void* h, int64_t rows, int32_t hidden, int gate_at,
                 cudaStream_t st) {
    const int64_t octets = hidden / 8, width = octets * (MODE == 2 ? 2 : 1);
    const int64_t chunk = kMaxItems / octets;
    for (int64_t r = 0; r < rows; r += chunk) {
        const int64_t n = rows - r < chunk ? rows - r : chunk;
        launch_chained(gate_bwd_kernel<T, MODE, KEPT>, grid_of(n * octets, 64), kThreads, 0, st,
                       static_cast<const void*>(static_cast<const uint8_t*>(from) + r * width * 8 * (KEPT ? 1 : sizeof(T))),
                       KEPT ? scales + r * width / 16 : nullptr, MODE == 0 ? nullptr : static_cast<const T*>(dh) + r * hidden,
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
    if (scales == nullptr)
        return gated ? run_gate_bwd<T, 2, false>(q, scales, dh, dup, h, rows, hidden, gate_at, st)
                     : run_gate_bwd<T, 1, false>(q, scales, dh, dup, h, rows, hidden, 0, st);
    return gated ? run_gate_bwd<T, 2, true>(q, scales, dh, dup, h, rows, hidden, gate_at, st) : run_gate_bwd<T, 1, true>(q, scales, dh, dup, h, rows, hidden, 0, st);
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
        case TB200_F32: return run_gate_bwd<float, 0, true>(q, scales, nullptr, x, nullptr, rows, cols, 0, st);
        case TB200_F16: return run_gate_bwd<__half, 0, true>(q, scales, nullptr, x, nullptr, rows, cols, 0, st);
        default: return run_gate_bwd<__nv_bfloat16, 0, true>(q, scales, nullptr, x, nullptr, rows, cols, 0, st);
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
    if (q == nullptr || dh == nullptr || dup == nullptr) return TB200_ERR_NULL;
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
