// What the operator kernels (layer norm, linear, gated) share: element types and their
// conversions, activations and their slopes, and the host-side argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <limits>
#include <string>

#include "common.cuh"

namespace t8b {
namespace op {

using bf16 = __nv_bfloat16;
using f16 = __half;

// ------------------------------------------------------------------ element types
template <typename T>
struct Element;
template <>
struct Element<float> {
    static constexpr int kType = T8B_F32;
    __device__ static float load(float v) { return v; }
    __device__ static float store(float v) { return v; }
};
template <>
struct Element<bf16> {
    static constexpr int kType = T8B_BF16;
    __device__ static float load(bf16 v) { return __bfloat162float(v); }
    __device__ static bf16 store(float v) { return __float2bfloat16_rn(v); }
    __device__ static float2 unpack(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
    __device__ static uint32_t pack(float a, float b) {
        __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&p);
    }
};
template <>
struct Element<f16> {
    static constexpr int kType = T8B_F16;
    __device__ static float load(f16 v) { return __half2float(v); }
    __device__ static f16 store(float v) { return __float2half_rn(v); }
    __device__ static float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
    __device__ static uint32_t pack(float a, float b) {
        __half2 p = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&p);
    }
};

// One element of an array whose type is known at run time (parameters: read once per block).
__device__ __forceinline__ float load_any(const void* p, int type, size_t i) {
    if (type == T8B_F32) return static_cast<const float*>(p)[i];
    if (type == T8B_BF16) return __bfloat162float(static_cast<const bf16*>(p)[i]);
    return __half2float(static_cast<const f16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, size_t i, float v) {
    if (type == T8B_F32) {
        static_cast<float*>(p)[i] = v;
    } else if (type == T8B_BF16) {
        static_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
    } else {
        static_cast<f16*>(p)[i] = __float2half_rn(v);
    }
}

// V consecutive elements as they lie in memory, moved by the widest access that V allows
// (p aligned to the pack's size, or V = 1).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// Two fp32 values in a register pair, and the machine's packed operations on them: one instruction
// for both, each rounded as its scalar form.
struct Two {
    unsigned long long bits;
    __device__ __forceinline__ Two() : bits(0) {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
    __device__ __forceinline__ float2 get() const {
        float2 v;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(bits));
        return v;
    }
    __device__ __forceinline__ float sum() const {
        const float2 v = get();
        return v.x + v.y;
    }
};
__device__ __forceinline__ Two operator+(const Two& a, const Two& b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two operator*(const Two& a, const Two& b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two multiply_add(const Two& a, const Two& b, const Two& c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}

// ------------------------------------------------------------------ activations
// In fp32, from the machine's 2^x and 1/x (each good to about 2^-22): exp(v) = 2^(v log2 e), whose argument is
// rounded once and adds |v| 2^-24,
//   sigmoid(z) = 1 / (1 + exp(-z)),
//   tanh(z) = 1 - 2 / (1 + exp(2z)), and below |z| = 0.2, where that difference cancels, the
//     series z - z^3/3 + 2 z^5/15 - 17 z^7/315 (its next term is at most 2^-24 of z there),
//   Phi(z) = (1 + erf(z / sqrt 2)) / 2 with erfc(x) = t (a1 + t (a2 + ... t a5)) exp(-x^2),
//     t = 1 / (1 + p x), x >= 0: Abramowitz and Stegun, Handbook of Mathematical Functions,
//     7.1.26. Its error is 1.5e-7 absolute, so Phi is good to 7e-8 and fp32's roundings. The lower tail is
//     that product itself, not a difference from 1, but its relative error grows all the same: 5e-5 at z =
//     -3, 5e-4 at -4, 1.6e-3 at -5, 3.6e-3 at -6 (half a bf16 spacing is 3.9e-3; gelu(-6) is 6e-9).
// Where z is infinite they give what the formulas do: silu(-inf) and gelu(-inf) are NaN (0 * inf).
__device__ __forceinline__ float power_of_two(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid(float z) { return reciprocal(1.0f + power_of_two(-kLog2E * z)); }
__device__ __forceinline__ float hyperbolic_tangent(float z) {
    const float square = z * z;
    const float near = z * fmaf(square, fmaf(square, fmaf(square, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    const float far = fmaf(-2.0f, reciprocal(1.0f + power_of_two(2.0f * kLog2E * z)), 1.0f);
    return fabsf(z) < 0.2f ? near : far;
}
// Phi(z), and exp(-z^2 / 2) on the way
__device__ __forceinline__ float normal_cdf(float z, float& gauss) {
    gauss = power_of_two(-0.5f * kLog2E * z * z);
    const float t = reciprocal(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
    const float series =
        t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * series * gauss;
    return z > 0.0f ? 1.0f - tail : tail;
}
template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if (ACT == T8B_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (ACT == T8B_GELU) {
        float gauss;
        return z * normal_cdf(z, gauss);
    }
    if (ACT == T8B_SILU) return z * sigmoid(z);
    if (ACT == T8B_TANH) return hyperbolic_tangent(z);
    return z;
}
// activate(z) and its derivative
template <int ACT>
__device__ __forceinline__ void activate_slope(float z, float& value, float& slope) {
    if (ACT == T8B_RELU) {
        value = activate<T8B_RELU>(z);
        slope = z > 0.0f ? 1.0f : 0.0f;
    } else if (ACT == T8B_GELU) {
        float gauss;
        const float cdf = normal_cdf(z, gauss);
        value = z * cdf;
        slope = fmaf(0.39894228040143268f * z, gauss, cdf);
    } else if (ACT == T8B_SILU) {
        const float s = sigmoid(z);
        value = z * s;
        slope = s * fmaf(z, 1.0f - s, 1.0f);
    } else if (ACT == T8B_TANH) {
        value = hyperbolic_tangent(z);
        slope = fmaf(-value, value, 1.0f);
    } else {
        value = z;
        slope = 1.0f;
    }
}

// Calls body with the activation as a compile-time constant.
template <int N>
struct Constant {
    static constexpr int value = N;
};
template <typename Body>
__host__ __device__ __forceinline__ void with_activation(int act, Body&& body) {
    switch (act) {
        case T8B_RELU: body(Constant<T8B_RELU>{}); break;
        case T8B_GELU: body(Constant<T8B_GELU>{}); break;
        case T8B_SILU: body(Constant<T8B_SILU>{}); break;
        case T8B_TANH: body(Constant<T8B_TANH>{}); break;
        default: body(Constant<T8B_LINEAR>{}); break;
    }
}

// ------------------------------------------------------------------ host checks
inline size_t type_size(int type) { return type == T8B_F32 ? 4 : 2; }
inline bool is_type(int type) { return type == T8B_F32 || type == T8B_BF16 || type == T8B_F16; }
inline bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }
inline size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// An array argument (or NULL): the kernels read it by whole elements.
inline void check_elements(const char* what, const void* data, size_t size) {
    if (!aligned(data, size)) raise(T8B_EINVAL, std::string(what) + ": a pointer that is not aligned to its elements");
}
// A row-major matrix argument: its rows must not overlap, its last element must be addressable.
inline void check_matrix(const char* what, const void* data, int64_t rows, int64_t columns, int64_t stride, size_t size) {
    if (rows == 0) return;
    if (data == nullptr) raise(T8B_EINVAL, std::string(what) + " is null");
    check_elements(what, data, size);
    if (rows > 1 && stride < columns) raise(T8B_EINVAL, std::string(what) + ": a row stride below the row's length");
    if (stride < 0 || (rows > 1 && stride > std::numeric_limits<int64_t>::max() / 8 / rows)) {
        raise(T8B_EINVAL, std::string(what) + ": the row stride is out of range");
    }
}

// [first, last) of the bytes a matrix spans.
struct Span {
    uintptr_t first, last;
    Span(const void* data, int64_t rows, int64_t columns, int64_t stride, size_t size)
        : first(reinterpret_cast<uintptr_t>(data)), last(first) {
        if (data != nullptr && rows > 0 && columns > 0) last = first + ((rows - 1) * stride + columns) * size;
    }
    bool overlaps(const Span& o) const { return first < o.last && o.first < last; }
};

// A kernel's dynamic shared memory, allowed once per device.
template <typename Kernel>
inline void allow_smem(Kernel kernel, size_t bytes, uint64_t& configured) {
    if (bytes <= 32 * 1024) return;  // with the static part, below what needs no leave
    int device = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    const uint64_t bit = 1ull << (device & 63);
    if ((__atomic_load_n(&configured, __ATOMIC_ACQUIRE) & bit) != 0) return;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)), "shared memory");
    __atomic_fetch_or(&configured, bit, __ATOMIC_RELEASE);
}

// A launch behind whatever the stream holds: with `chained` its blocks may start before the kernel
// before it has ended, as soon as every block of that one has passed release_next() (or ended, for
// a kernel that does not call it), so launch latency and prologues overlap its tail. They call
// wait_previous() before they touch memory that it may read or write, and only then release the next,
// so that by induction everything earlier has ended too.
template <typename Kernel, typename... Args>
inline void launch_chain(const char* label, Kernel kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool chained,
                         const Args&... args) {
    LaunchScope scope(label, stream);
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = chained ? 1 : 0;
    check(cudaLaunchKernelEx(&config, kernel, args...), label);
}
// What the kernel before it is to a kernel. kInput: anything, so this one waits for it first. kBeside:
// another of the same call that shares nothing with this one, whose blocks fill the SMs that it leaves
// idle and wait for it before they end; what came before it had ended before any of its blocks let
// this one start.
enum { kInput = 1, kBeside = 2 };
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace op
}  // namespace t8b
