// What the sequence operators (causal convolution, selective scan) share: tracks, resets and lengths on
// the device, and their checks on the host.
#pragma once

#include <algorithm>
#include <type_traits>

#include "ops.cuh"

namespace t8b {
namespace op {

// Row t of sequence s of a track.
template <typename T>
struct Track {
    T* data;
    int64_t sequence, step;
    Track() = default;
    explicit Track(const t8b_track_t& t) : data(static_cast<T*>(t.data)), sequence(t.sequence), step(t.step) {}
    __device__ __forceinline__ T* at(int64_t s) const { return data + s * sequence; }
};

struct Sequences {
    int64_t sequences;
    int steps, channels;
    const uint8_t* reset;
    int64_t reset_sequence, reset_step;
    const int32_t* lengths;
    Sequences() = default;
    explicit Sequences(const t8b_sequences_t& q)
        : sequences(q.sequences), steps(static_cast<int>(q.steps)), channels(static_cast<int>(q.channels)), reset(q.reset),
          reset_sequence(q.reset_sequence), reset_step(q.reset_step), lengths(q.lengths) {}
    // steps of sequence s that count
    __device__ __forceinline__ int live(int64_t s) const {
        return lengths == nullptr ? steps : min(max(lengths[s], 0), steps);
    }
    __device__ __forceinline__ bool resets(int64_t s, int t) const {
        return reset != nullptr && reset[s * reset_sequence + t * reset_step] != 0;
    }
};

// Keeps the compiler from moving an unrolled step's loads in front of the steps before it, where they
// would wait in registers.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// 4, 8 or 16 bytes into shared memory without waiting for them.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "n"(BYTES)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// V consecutive elements as they lie in memory: whole words where they make one, so that no register holds half of
// what it could (a struct of 16-bit elements is taken apart into them when it is copied).
template <typename T, int V>
struct alignas(sizeof(T) * V) Words {
    uint32_t w[sizeof(T) * V / 4];
};
template <typename T, int V>
using Held = std::conditional_t<(sizeof(T) * V >= 4), Words<T, V>, Pack<T, V>>;  // Held<T, V>{} are zeros
template <typename T, int V>
__device__ __forceinline__ Held<T, V> load_held(const T* p) {
    return *reinterpret_cast<const Held<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_held(T* p, const Held<T, V>& v) {
    *reinterpret_cast<Held<T, V>*>(p) = v;
}
// In fp32,
template <typename T, int V>
__device__ __forceinline__ void unpack(const Held<T, V>& p, float (&v)[V]) {
    if constexpr (sizeof(T) * V < 4) {
        v[0] = Element<T>::load(p.v[0]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __uint_as_float(p.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = Element<T>::unpack(p.w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ Held<T, V> pack(const float (&v)[V]) {
    Held<T, V> p;
    if constexpr (sizeof(T) * V < 4) {
        p.v[0] = Element<T>::store(v[0]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) p.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) p.w[i] = Element<T>::pack(v[2 * i], v[2 * i + 1]);
    }
    return p;
}
// and as register pairs; a single element has 0 beside it.
template <typename T, int V>
__device__ __forceinline__ void unpack(const Held<T, V>& p, Two (&v)[(V + 1) / 2]) {
    float f[V];
    unpack<T, V>(p, f);
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) v[i] = Two(f[2 * i], 2 * i + 1 < V ? f[2 * i + 1 < V ? 2 * i + 1 : 0] : 0.0f);
}
template <typename T, int V>
__device__ __forceinline__ Held<T, V> pack(const Two (&v)[(V + 1) / 2]) {
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 w = v[i / 2].get();
        f[i] = i % 2 ? w.y : w.x;
    }
    return pack<T, V>(f);
}

constexpr float kLn2 = 0.69314718055994531f;
// exp(v), v <= 0, the argument's product with log2 e to twice the precision: good to 2^x's own 2^-22, and without
// the bias that it has for x below -0.25 (4.8e-8 of the value in the mean; above it next to none).
__device__ __forceinline__ float exponential(float v) {
    const float high = v * kLog2E;
    const float low = fmaf(v, 1.925963033e-8f, fmaf(v, kLog2E, -high));  // log2 e - fp32(log2 e)
    const float r = power_of_two(high);
    return fabsf(high) < 200.0f ? fmaf(r, fmaf(low, kLn2, high < -0.25f ? 4.8e-8f : 0.0f), r) : r;
}

// ------------------------------------------------------------------ host checks
constexpr int64_t kMostElements = int64_t{1} << 61;
constexpr int64_t kMostSequences = int64_t{1} << 30, kMostSteps = int64_t{1} << 30, kMostChannels = int64_t{1} << 20;

// Whether the plans may count these sequences: the kernels' numbers of steps, channels and blocks have 32 bits. The
// queries answer 0 for others, which the calls refuse.
inline bool countable(const t8b_sequences_t& q) {
    return q.sequences >= 0 && q.sequences <= kMostSequences && q.steps >= 0 && q.steps <= kMostSteps && q.channels >= 1 &&
        q.channels <= kMostChannels;
}
inline void check_sequences(const char* what, const t8b_sequences_t* q, bool step) {
    const std::string name(what);
    if (q == nullptr) raise(T8B_EINVAL, name + ": the sequences are null");
    if (q->sequences < 0 || q->sequences > kMostSequences) raise(T8B_EINVAL, name + ": 0 to 2^30 sequences");
    if (!step && (q->steps < 0 || q->steps > kMostSteps)) raise(T8B_EINVAL, name + ": 0 to 2^30 steps");
    if (q->channels < 1 || q->channels > kMostChannels) raise(T8B_EINVAL, name + ": 1 to 2^20 channels");
    const int64_t steps = step ? 1 : std::max<int64_t>(q->steps, 1);
    if (q->reset != nullptr &&
        (q->reset_sequence < 0 || q->reset_step < 0 || q->reset_sequence > kMostElements / std::max<int64_t>(q->sequences, 1) ||
         q->reset_step > kMostElements / steps)) {
        raise(T8B_EINVAL, name + ": the strides of reset are out of range");
    }
    check_elements(what, q->lengths, sizeof(int32_t));
}
inline void check_track(const char* what, const t8b_sequences_t& q, bool step, const t8b_track_t& t, int64_t width, size_t size,
                        bool output) {
    const std::string name(what);
    const int64_t steps = step ? 1 : q.steps;
    if (q.sequences == 0 || steps == 0) return;
    if (t.data == nullptr) raise(T8B_EINVAL, name + " is null");
    check_elements(what, t.data, size);
    const int64_t s = q.sequences > 1 ? t.sequence : 0, r = steps > 1 ? t.step : 0;
    if (s < 0 || r < 0 || s > kMostElements / q.sequences || r > kMostElements / steps) {
        raise(T8B_EINVAL, name + ": a stride is out of range");
    }
    if (!output) return;
    // no two of its rows may share an element: one axis lies within the other's stride
    const int64_t of_steps = (steps - 1) * r + width, of_sequences = (q.sequences - 1) * s + width;
    const bool inner_steps = (steps == 1 || r >= width) && (q.sequences == 1 || s >= of_steps);
    const bool inner_sequences = (q.sequences == 1 || s >= width) && (steps == 1 || r >= of_sequences);
    if (!inner_steps && !inner_sequences) raise(T8B_EINVAL, name + ": its rows overlap");
}
// The bytes that a track spans.
inline Span span_of(const t8b_sequences_t& q, bool step, const t8b_track_t& t, int64_t width, size_t size) {
    const int64_t steps = step ? 1 : q.steps;
    Span span(t.data, 0, 0, 0, 0);
    if (t.data != nullptr && q.sequences > 0 && steps > 0) {
        const int64_t s = q.sequences > 1 ? t.sequence : 0, r = steps > 1 ? t.step : 0;
        span.last = span.first + ((q.sequences - 1) * s + (steps - 1) * r + width) * size;
    }
    return span;
}
inline Span span_of(const void* data, int64_t count, size_t size) { return Span(data, 1, count, count, size); }
// No output may overlap an input or another output.
struct Overlaps {
    const char* what;
    std::vector<Span> inputs, outputs;
    void input(const Span& s) { inputs.push_back(s); }
    void output(const Span& s) {
        for (const auto* others : {&inputs, &outputs}) {
            for (const Span& o : *others) {
                if (s.overlaps(o)) raise(T8B_EINVAL, std::string(what) + ": an output overlaps an input or another output");
            }
        }
        outputs.push_back(s);
    }
};
// Whether every row of a track starts on `bytes`.
inline bool rows_aligned(const t8b_sequences_t& q, bool step, const t8b_track_t& t, size_t size, size_t bytes) {
    const bool s = q.sequences <= 1 || t.sequence * size % bytes == 0;
    const bool r = step || q.steps <= 1 || t.step * size % bytes == 0;
    return aligned(t.data, bytes) && s && r;
}

template <typename Body>
void with_type(int type, Body&& body) {
    switch (type) {
        case T8B_F32: body(float{}); break;
        case T8B_BF16: body(bf16{}); break;
        default: body(f16{}); break;
    }
}

}  // namespace op
}  // namespace t8b
