// Clipped policy loss over each row's legal logits, with entropy and the divergence from a reference
// policy, and its gradient in the same pass.
//
//   lp = z[a] - lse(z),  r = exp(lp - old),  loss = -min(r A, clip(r) A) + kl K - entropy H
//   dloss/dz_i = p_i (c + kl log(p_i / q_i) + entropy log p_i) + [i = a] slope,
//   slope = dloss/dlp = -r A where the unclipped term is the smaller (0 where not) + the sampled K's 1 - exp(e)
//
// where c gathers what is the same for a whole row. Bound by memory: logits (and a reference's) once in,
// the gradient once out. A row of up to 1,024 logits lies in the registers of 8, 16 or 32 lanes, as few as hold it with 32
// each: what a row costs beside its logits is shared by the rows of a warp. A longer one belongs to a
// block that reads it twice, for its sums and for its gradient; the second read comes from L2, where
// the rows that are worked on at once fit many times over. 65,536 x 368 in fp32 with bits and a reference: 78 us (58 %
// of the copy rate; a row's load, work and store follow one another), 4,096 x 50,257 in bf16 242 us (52 %: 21
// instructions a logit in both passes).
// With m the largest legal logit and t_i = log2(e) (z_i - m): e_i = 2^t_i, and every logarithm of a
// probability is ln 2 t_i - ln(sum e), with the last taken in 64 bits, since the ratio and the divergence are
// differences of it.
#include "ops_memory.cuh"

namespace t8b {
namespace op {
namespace {

constexpr int kWarps = 4;          // warps of a block that gives a row to each
constexpr int kMostHeld = 32;      // logits of a lane there
constexpr int kMostShort = 32 * kMostHeld;
constexpr int kMostThreads = 256;  // threads of a block that shares a row

// Blocks of that form that an SM is to hold: their loads wait together, and more of them hide more
// (65,536 x 368 in fp32 with a reference, 24 logits a lane: 87 us with 4 blocks, 80 with 5, 77 with 6).
__host__ __device__ constexpr int resident_blocks(int held) { return held <= 16 ? 8 : held <= 24 ? 6 : 4; }

struct Loss {
    const void* logits;
    const void* reference;
    const void* mask;
    const int64_t* actions;
    const float *old, *advantages, *weights;
    float *loss, *log_probabilities, *entropies, *divergences;
    void* gradient;
    int64_t logits_stride, reference_stride, mask_stride, gradient_stride, rows;
    int n, mask_kind, reference_kind;
    float low, high, kl, entropy, even;  // the clipped ratio's range; even: the weight without weights
};

// Which of `count` consecutive actions from e on are legal, a bit each; they lie in one word.
template <int COUNT>
__device__ __forceinline__ uint32_t legal_bits(const Loss& a, int64_t row, int e) {
    uint32_t bits = COUNT == 32 ? 0xffffffffu : (1u << COUNT) - 1;
    if (a.mask_kind == T8B_MASK_BITS) {
        bits &= static_cast<const uint32_t*>(a.mask)[row * a.mask_stride + e / 32] >> (e % 32);
    } else if (a.mask_kind == T8B_MASK_BYTES) {
        const uint8_t* m = static_cast<const uint8_t*>(a.mask) + row * a.mask_stride + e;
        bits = 0;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) bits |= e + i < a.n && m[i] != 0 ? 1u << i : 0u;
    }
    return e + COUNT <= a.n ? bits : bits & ((1u << max(a.n - e, 0)) - 1);
}
__device__ __forceinline__ bool legal(const Loss& a, int64_t row, int64_t action) {
    return action >= 0 && action < a.n && (legal_bits<1>(a, row, static_cast<int>(action)) & 1) != 0;
}

constexpr float kLn2 = 0.69314718055994531f;
constexpr double kExactLn2 = 0.693147180559945309;
// The machine's 2^x is off by -4.5e-8 to -5.1e-8 of the value in the mean for x below -0.25 (a million values of each range),
// which all of a row's exponentials and their sum share: arguments are longer by what makes up for it. (Above -0.25 it
// is off by less than 2.6e-8: those are up to 4.8e-8 too large.) Where t stands for a logarithm that is taken out again.
constexpr float kUnbiased = 6.9e-8f;
constexpr float kNever = -1000.0f;  // 2^kNever is 0, and a factor of 0 beside it gives 0, not NaN

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// ln(v), v from about 2^-100 to 2^100, to 2^-34: v = 2^k w with w in [3/4, 3/2), ln w = 2 atanh(q), q = (w - 1) /
// (w + 1) in [-1/7, 1/5], by its series (the next term is 2 q^15 / 15). Others (0, NaN, inf) by log().
__device__ __forceinline__ double natural_log(double v) {
    const int high = __double2hiint(v);
    if (static_cast<unsigned>(high - ((1023 - 100) << 20)) > 200u << 20) return log(v);
    const int k = ((high + (1 << 19)) >> 20) - 1023;
    const double w = __hiloint2double(high - (k << 20), __double2loint(v));
    const double below = w + 1.0;
    double r = static_cast<double>(reciprocal(static_cast<float>(below)));  // two steps of Newton's method: 2^-22, 2^-44
    r = fma(r, fma(-below, r, 1.0), r);
    const double q = (w - 1.0) * r, square = q * q;
    double p = fma(square, 1.0 / 13.0, 1.0 / 11.0);
    p = fma(square, p, 1.0 / 9.0);
    p = fma(square, p, 1.0 / 7.0);
    p = fma(square, p, 1.0 / 5.0);
    p = fma(square, p, 1.0 / 3.0);
    return fma(static_cast<double>(k), kExactLn2, 2.0 * fma(q * square, p, q));
}

// A row's sums: m as above, total = sum e, spread = sum e t, apart = sum e (t - t of the reference); the first
// two of the reference as far as it is needed.
struct Sums {
    float m = -INFINITY, q_m = -INFINITY;
    float spread = 0.0f, apart = 0.0f;
    double total = 0.0, q_total = 0.0;
};
// A row's gradient: e scale (base + of_t t + of_apart (t - t of the reference)) + [i = action] slope
struct Slopes {
    float scale, slope, base, of_t, of_apart;
    // Whether 0 times the rest is 0: an infinite divergence or advantage, say, makes NaN of a logit that is not legal.
    __device__ __forceinline__ bool finite() const { return fabsf(scale) + fabsf(base) - kNever * fabsf(of_t) < INFINITY; }
};

// What a row has beside its logits.
struct Scalars {
    int64_t action = -1;
    float old = 0.0f, advantage = 0.0f, weight = 0.0f, sampled = 0.0f;
    __device__ __forceinline__ void load(const Loss& a, int64_t row) {
        action = a.actions[row];
        old = a.old[row];
        advantage = a.advantages[row];
        weight = a.weights ? a.weights[row] : a.even;
        if (a.reference_kind == T8B_REFERENCE_SAMPLED) sampled = static_cast<const float*>(a.reference)[row];
    }
};

// The row's outputs from its sums; every thread that calls it gets the slopes, `writes` stores.
__device__ __forceinline__ Slopes finish(const Loss& a, int64_t row, const Scalars& given, float chosen, const Sums& s, bool writes) {
    const double log_total = natural_log(s.total);
    const double lp = (static_cast<double>(chosen) - static_cast<double>(s.m)) - log_total;
    const float share = 1.0f / static_cast<float>(s.total), log_sum = static_cast<float>(log_total);
    // spread has t in it as it is lengthened, and so has the gradient
    const float entropy = static_cast<float>(log_total - static_cast<double>(kLn2 * (s.spread * share - kUnbiased)));
    const float advantage = given.advantage;
    const float ratio = expf(static_cast<float>(lp - static_cast<double>(given.old)));
    const float free = ratio * advantage, held = fminf(fmaxf(ratio, a.low), a.high) * advantage;
    const bool unclipped = free <= held || free != free;
    float loss = -(unclipped ? free : held), slope = unclipped ? -free : 0.0f, divergence = 0.0f;
    Slopes out;
    out.base = a.entropy * ((entropy - log_sum) - kLn2 * kUnbiased);
    out.of_t = a.entropy * kLn2;
    out.of_apart = 0.0f;
    if (a.reference_kind == T8B_REFERENCE_LOGITS) {
        // log p_i - log q_i = ln 2 (t_i - t of q_i) - gap
        const double gap = log_total - natural_log(s.q_total);  // t has the rows' own largest logits in it
        divergence = static_cast<float>(static_cast<double>(kLn2 * (s.apart * share)) - gap);
        out.base -= a.kl * (static_cast<float>(gap) + divergence);
        out.of_apart = a.kl * kLn2;
    } else if (a.reference_kind == T8B_REFERENCE_SAMPLED) {
        const float e = static_cast<float>(static_cast<double>(given.sampled) - lp);
        // exp(e) - 1 - e, by its series where the difference would cancel
        const float grown = expm1f(e);
        divergence = fabsf(e) < 0.1f
            ? e * e * fmaf(e, fmaf(e, fmaf(e, fmaf(e, 1.0f / 720.0f, 1.0f / 120.0f), 1.0f / 24.0f), 1.0f / 6.0f), 0.5f)
            : grown - e;
        slope -= a.kl * grown;
    }
    out.base -= slope;
    loss += a.kl * divergence - a.entropy * entropy;
    if (writes) {
        if (a.loss) a.loss[row] = loss;
        if (a.log_probabilities) a.log_probabilities[row] = static_cast<float>(lp);
        if (a.entropies) a.entropies[row] = entropy;
        if (a.divergences) a.divergences[row] = divergence;
    }
    out.scale = given.weight * share;
    out.slope = given.weight * slope;
    return out;
}
__device__ __forceinline__ void finish_nothing(const Loss& a, int64_t row) {
    for (float* p : {a.loss, a.log_probabilities, a.entropies, a.divergences}) {
        if (p) p[row] = 0.0f;
    }
}
__device__ __forceinline__ Two powers_of_two(const Two& v) {
    const float2 f = v.get();
    return Two(power_of_two(f.x), power_of_two(f.y));
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* to, const float (&v)[V]) {
    *reinterpret_cast<Held<T, V>*>(to) = pack<T, V>(v);
}
template <int V>
__device__ __forceinline__ void add_chosen(float (&v)[V], int64_t e, int64_t action, float slope) {
    if (action < e || action >= e + V) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (e + j == action) v[j] += slope;
    }
}

// 0 at the logits of a thread's pack that are not legal, behind its store.
template <typename T, int V>
__device__ __forceinline__ void clear_masked(const Loss& a, int64_t row, T* g, int e) {
    const uint32_t bits = legal_bits<V>(a, row, e);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if ((bits >> j & 1) == 0) g[e + j] = Element<T>::store(0.0f);
    }
}

// LANES lanes a row; lane l holds the packs l, l + LANES, ... of V logits.
template <typename T, int V, int LANES, int HELD, bool REFERENCE>
__global__ void __launch_bounds__(32 * kWarps, resident_blocks(HELD)) k_policy_loss(Loss a) {
    constexpr int PACKS = HELD / V, H = HELD / 2;
    wait_previous();
    release_next();
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (32 * kWarps / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    const bool mine = at < a.rows;  // the last warp's lanes go along without a row of their own
    const int64_t row = mine ? at : a.rows - 1;
    const T* z = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const T* q = REFERENCE ? static_cast<const T*>(a.reference) + row * a.reference_stride : nullptr;
    T* g = a.gradient ? static_cast<T*>(a.gradient) + row * a.gradient_stride : nullptr;
    Held<T, V> raw[PACKS], raw_q[REFERENCE ? PACKS : 1];
    uint32_t bits[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        const int e = (i * LANES + lane) * V;
        bits[i] = 0;
        if (e < a.n) {  // n is a multiple of V
            raw[i] = load_held<T, V>(z + e);
            if (REFERENCE) raw_q[REFERENCE ? i : 0] = load_held<T, V>(q + e);
            bits[i] = legal_bits<V>(a, row, e);
        }
    }
    Scalars scalars;
    scalars.load(a, row);
    const int64_t action = scalars.action;
    const bool counts = legal(a, row, action);
    const float chosen = counts ? Element<T>::load(z[action]) : 0.0f;
    Sums s;
    float v[HELD], w[REFERENCE ? HELD : 1];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        float x[V], y[V];
        unpack<T, V>(raw[i], x);
        if (REFERENCE) unpack<T, V>(raw_q[REFERENCE ? i : 0], y);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool in = bits[i] >> j & 1;
            v[i * V + j] = in ? x[j] : -INFINITY;
            s.m = fmaxf(s.m, v[i * V + j]);
            if (REFERENCE) {
                w[REFERENCE ? i * V + j : 0] = in ? y[j] : -INFINITY;
                s.q_m = fmaxf(s.q_m, w[REFERENCE ? i * V + j : 0]);
            }
        }
    }
#pragma unroll
    for (int o = LANES / 2; o >= 1; o >>= 1) {
        s.m = fmaxf(s.m, __shfl_xor_sync(0xffffffffu, s.m, o));
        if (REFERENCE) s.q_m = fmaxf(s.q_m, __shfl_xor_sync(0xffffffffu, s.q_m, o));
    }
    // t, and t less the reference's
    Two t[H], away[REFERENCE ? H : 1], total, q_total, spread, apart;
    const Two scale(kLog2E, kLog2E), unbiased(kUnbiased, kUnbiased), from(-s.m, -s.m), q_from(-s.q_m, -s.q_m);
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const float2 x = multiply_add(Two(v[2 * i], v[2 * i + 1]) + from, scale, unbiased).get();
        t[i] = Two(max_nan(x.x, kNever), max_nan(x.y, kNever));
        const Two e = powers_of_two(t[i]);
        total = total + e;
        spread = multiply_add(e, t[i], spread);
        if (REFERENCE) {
            const Two u = multiply_add(Two(w[REFERENCE ? 2 * i : 0], w[REFERENCE ? 2 * i + 1 : 0]) + q_from, scale, unbiased);
            q_total = q_total + powers_of_two(u);
            const float2 f = e.get(), d = multiply_add(u, Two(-1.0f, -1.0f), t[i]).get();
            away[REFERENCE ? i : 0] = Two(f.x != 0.0f ? d.x : 0.0f, f.y != 0.0f ? d.y : 0.0f);
            apart = multiply_add(e, away[REFERENCE ? i : 0], apart);
        }
    }
    s.total = total.sum();
    s.q_total = q_total.sum();
    s.spread = spread.sum();
    s.apart = apart.sum();
#pragma unroll
    for (int o = LANES / 2; o >= 1; o >>= 1) {
        s.total += __shfl_xor_sync(0xffffffffu, s.total, o);
        s.spread += __shfl_xor_sync(0xffffffffu, s.spread, o);
        if (REFERENCE) {
            s.q_total += __shfl_xor_sync(0xffffffffu, s.q_total, o);
            s.apart += __shfl_xor_sync(0xffffffffu, s.apart, o);
        }
    }
    if (!mine) return;
    if (!counts) {
        if (lane == 0) finish_nothing(a, row);
        if (g == nullptr) return;
        const float zero[V] = {};
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int e = (i * LANES + lane) * V;
            if (e < a.n) store_pack<T, V>(g + e, zero);
        }
        return;
    }
    const Slopes k = finish(a, row, scalars, chosen, s, lane == 0);
    if (g == nullptr) return;
    const Two of_t(k.of_t, k.of_t), base(k.base, k.base), of_apart(k.of_apart, k.of_apart), part(k.scale, k.scale);
#pragma unroll
    for (int i = 0; i < H; ++i) {
        Two inner = multiply_add(of_t, t[i], base);
        if (REFERENCE) inner = multiply_add(of_apart, away[REFERENCE ? i : 0], inner);
        const float2 out = (powers_of_two(t[i]) * part * inner).get();
        v[2 * i] = out.x;
        v[2 * i + 1] = out.y;
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
        const int e = (i * LANES + lane) * V;
        if (e >= a.n) continue;
        float out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = v[i * V + j];
        add_chosen<V>(out, e, action, k.slope);
        store_pack<T, V>(g + e, out);
    }
    if (a.mask_kind == T8B_MASK_NONE || k.finite()) return;
    for (int e = lane * V; e < a.n; e += LANES * V) clear_masked<T, V>(a, row, g, e);
}

// What a new largest logit adds to every t, far enough down for 2^gap to be 0 where the old one was -inf or the lowest
// value; and what the reference's adds to t less its t, where it had one before.
__device__ __forceinline__ float gap_of(float m, float next) { return fmaxf((m - next) * kLog2E, -10000.0f); }
__device__ __forceinline__ float back_of(float m, float next) {
    return m == -INFINITY ? 0.0f : fminf((next - m) * kLog2E, 3.402823466e38f);
}

// One block a row, V consecutive logits a thread and a turn. MASKED: some may not be legal.
template <typename T, int V, bool REFERENCE, bool MASKED>
__global__ void __launch_bounds__(kMostThreads, REFERENCE ? 4 : 5) k_policy_loss_long(Loss a) {
    wait_previous();
    release_next();
    __shared__ float most[2][kMostThreads / 32], sums[2][kMostThreads / 32];
    __shared__ double totals[2][kMostThreads / 32];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const T* z = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const T* q = REFERENCE ? static_cast<const T*>(a.reference) + row * a.reference_stride : nullptr;
    T* g = a.gradient ? static_cast<T*>(a.gradient) + row * a.gradient_stride : nullptr;
    Scalars scalars;
    scalars.load(a, row);
    const int64_t action = scalars.action;
    const int whole = a.n / V * V, step = blockDim.x * V;
    if (!legal(a, row, action)) {
        if (threadIdx.x == 0) finish_nothing(a, row);
        if (g == nullptr) return;
        const float zero[V] = {};
        for (int e = threadIdx.x * V; e < whole; e += step) store_pack<T, V>(g + e, zero);
        for (int e = whole + threadIdx.x; e < a.n; e += blockDim.x) g[e] = Element<T>::store(0.0f);
        return;
    }
    const float chosen = Element<T>::load(z[action]);
    const Two scale(kLog2E, kLog2E), unbiased(kUnbiased, kUnbiased);
    Sums s;
    Two total, q_total, spread, apart;  // two parts of each sum, alike in m
    auto masked = [&](auto count, const T* from, int e, uint32_t bits, auto& x) {  // logits, -inf where they are not legal
        constexpr int COUNT = decltype(count)::value;
        unpack<T, COUNT>(load_held<T, COUNT>(from + e), x);
        if (COUNT == 1) x[0] = Two(x[0].get().x, -INFINITY);
        if constexpr (MASKED) {
#pragma unroll
            for (int i = 0; i < (COUNT + 1) / 2; ++i) {
                const float2 f = x[i].get();
                x[i] = Two(bits >> (2 * i) & 1 ? f.x : -INFINITY, bits >> (2 * i + 1) & 1 ? f.y : -INFINITY);
            }
        }
    };
    // COUNT logits into the sums, which move to a new largest one first. While a thread has seen nothing but
    // -inf its m is 0 here: every e is 0.
    auto take = [&](auto count, int e) {
        constexpr int COUNT = decltype(count)::value, H = (COUNT + 1) / 2;
        const uint32_t bits = MASKED ? legal_bits<COUNT>(a, row, e) : 0;
        Two x[H], y[H];
        float m = -INFINITY, q_m = -INFINITY;
        masked(count, z, e, bits, x);
        if (REFERENCE) masked(count, q, e, bits, y);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float2 f = x[i].get();
            m = fmaxf(m, fmaxf(f.x, f.y));
            if (REFERENCE) {
                const float2 k = y[i].get();
                q_m = fmaxf(q_m, fmaxf(k.x, k.y));
            }
        }
        if (m > s.m) {
            const float gap = gap_of(s.m, m), f = power_of_two(gap);
            const Two by(f, f), away(gap, gap);
            spread = f == 0.0f ? Two() : by * multiply_add(away, total, spread);
            apart = f == 0.0f ? Two() : by * multiply_add(away, total, apart);
            total = by * total;
            s.m = m;
        }
        if (REFERENCE && q_m > s.q_m) {
            const float back = back_of(s.q_m, q_m), f = power_of_two(gap_of(s.q_m, q_m));
            apart = multiply_add(Two(back, back), total, apart);
            q_total = Two(f, f) * q_total;
            s.q_m = q_m;
        }
        const float from = s.m == -INFINITY ? 0.0f : -s.m, q_from = s.q_m == -INFINITY ? 0.0f : -s.q_m;
        const Two off(from, from), q_off(q_from, q_from);
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float2 f = multiply_add(x[i] + off, scale, unbiased).get();
            const Two t(max_nan(f.x, kNever), max_nan(f.y, kNever)), p = powers_of_two(t);
            total = total + p;
            spread = multiply_add(p, t, spread);
            if (REFERENCE) {
                const Two u = multiply_add(y[i] + q_off, scale, unbiased);
                q_total = q_total + powers_of_two(u);
                const float2 d = multiply_add(u, Two(-1.0f, -1.0f), t).get(), k = p.get();
                apart = multiply_add(p, Two(k.x != 0.0f ? d.x : 0.0f, k.y != 0.0f ? d.y : 0.0f), apart);
            }
        }
    };
#pragma unroll 4
    for (int e = threadIdx.x * V; e < whole; e += step) take(Constant<V>{}, e);
    for (int e = whole + threadIdx.x; e < a.n; e += blockDim.x) take(Constant<1>{}, e);
    // the threads' sums, each moved to the row's largest logit
    float m = s.m, q_m = s.q_m;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (REFERENCE) q_m = fmaxf(q_m, __shfl_xor_sync(0xffffffffu, q_m, o));
    }
    if (lane == 0) {
        most[0][warp] = m;
        most[1][warp] = q_m;
    }
    __syncthreads();
    for (int i = 0; i < warps; ++i) {
        m = fmaxf(m, most[0][i]);
        if (REFERENCE) q_m = fmaxf(q_m, most[1][i]);
    }
    float sum = total.sum();
    s.spread = spread.sum();
    s.apart = apart.sum();
    s.q_total = q_total.sum();
    if (sum != 0.0f) {
        const float gap = gap_of(s.m, m), f = power_of_two(gap);
        s.spread = f == 0.0f ? 0.0f : f * fmaf(gap, sum, s.spread);
        if (REFERENCE) s.apart = f == 0.0f ? 0.0f : f * fmaf(gap + back_of(s.q_m, q_m), sum, s.apart);
        sum *= f;
    }
    if (REFERENCE && s.q_total != 0.0) s.q_total *= power_of_two(gap_of(s.q_m, q_m));
    s.m = m;
    s.q_m = q_m;
    s.total = sum;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        s.total += __shfl_xor_sync(0xffffffffu, s.total, o);
        s.spread += __shfl_xor_sync(0xffffffffu, s.spread, o);
        if (REFERENCE) {
            s.q_total += __shfl_xor_sync(0xffffffffu, s.q_total, o);
            s.apart += __shfl_xor_sync(0xffffffffu, s.apart, o);
        }
    }
    if (lane == 0) {
        totals[0][warp] = s.total;
        totals[1][warp] = s.q_total;
        sums[0][warp] = s.spread;
        sums[1][warp] = s.apart;
    }
    __syncthreads();
    s.total = s.q_total = 0.0;
    s.spread = s.apart = 0.0f;
    for (int i = 0; i < warps; ++i) {
        s.total += totals[0][i];
        s.q_total += totals[1][i];
        s.spread += sums[0][i];
        s.apart += sums[1][i];
    }
    const Slopes k = finish(a, row, scalars, chosen, s, threadIdx.x == 0);
    if (g == nullptr) return;
    const Two off(-s.m, -s.m), q_off(-s.q_m, -s.q_m);
    const Two of_t(k.of_t, k.of_t), base(k.base, k.base), of_apart(k.of_apart, k.of_apart), part(k.scale, k.scale);
    auto leave = [&](auto count, int e) {
        constexpr int COUNT = decltype(count)::value, H = (COUNT + 1) / 2;
        const uint32_t bits = MASKED ? legal_bits<COUNT>(a, row, e) : 0;
        Two x[H], y[H];
        masked(count, z, e, bits, x);
        if (REFERENCE) masked(count, q, e, bits, y);
        float out[2 * H];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float2 f = multiply_add(x[i] + off, scale, unbiased).get();
            const Two t(max_nan(f.x, kNever), max_nan(f.y, kNever)), p = powers_of_two(t);
            Two inner = multiply_add(of_t, t, base);
            if (REFERENCE) {
                const float2 d = multiply_add(multiply_add(y[i] + q_off, scale, unbiased), Two(-1.0f, -1.0f), t).get(), w = p.get();
                inner = multiply_add(of_apart, Two(w.x != 0.0f ? d.x : 0.0f, w.y != 0.0f ? d.y : 0.0f), inner);
            }
            const float2 d = (p * part * inner).get();
            out[2 * i] = d.x;
            out[2 * i + 1] = d.y;
        }
        float kept[COUNT];
#pragma unroll
        for (int i = 0; i < COUNT; ++i) kept[i] = out[i];
        add_chosen<COUNT>(kept, e, action, k.slope);
        store_pack<T, COUNT>(g + e, kept);
    };
#pragma unroll 4
    for (int e = threadIdx.x * V; e < whole; e += step) leave(Constant<V>{}, e);
    for (int e = whole + threadIdx.x; e < a.n; e += blockDim.x) leave(Constant<1>{}, e);
    if constexpr (MASKED) {
        if (k.finite()) return;
        for (int e = threadIdx.x * V; e < whole; e += step) clear_masked<T, V>(a, row, g, e);
        for (int e = whole + threadIdx.x; e < a.n; e += blockDim.x) clear_masked<T, 1>(a, row, g, e);
    }
}

// ------------------------------------------------------------------ dispatch
template <typename T, int V, bool REFERENCE, int LANES, int HELD>
void launch_short(const Loss& a, cudaStream_t stream) {
    launch_chain("k_policy_loss", k_policy_loss<T, V, LANES, HELD, REFERENCE>, blocks(a.rows, 32 * kWarps / LANES), 32 * kWarps, 0, stream, true, a);
}
template <typename T, int V, bool REFERENCE>
void launch_loss(const Loss& a, cudaStream_t stream) {
    if (a.n <= kMostShort && a.n % V == 0) {
        // as few lanes as hold the row, and as few logits a lane, in steps of 8
        const int lanes = a.n <= 8 * kMostHeld ? 8 : a.n <= 16 * kMostHeld ? 16 : 32;
        const int held = static_cast<int>(round_up((a.n + lanes - 1) / lanes, 8));
        if (lanes == 8 && held <= 8) return launch_short<T, V, REFERENCE, 8, 8>(a, stream);
        if (lanes == 8 && held <= 16) return launch_short<T, V, REFERENCE, 8, 16>(a, stream);
        if (lanes == 8 && held <= 24) return launch_short<T, V, REFERENCE, 8, 24>(a, stream);
        if (lanes == 8) return launch_short<T, V, REFERENCE, 8, 32>(a, stream);
        if (lanes == 16 && held <= 24) return launch_short<T, V, REFERENCE, 16, 24>(a, stream);
        if (lanes == 16) return launch_short<T, V, REFERENCE, 16, 32>(a, stream);
        if (held <= 24) return launch_short<T, V, REFERENCE, 32, 24>(a, stream);
        return launch_short<T, V, REFERENCE, 32, 32>(a, stream);
    }
    const int threads = a.n <= 4096 ? 128 : kMostThreads;
    auto kernel = a.mask_kind ? k_policy_loss_long<T, V, REFERENCE, true> : k_policy_loss_long<T, V, REFERENCE, false>;
    launch_chain("k_policy_loss_long", kernel, static_cast<unsigned>(a.rows), threads, 0, stream, true, a);
}

}  // namespace
}  // namespace op
}  // namespace t8b

using namespace t8b;
using namespace t8b::op;

extern "C" int t8b_policy_loss(const t8b_policy_loss_t* call, float* loss, float* log_probabilities, float* entropies, float* divergences,
                               void* dlogits, int64_t dlogits_stride, void* stream) {
    return guarded([&] {
        if (call == nullptr) raise(T8B_EINVAL, "policy loss: the call is null");
        const t8b_policy_loss_t& c = *call;
        if (!is_type(c.type)) raise(T8B_EINVAL, "policy loss: unknown type");
        if (c.mask_kind < T8B_MASK_NONE || c.mask_kind > T8B_MASK_BYTES) raise(T8B_EINVAL, "policy loss: unknown kind of mask");
        if (c.reference_kind < T8B_REFERENCE_NONE || c.reference_kind > T8B_REFERENCE_SAMPLED) {
            raise(T8B_EINVAL, "policy loss: unknown kind of reference");
        }
        for (float v : {c.clip_low, c.clip_high}) {
            if (!(v >= 0.0f) || v > std::numeric_limits<float>::max()) raise(T8B_EINVAL, "policy loss: the clipped range must be finite and not negative");
        }
        for (float v : {c.kl, c.entropy}) {
            if (!(std::abs(v) <= std::numeric_limits<float>::max())) raise(T8B_EINVAL, "policy loss: the coefficients must be finite");
        }
        if (c.rows < 0 || c.rows > std::numeric_limits<int32_t>::max()) raise(T8B_EINVAL, "policy loss: 0 to 2^31 - 1 rows");
        if (c.n < 1 || c.n > (1 << 24)) raise(T8B_EINVAL, "policy loss: 1 to 2^24 logits a row");
        const size_t size = type_size(c.type);
        const int64_t words = c.mask_kind == T8B_MASK_BITS ? (c.n + 31) / 32 : c.n;
        const size_t word = c.mask_kind == T8B_MASK_BITS ? 4 : 1;
        check_matrix("policy loss logits", c.logits, c.rows, c.n, c.logits_stride, size);
        if (dlogits) check_matrix("policy loss dlogits", dlogits, c.rows, c.n, dlogits_stride, size);
        if (c.mask_kind) check_matrix("policy loss mask", c.mask, c.rows, words, c.mask_stride, word);
        if (c.reference_kind == T8B_REFERENCE_LOGITS) check_matrix("policy loss reference", c.reference, c.rows, c.n, c.reference_stride, size);
        if (c.reference_kind == T8B_REFERENCE_SAMPLED) check_matrix("policy loss reference", c.reference, 1, c.rows, c.rows, sizeof(float));
        check_elements("policy loss actions", c.actions, sizeof(int64_t));
        for (const float* p : {c.old_log_probabilities, c.advantages, c.weights, static_cast<const float*>(loss),
                               static_cast<const float*>(log_probabilities), static_cast<const float*>(entropies), static_cast<const float*>(divergences)}) {
            check_elements("policy loss", p, sizeof(float));
        }
        if (c.rows == 0) return;
        if (c.actions == nullptr || c.old_log_probabilities == nullptr || c.advantages == nullptr) {
            raise(T8B_EINVAL, "policy loss: actions, old log-probabilities or advantages are null");
        }
        Overlaps o{"policy loss"};
        o.input(Span(c.logits, c.rows, c.n, c.logits_stride, size));
        if (c.mask_kind) o.input(Span(c.mask, c.rows, words, c.mask_stride, word));
        if (c.reference_kind == T8B_REFERENCE_LOGITS) o.input(Span(c.reference, c.rows, c.n, c.reference_stride, size));
        if (c.reference_kind == T8B_REFERENCE_SAMPLED) o.input(span_of(c.reference, c.rows, sizeof(float)));
        o.input(span_of(c.actions, c.rows, sizeof(int64_t)));
        for (const float* p : {c.old_log_probabilities, c.advantages, c.weights}) o.input(span_of(p, c.rows, sizeof(float)));
        for (float* p : {loss, log_probabilities, entropies, divergences}) o.output(span_of(p, c.rows, sizeof(float)));
        if (dlogits) o.output(Span(dlogits, c.rows, c.n, dlogits_stride, size));
        Loss a{};
        a.logits = c.logits;
        a.reference = c.reference;
        a.mask = c.mask;
        a.actions = c.actions;
        a.old = c.old_log_probabilities;
        a.advantages = c.advantages;
        a.weights = c.weights;
        a.loss = loss;
        a.log_probabilities = log_probabilities;
        a.entropies = entropies;
        a.divergences = divergences;
        a.gradient = dlogits;
        a.logits_stride = c.logits_stride;
        a.reference_stride = c.reference_stride;
        a.mask_stride = c.mask_stride;
        a.gradient_stride = dlogits_stride;
        a.rows = c.rows;
        a.n = static_cast<int>(c.n);
        a.mask_kind = c.mask_kind;
        a.reference_kind = c.reference_kind;
        a.low = 1.0f - c.clip_low;
        a.high = 1.0f + c.clip_high;
        a.kl = c.kl;
        a.entropy = c.entropy;
        a.even = 1.0f / static_cast<float>(c.rows);
        const bool reference = c.reference_kind == T8B_REFERENCE_LOGITS;
        auto rows_on_packs = [&](const void* data, int64_t stride) { return aligned(data, 16) && (c.rows == 1 || stride * size % 16 == 0); };
        // 16 bytes a lane where every row starts on 16 bytes, single logits otherwise
        const bool wide = rows_on_packs(c.logits, c.logits_stride) && (!reference || rows_on_packs(c.reference, c.reference_stride)) &&
            (!dlogits || rows_on_packs(dlogits, dlogits_stride));
        with_type(c.type, [&](auto element) {
            using T = decltype(element);
            constexpr int V = 16 / sizeof(T);
            cudaStream_t st = static_cast<cudaStream_t>(stream);
            if (wide) {
                reference ? launch_loss<T, V, true>(a, st) : launch_loss<T, V, false>(a, st);
            } else {
                reference ? launch_loss<T, 1, true>(a, st) : launch_loss<T, 1, false>(a, st);
            }
        });
        check(cudaGetLastError(), "policy loss launch");
    });
}
