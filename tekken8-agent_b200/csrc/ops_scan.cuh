// Selective state space scan, forward and backward, over sequences with resets and lengths.
//
//   h_t = exp(D_t a) h_(t-1) + D_t u_t B_t,   s_t = sum_n C_t[n] h_t[n] + d u_t,   y_t = s_t silu(z_t)
//   D_t = softplus(delta_t + bias), or without it
// and with gs = dy silu(z), e_t = exp(D_t a), g_t = C_t gs_t + e_(t+1) g_(t+1) (the gradient of h_t):
//   dC = sum_c gs h,   dB = sum_c D u g,   du = d gs + D sum_n B g,   dz = dy s silu'(z),
//   dD = u sum_n B g + sum_n a e h_(t-1) g,   da = sum_t D e h_(t-1) g
// At a reset e_t is 0, whatever h_(t-1) is.
//
// Forward: LN lanes share a channel and hold 16 of its states each in registers, a block 128 / LN channels
// that one group of B and C serves; rows and B and C of 8 steps at a time lie in shared memory, the next ones on
// their way. Per (step, channel, state) one 2^x and four multiplications or additions, two of a kind to an
// instruction; per (step, channel) three more results of the 2^x unit, whose 16 a clock and SM bound the pass
// rather than memory: 65,536 x 1,024 x 16 in bf16 465 us, 284 by that unit, 93 by the bytes.
// Backward: each thread holds a tile of 2 channels x 4 states and goes through half of 8 steps forward,
// from what the forward pass kept (the state before every eighth step), its states in registers, then back; the later half
// first. Sums over states and over channels leave the threads as partial sums in shared memory and are added up there by
// 16 bytes a thread. 65,536 x 1,024 x 16 in bf16 1,700 us: some 230 instructions for a warp's step of 256 (channel,
// state) pairs, at 60 % of the issue slots with 16 warps an SM; with a whole tile's states in registers and 12 warps 1,755.
// Sequences are cut into chunks where there are too few of them: a first pass takes each
// chunk from a zero state, a second joins the chunks' ends, the last starts each where it belongs (1 x 8,192 x 1,024 x
// 16: 56, 18 and 74 us; 8 blocks would take it in one piece).
#pragma once

#include "ops_memory.cuh"

namespace t8b {
namespace op {
namespace scan {

constexpr int kThreads = 128;
constexpr int kTile = 8;  // steps between two kept states, and of a tile
constexpr int kHalf = 4;  // steps whose states a thread of the backward pass holds at once
constexpr int kSms = 148;
constexpr int kMostStates = 64;
constexpr int kHeld = 16;            // states of a channel that one of its threads holds

struct Call {
    Sequences q;
    Track<void> u, delta, z, b, c, y, dy;
    Track<void> du, ddelta, dz, db, dc;
    int64_t b_group, c_group, db_group, dc_group;
    const float *a, *d, *delta_bias, *state, *final_gradient;
    float* final_state;
    float* saved;    // [sequences][tiles][states][channels]: h before each tile
    float* dstate;
    // workspace
    float* carry;    // [sequences][chunks][states][channels]: a chunk's end from zero, then what it starts from
    float* sizes;    // [sequences][chunks][channels]: the sum of D over a chunk
    float* keep;     // [sequences][chunks]: 0 where a chunk has a reset
    float* shared;   // [blocks of a group][groups][sequences][steps][2][states]: sums of dB and dC
    float* partial;  // [workers][states + 2][channels]: sums of da, dd and ddelta_bias
    int groups, per, states, softplus;  // per: channels of a group
    int wide, paired, saved_paired;     // whether a row may be accessed by 16 bytes; by neighbouring channels
    int chunks, chunk;                  // a chunk's steps, a multiple of kTile
    int group_blocks, workers;
    int splits;                         // blocks of a group in a single step
};

// ------------------------------------------------------------------ arithmetic
__device__ __forceinline__ Two both(float v) { return Two(v, v); }
__device__ __forceinline__ Two two(float2 v) { return Two(v.x, v.y); }
// The machine's 2^x is off by a bias too: over x in -0.25 ... 0 by -1.7e-8 to -2.6e-8 of the value in the mean (a million
// values of each range; 3e-8 at random), which a state that lasts for hundreds of steps gathers. Decays are
// taken of an argument that is longer by what makes up for it, at no cost: the product with the rate becomes a
// multiply-add.
constexpr float kUnbiased = 3.2e-8f;
__device__ __forceinline__ float decay(float size, float rate) { return power_of_two(fmaf(size, rate, kUnbiased)); }
__device__ __forceinline__ Two powers_of_two(const Two& v) {
    const float2 f = v.get();
    return Two(power_of_two(f.x), power_of_two(f.y));
}
__device__ __forceinline__ Two decay(const Two& size, const Two& rate) { return powers_of_two(multiply_add(size, rate, both(kUnbiased))); }
// log(1 + x), 0 <= x <= 1: x + x^2 p(x), p fitted for the least relative error (2^-27.5, one coefficient after the other
// rounded to fp32 and the rest fitted again). In fp32 arithmetic at most 1.1e-7 off, within 6e-10 in the mean.
__device__ __forceinline__ float log_one_plus(float x) {
    float p = fmaf(-3.2904686e-3f, x, 2.0086242e-2f);
    p = fmaf(p, x, -5.7457231e-2f);
    p = fmaf(p, x, 0.10661128f);
    p = fmaf(p, x, -0.15344881f);
    p = fmaf(p, x, 0.19692102f);
    p = fmaf(p, x, -0.24958019f);
    p = fmaf(p, x, 0.33330464f);
    p = fmaf(p, x, -0.49999931f);
    return fmaf(x * x, p, x);
}
// softplus(v) = max(v, 0) + log(1 + exp(-|v|)), and its slope sigmoid(v)
__device__ __forceinline__ float softplus(float v) {
    return log_one_plus(exponential(-fabsf(v))) + (v > 0.0f ? v : 0.0f);
}
__device__ __forceinline__ float softplus(float v, float& slope) {
    const float x = exponential(-fabsf(v)), r = reciprocal(1.0f + x);
    slope = v > 0.0f ? r : x * r;
    return log_one_plus(x) + (v > 0.0f ? v : 0.0f);
}

// Which of a tile's steps are resets, one bit each: the same in every lane of a warp.
__device__ __forceinline__ unsigned reset_bits(const Sequences& q, int64_t s, int t0, int end) {
    if (q.reset == nullptr) return 0;
    const int t = t0 + static_cast<int>(threadIdx.x & 7);
    return __ballot_sync(0xffffffffu, t < end && q.resets(s, t)) & 0xffu;
}

// ------------------------------------------------------------------ forward
// Where a block stands: block = (s * chunks + chunk) * (blocks of all groups) + group * group_blocks + part.
struct Place {
    int64_t s;
    int chunk, group, part;
    __device__ __forceinline__ Place(const Call& a, int64_t block) {
        const int per_chunk = a.groups * a.group_blocks;
        const int64_t at = block / per_chunk;
        const int rest = static_cast<int>(block - at * per_chunk);
        group = rest / a.group_blocks;
        part = rest - group * a.group_blocks;
        s = at / a.chunks;
        chunk = static_cast<int>(at - s * a.chunks);
    }
};
__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }

// A thread has kHeld states of a channel; LN lanes share a channel, a block the channels that one group of
// B and C serves. A tile's rows come into shared memory 16 bytes at a time while the one before is worked on,
// and y leaves the same way; where rows do not start on 16 bytes (a.wide 0), element by element.
// ENDS: a chunk's end from a zero state, the sum of its D, and whether a reset cuts it, in place of y.
template <typename T, int LN, bool ENDS>
__global__ void __launch_bounds__(kThreads, 5) k_scan_forward(Call a) {
    constexpr int NP = kHeld * LN, CB = kThreads / LN;
    constexpr int V = 16 / sizeof(T), PACKS = CB / V;  // of a row
    wait_previous();
    release_next();
    __shared__ __align__(16) float bc[2][kTile][2][NP];
    __shared__ __align__(16) T rows[2][3][kTile][CB];  // u, delta, z
    __shared__ __align__(16) T ys[2][kTile][CB];
    const Sequences& q = a.q;
    const Place place(a, blockIdx.x);
    const int64_t s = place.s;
    const int lane = threadIdx.x % LN, column = threadIdx.x / LN, base = place.part * CB;
    const int width = min(CB, a.per - base);  // channels of this block
    const bool mine = column < width;
    const int c = place.group * a.per + base + (mine ? column : 0);
    const int t0 = place.chunk * a.chunk, t1 = min(q.steps, t0 + a.chunk), last = q.live(s), end = min(t1, last);
    const int n0 = lane * kHeld, channels = q.channels;
    const bool gate = !ENDS && a.z.data != nullptr;
    const int64_t at_chunk = s * a.chunks + place.chunk;
    auto row_of = [&](const Track<void>& track, int t) {
        return static_cast<T*>(track.data) + s * track.sequence + t * track.step + (place.group * a.per + base);
    };

    Two rate[kHeld / 2], h[kHeld / 2];  // a log2 e, and the states
#pragma unroll
    for (int i = 0; i < kHeld; i += 2) {
        float r[2] = {0.0f, 0.0f}, from[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = n0 + i + j;
            if (n >= a.states) continue;
            r[j] = a.a[static_cast<int64_t>(c) * a.states + n] * kLog2E;
            if (r[j] == -INFINITY) r[j] = -3.402823466e38f;  // (a reset's size of 0 makes 1 of it, not NaN)
            if (!ENDS && a.chunks > 1) {
                from[j] = a.carry[(at_chunk * a.states + n) * channels + c];
            } else if (!ENDS && a.state) {
                from[j] = a.state[(s * channels + c) * a.states + n];
            }
        }
        rate[i / 2] = Two(r[0], r[1]);
        h[i / 2] = Two(from[0], from[1]);
    }
    const float skip = a.d ? a.d[c] : 0.0f, bias = a.delta_bias ? a.delta_bias[c] : 0.0f;

    constexpr int PER = 2 * kTile * NP / kThreads;
    T raw_bc[PER];
    bool flag = false;  // whether the next tile's step threadIdx % 8 is a reset
    auto fetch = [&](int t, int buffer) {
        if (a.wide) {
            auto copy = [&](int k, const Track<void>& track) {
                for (int e = threadIdx.x; e < kTile * PACKS; e += kThreads) {
                    const int i = e / PACKS, at = e % PACKS * V;
                    if (t + i < end && at < width) copy_async<16>(&rows[buffer][k][i][at], row_of(track, t + i) + at);
                }
            };
            copy(0, a.u);
            copy(1, a.delta);
            if (gate) copy(2, a.z);
        } else if (mine) {
            for (int i = lane; i < kTile; i += LN) {
                if (t + i >= end) break;
                rows[buffer][0][i][column] = row_of(a.u, t + i)[column];
                rows[buffer][1][i][column] = row_of(a.delta, t + i)[column];
                if (gate) rows[buffer][2][i][column] = row_of(a.z, t + i)[column];
            }
        }
        copies_commit();
        const T* b = static_cast<const T*>(a.b.data) + s * a.b.sequence + place.group * a.b_group;
        const T* cc = static_cast<const T*>(a.c.data) + s * a.c.sequence + place.group * a.c_group;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = i * kThreads + threadIdx.x, step = e / (2 * NP), which = e / NP % 2, n = e % NP;
            raw_bc[i] = Element<T>::store(0.0f);
            if (t + step < end && n < a.states) raw_bc[i] = which ? cc[(t + step) * a.c.step + n] : b[(t + step) * a.b.step + n];
        }
        const int at = t + static_cast<int>(threadIdx.x & 7);
        flag = at < end && q.resets(s, at);
    };
    auto leave = [&](int t, int buffer) {  // a finished tile's y
        if constexpr (!ENDS) {
            if (!a.wide) return;
            for (int e = threadIdx.x; e < kTile * PACKS; e += kThreads) {
                const int i = e / PACKS, at = e % PACKS * V;
                if (t + i < end && at < width) {
                    store_held<T, V>(row_of(a.y, t + i) + at, load_held<T, V>(&ys[buffer][i][at]));
                }
            }
        }
    };
    int buffer = 0;
    float total = 0.0f;
    bool cut = false;
    if (t0 < end) fetch(t0, 0);
    for (int t = t0; t < end; t += kTile, buffer ^= 1) {
#pragma unroll
        for (int i = 0; i < PER; ++i) (&bc[buffer][0][0][0])[i * kThreads + threadIdx.x] = Element<T>::load(raw_bc[i]);
        copies_wait<0>();
        const unsigned resets = q.reset ? __ballot_sync(0xffffffffu, flag) & 0xffu : 0u;
        __syncthreads();  // this tile is there, and every thread is done with the one before
        if (t + kTile < end) fetch(t + kTile, buffer ^ 1);
        if (t > t0) leave(t - kTile, buffer ^ 1);
        if (!ENDS && a.saved && mine) {
            float* to = a.saved + ((s * ((q.steps + kTile - 1) / kTile) + t / kTile) * a.states + n0) * channels + c;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (n0 + i < a.states) *to = i % 2 ? h[i / 2].get().y : h[i / 2].get().x;
                to += channels;
            }
        }
        // a step's D, D u, u and gate; and the states' part of it
        struct Step {
            float size, in, u, gate;
        };
        auto elementwise = [&](int i) {
            Step v;
            v.u = Element<T>::load(rows[buffer][0][i][column]);
            v.size = Element<T>::load(rows[buffer][1][i][column]) + bias;
            if (a.softplus) v.size = softplus(v.size);
            v.in = v.size * v.u;
            if (resets >> i & 1) v.size = 0.0f;  // its decay of nothing is 1: its own may be infinite, and 0 of that NaN
            v.gate = gate ? silu(Element<T>::load(rows[buffer][2][i][column])) : 1.0f;
            return v;
        };
        auto advance = [&](int i, const Step& v) {
            Two out;
            const Two by = both(v.size), in = both(v.in);
#pragma unroll
            for (int n = 0; n < kHeld; n += 4) {
                const Pack<float, 4> b = *reinterpret_cast<const Pack<float, 4>*>(&bc[buffer][i][0][n0 + n]);
                const Pack<float, 4> c = ENDS ? b : *reinterpret_cast<const Pack<float, 4>*>(&bc[buffer][i][1][n0 + n]);
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    h[(n + j) / 2] = multiply_add(decay(by, rate[(n + j) / 2]), h[(n + j) / 2], in * Two(b.v[j], b.v[j + 1]));
                    out = multiply_add(h[(n + j) / 2], Two(c.v[j], c.v[j + 1]), out);
                }
            }
            if (ENDS) {
                total += v.size;
                return;
            }
            float sum = out.sum();
#pragma unroll
            for (int o = LN / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            sum = fmaf(skip, v.u, sum) * v.gate;
            if (lane != 0) return;
            if (a.wide) {
                ys[buffer][i][column] = Element<T>::store(sum);
            } else if (mine) {
                row_of(a.y, t + i)[column] = Element<T>::store(sum);
            }
        };
        auto begin = [&](int i) {
            if ((resets >> i & 1) == 0) return;
            cut = true;
            total = 0.0f;
#pragma unroll
            for (int n = 0; n < kHeld / 2; ++n) h[n] = Two();
        };
        if (t + kTile <= end) {
            // the next step's elementwise part, a chain of latencies, beside this one's states
            Step v = elementwise(0);
#pragma unroll
            for (int i = 0; i < kTile; ++i) {
                in_order();
                begin(i);
                const Step next = i + 1 < kTile ? elementwise(i + 1) : v;
                advance(i, v);
                v = next;
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < end - t; ++i) {
                begin(i);
                advance(i, elementwise(i));
            }
        }
    }
    if (!ENDS && t0 < end) {
        __syncthreads();
        leave(t0 + (end - 1 - t0) / kTile * kTile, buffer ^ 1);
    }
    if (!mine) return;
    if (ENDS) {
        float* to = a.carry + (at_chunk * a.states + n0) * channels + c;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (n0 + i < a.states) *to = i % 2 ? h[i / 2].get().y : h[i / 2].get().x;
            to += channels;
        }
        if (lane == 0) a.sizes[at_chunk * channels + c] = total;
        if (lane == 0 && base + column == 0 && place.group == 0) a.keep[at_chunk] = cut ? 0.0f : 1.0f;
        return;
    }
    if (lane == 0) {
        for (int t = max(t0, end); t < t1; ++t) row_of(a.y, t)[column] = Element<T>::store(0.0f);
    }
    if (a.final_state && (last > t0 ? last <= t1 : last == 0 && t0 == 0)) {
        float* to = a.final_state + (s * channels + c) * a.states + n0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (n0 + i < a.states) to[i] = i % 2 ? h[i / 2].get().y : h[i / 2].get().x;
        }
    }
}

// The cube root of 2^x, as which a chunk's decay is multiplied: 2^x alone may have no place in fp32 where its product with
// the state has one. Over negative sizes x passes 128 while the state is 0 (infinity times 0 is NaN) or small, and below
// -126 a large state still leaves something. 2^300 takes the least state to infinity, 2^-300 the largest to 0; NaN stays.
// (Three products a chunk in a row: 18 us for 1 x 8,192 x 1,024 x 16, 103 chunks; with ldexp() of the product 36.)
__device__ __forceinline__ float decay_root(float x) {
    const float third = x * (1.0f / 3.0f);
    return power_of_two((fabsf(third) > 100.0f ? copysignf(100.0f, third) : third) + kUnbiased);
}
// The chunks of a sequence in order (backward: in reverse): what each starts from takes the place of its
// own end. A thread has one state of one channel.
static __global__ void __launch_bounds__(256) k_scan_join(Call a, bool backward) {
    wait_previous();
    release_next();
    const int channels = a.q.channels;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t s = index / (static_cast<int64_t>(a.states) * channels);
    if (s >= a.q.sequences) return;
    const int rest = static_cast<int>(index - s * a.states * channels), n = rest / channels, c = rest - n * channels;
    const float rate = a.a[static_cast<int64_t>(c) * a.states + n] * kLog2E;
    const float* first = backward ? a.final_gradient : a.state;
    float h = first ? first[(s * channels + c) * a.states + n] : 0.0f;
    const int64_t apart = static_cast<int64_t>(a.states) * channels, from = s * a.chunks + (backward ? a.chunks - 1 : 0);
    const int64_t carry_step = backward ? -apart : apart, sizes_step = backward ? -channels : channels, keep_step = backward ? -1 : 1;
    float* carry = a.carry + from * apart + rest;
    const float *sizes = a.sizes + from * channels + c, *keep = a.keep + from;
    float* to = carry;
    constexpr int AHEAD = 8;
    struct Chunks {
        float ends[AHEAD], size[AHEAD], kept[AHEAD];
    };
    auto load = [&](int k) {
        Chunks v;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {  // past the last chunk it is read again: loads without branches wait together
            v.ends[i] = *carry;
            v.size[i] = *sizes;
            v.kept[i] = *keep;
            const bool more = k + i + 1 < a.chunks;
            carry += more ? carry_step : 0;
            sizes += more ? sizes_step : 0;
            keep += more ? keep_step : 0;
        }
        return v;
    };
    Chunks next = load(0);
    for (int k = 0; k < a.chunks; k += AHEAD) {
        const Chunks now = next;
        next = load(k + AHEAD);
        float root[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) root[i] = decay_root(rate * now.size[i]);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (k + i >= a.chunks) break;
            *to = h;
            to += carry_step;
            h = now.kept[i] != 0.0f ? fmaf(root[i], root[i] * (root[i] * h), now.ends[i]) : now.ends[i];
        }
    }
}

// ------------------------------------------------------------------ backward
// What a chunk adds to the gradient of the state before it, the sum of its D, and whether a reset cuts it.
template <typename T, int NS, int LN>
__global__ void __launch_bounds__(kThreads) k_scan_back_ends(Call a) {
    constexpr int NP = NS * LN, CB = kThreads / LN;
    wait_previous();
    release_next();
    __shared__ __align__(16) float vc[kTile][NP];
    const Sequences& q = a.q;
    const Place place(a, blockIdx.x);
    const int64_t s = place.s;
    const int lane = threadIdx.x % LN, local = place.part * CB + threadIdx.x / LN;
    const bool mine = local < a.per;
    const int c = place.group * a.per + (mine ? local : 0);
    const int t0 = place.chunk * a.chunk, t1 = min(q.steps, t0 + a.chunk), end = min(t1, q.live(s));
    const int n0 = lane * NS, channels = q.channels;
    const T* delta = static_cast<const T*>(a.delta.data) + s * a.delta.sequence + c;
    const T* z = a.z.data ? static_cast<const T*>(a.z.data) + s * a.z.sequence + c : nullptr;
    const T* dy = static_cast<const T*>(a.dy.data) + s * a.dy.sequence + c;
    const T* cc = static_cast<const T*>(a.c.data) + s * a.c.sequence + place.group * a.c_group;
    Two rate[NS / 2], g[NS / 2];
#pragma unroll
    for (int i = 0; i < NS / 2; ++i) {
        float2 r = make_float2(0.0f, 0.0f);
        if (n0 + 2 * i < a.states) r.x = a.a[static_cast<int64_t>(c) * a.states + n0 + 2 * i] * kLog2E;
        if (n0 + 2 * i + 1 < a.states) r.y = a.a[static_cast<int64_t>(c) * a.states + n0 + 2 * i + 1] * kLog2E;
        rate[i] = two(r);
    }
    const float bias = a.delta_bias ? a.delta_bias[c] : 0.0f;
    float total = 0.0f;
    bool cut = false;
    for (int t = t0 + (end - 1 - t0) / kTile * kTile; end > t0 && t >= t0; t -= kTile) {
        float size[kTile], given[kTile];
#pragma unroll
        for (int i = 0; i < kTile; ++i) {
            const bool live = mine && t + i < end;
            const float v = live ? Element<T>::load(delta[(t + i) * a.delta.step]) + bias : 0.0f;
            given[i] = live ? Element<T>::load(dy[(t + i) * a.dy.step]) : 0.0f;
            if (z && live) {
                const float w = Element<T>::load(z[(t + i) * a.z.step]);
                given[i] *= w * sigmoid(w);
            }
            size[i] = live ? (a.softplus ? softplus(v) : v) : 0.0f;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < kTile * NP; e += kThreads) {
            const int step = e / NP, n = e % NP;
            vc[step][n] = t + step < end && n < a.states ? Element<T>::load(cc[(t + step) * a.c.step + n]) : 0.0f;
        }
        const unsigned resets = reset_bits(q, s, t, end);
        cut = cut || resets != 0;
        __syncthreads();
#pragma unroll
        for (int i = kTile - 1; i >= 0; --i) {
            const Two by = both(size[i]), in = both(given[i]);
            total += size[i];
#pragma unroll
            for (int k = 0; k < NS / 2; ++k) {
                const float2 w = *reinterpret_cast<const float2*>(&vc[i][n0 + 2 * k]);
                g[k] = multiply_add(in, two(w), g[k]) * decay(by, rate[k]);
            }
            if (resets >> i & 1) {
#pragma unroll
                for (int k = 0; k < NS / 2; ++k) g[k] = Two();
            }
        }
    }
    if (!mine) return;
    const int64_t at_chunk = s * a.chunks + place.chunk;
    float* to = a.carry + (at_chunk * a.states + n0) * channels + c;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const float2 v = g[i / 2].get();
        if (n0 + i < a.states) to[static_cast<int64_t>(i) * channels] = i % 2 ? v.y : v.x;
    }
    if (lane == 0) a.sizes[at_chunk * channels + c] = total;
    if (lane == 0 && local == 0 && place.group == 0) a.keep[at_chunk] = cut ? 0.0f : 1.0f;
}

// Shared memory of a block of the backward pass, for LN lanes along the states (4 each).
template <typename T, int LN>
struct Backward {
    static constexpr int NP = 4 * LN, LC = 32 / LN;          // states; lanes along the channels
    static constexpr int CB = (kThreads / 32) * LC * 2;      // channels of a block
    static constexpr int EV = kTile * CB / kThreads;         // channels of a thread's elementwise part: 4, 2 or 1
    static constexpr int PARTS = LC * (kThreads / 32);       // pairs of channels, and partial sums of a state
    static constexpr int SPLIT = kThreads / (kHalf * 2 * LN);  // threads that add up four states' partial sums
    // Where pair p's sums of lane `along` lie: rows are rotated, so that neither the threads that write
    // them nor those that add them up meet in a bank.
    __device__ __forceinline__ static int channel_at(int p, int along) { return (p + LC * along) % (CB / 2); }
    __device__ __forceinline__ static int state_at(int p, int along) { return (p + SPLIT * along) % PARTS; }
    struct Shared {
        Held<T, EV> rows[4][kThreads];                           // u, delta, dy and z of a tile: each thread writes and reads its own
        float2 before[4][kThreads];                              // the states before it: the same
        float size[kTile][CB], in[kTile][CB], given[kTile][CB];  // D, D u, gs
        float slope[kTile][CB], zslope[kTile][CB];               // softplus'(v), dy silu'(z)
        float bias[CB], skip[CB];
        float2 b[kTile][NP], c[kTile][NP];                       // each value twice: an operand of packed arithmetic
        // of half a tile
        float2 channel_sums[kHalf][3][LN][CB / 2];               // sum_n: C h, B g, a e h g, of each lane along the states
        float4 state_sums[kHalf][2][LN][PARTS];                  // sum_c: D u g, gs h, of each pair of channels
    };
};

// Four values that lie twice each.
__device__ __forceinline__ void twice(const float2* from, Two (&v)[4]) {
    const float4 x = reinterpret_cast<const float4*>(from)[0], y = reinterpret_cast<const float4*>(from)[1];
    v[0] = Two(x.x, x.y);
    v[1] = Two(x.z, x.w);
    v[2] = Two(y.x, y.y);
    v[3] = Two(y.z, y.w);
}

template <typename T, int LN>
__global__ void __launch_bounds__(kThreads, 4) k_scan_backward(Call a) {
    using Shape = Backward<T, LN>;
    constexpr int NP = Shape::NP, LC = Shape::LC, CB = Shape::CB, EV = Shape::EV, PARTS = Shape::PARTS;
    constexpr int ROW = CB / EV;  // threads of a row of the elementwise part: kThreads / ROW = kTile
    wait_previous();
    release_next();
    extern __shared__ __align__(16) unsigned char memory[];
    auto& m = *reinterpret_cast<typename Shape::Shared*>(memory);
    const Sequences& q = a.q;
    const int group = blockIdx.x / a.group_blocks, part = blockIdx.x - group * a.group_blocks;
    const int channels = q.channels, tiles = (q.steps + kTile - 1) / kTile;
    // this thread's tile: channels c0 and c0 + 1, states n0 to n0 + 3
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, across = lane % LC, along = lane / LC;
    const int pair = warp * LC + across, n0 = 4 * along;
    const int c0 = group * a.per + part * CB + 2 * pair;
    const bool has0 = part * CB + 2 * pair < a.per, has1 = part * CB + 2 * pair + 1 < a.per;
    // and its elementwise part: EV channels from ec on, step es of a tile
    const int el = threadIdx.x % ROW * EV, es = threadIdx.x / ROW;
    const int ecount = max(0, min(EV, a.per - part * CB - el));
    const int ec = group * a.per + (ecount > 0 ? part * CB + el : 0);

    Two rate[4], da[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        float2 r = make_float2(0.0f, 0.0f);
        if (n0 + n < a.states) {
            if (has0) r.x = a.a[static_cast<int64_t>(c0) * a.states + n0 + n] * kLog2E;
            if (has1) r.y = a.a[static_cast<int64_t>(c0 + 1) * a.states + n0 + n] * kLog2E;
        }
        rate[n] = two(r);
    }
    for (int i = threadIdx.x; i < CB; i += kThreads) {
        const bool in = part * CB + i < a.per;
        m.bias[i] = in && a.delta_bias ? a.delta_bias[group * a.per + part * CB + i] : 0.0f;
        m.skip[i] = in && a.d ? a.d[group * a.per + part * CB + i] : 0.0f;
    }
    __syncthreads();
    float dd[EV] = {}, dbias[EV] = {};
    float* partial = a.partial + static_cast<int64_t>(blockIdx.y) * (a.states + 2) * channels;
    // this worker's sums of da so far: kept apart from a few tiles' sums, which are added to them
    auto flush = [&](bool first) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float2 v = da[n].get();
            da[n] = Two();
            float* to = partial + static_cast<int64_t>(n0 + n) * channels + c0;
            if (n0 + n < a.states && has0) to[0] = first ? v.x : to[0] + v.x;
            if (n0 + n < a.states && has1) to[1] = first ? v.y : to[1] + v.y;
        }
    };
    bool first = true;

    constexpr int PER = (2 * kTile * NP + kThreads - 1) / kThreads;
    T raw_bc[PER];
    bool flag = false;  // whether the fetched tile's step threadIdx % 8 is a reset
    const bool gate = a.z.data != nullptr;
    const int64_t items = q.sequences * a.chunks;
    for (int64_t item = blockIdx.y; item < items; item += a.workers) {
        const int64_t s = item / a.chunks;
        const int chunk = static_cast<int>(item - s * a.chunks);
        const int t0 = chunk * a.chunk, t1 = min(q.steps, t0 + a.chunk), last = q.live(s), end = min(t1, last);
        auto row_of = [&](const Track<void>& track, int t) { return static_cast<const T*>(track.data) + s * track.sequence + t * track.step + ec; };
        auto fetch = [&](int t) {
            const int at = t + es;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k == 3 && !gate) continue;
                const Track<void>& track = k == 0 ? a.u : k == 1 ? a.delta : k == 2 ? a.dy : a.z;
                Held<T, EV>* to = &m.rows[k][threadIdx.x];
                if (at < end && ecount == EV && a.paired) {
                    const T* from = row_of(track, at);
                    if constexpr (EV * sizeof(T) >= 4) {
                        copy_async<EV * sizeof(T)>(to, from);
                    } else {
                        *to = load_held<T, EV>(from);
                    }
                } else {
                    const T* from = row_of(track, at < end ? at : 0);
#pragma unroll
                    for (int i = 0; i < EV; ++i) reinterpret_cast<T*>(to)[i] = at < end && i < ecount ? from[i] : Element<T>::store(0.0f);
                }
            }
            const T* b = static_cast<const T*>(a.b.data) + s * a.b.sequence + group * a.b_group;
            const T* cc = static_cast<const T*>(a.c.data) + s * a.c.sequence + group * a.c_group;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = i * kThreads + threadIdx.x, step = e / (2 * NP), which = e / NP % 2, n = e % NP;
                raw_bc[i] = Element<T>::store(0.0f);
                if (step < kTile && t + step < end && n < a.states) {
                    raw_bc[i] = which ? cc[(t + step) * a.c.step + n] : b[(t + step) * a.b.step + n];
                }
            }
        };
        auto fetch_flag = [&](int t) {
            const int at = t + static_cast<int>(threadIdx.x & 7);
            flag = at < end && q.resets(s, at);
        };
        auto fetch_before = [&](int t) {
            const float* from = a.saved + ((s * tiles + t / kTile) * a.states + n0) * channels + c0;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float2* to = &m.before[n][threadIdx.x];
                if (n0 + n < a.states && has1 && a.saved_paired) {
                    copy_async<8>(to, from);
                } else {
                    float2 v = make_float2(0.0f, 0.0f);
                    if (n0 + n < a.states && has0) v.x = from[0];
                    if (n0 + n < a.states && has1) v.y = from[1];
                    *to = v;
                }
                from += channels;
            }
            copies_commit();
        };
        // the gradient of the state after the chunk
        Two g[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            float2 v = make_float2(0.0f, 0.0f);
            if (n0 + n < a.states) {
                if (a.chunks > 1) {
                    const float* from = a.carry + (item * a.states + n0 + n) * channels + c0;
                    if (has0) v.x = from[0];
                    if (has1) v.y = from[1];
                } else if (a.final_gradient) {
                    const float* from = a.final_gradient + (s * channels + c0) * a.states + n0 + n;
                    if (has0) v.x = from[0];
                    if (has1) v.y = from[a.states];
                }
            }
            g[n] = two(v);
        }
        int t = t0 + (end - 1 - t0) / kTile * kTile, since = 0;
        if (end > t0) {
            fetch(t);
            fetch_flag(t);
            fetch_before(t);
        }
        for (; end > t0 && t >= t0; t -= kTile) {
            copies_wait<0>();
            // ---- elementwise: D, D u and gs of the tile into shared memory
            const Held<T, EV> raw_u = m.rows[0][threadIdx.x];
            {
                float slope[EV], zslope[EV];
                const bool live = t + es < end;
                float vu[EV], vdelta[EV], vdy[EV], vz[EV];
                unpack<T, EV>(raw_u, vu);
                unpack<T, EV>(m.rows[1][threadIdx.x], vdelta);
                unpack<T, EV>(m.rows[2][threadIdx.x], vdy);
                if (gate) unpack<T, EV>(m.rows[3][threadIdx.x], vz);
                float size[EV], in[EV], given[EV];
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    size[i] = vdelta[i] + m.bias[el + i];
                    slope[i] = 1.0f;
                    if (a.softplus) size[i] = softplus(size[i], slope[i]);
                    in[i] = size[i] * vu[i];
                }
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    given[i] = vdy[i];
                    zslope[i] = 0.0f;
                    if (gate) {
                        float value;
                        activate_slope<T8B_SILU>(vz[i], value, zslope[i]);
                        zslope[i] *= given[i];
                        given[i] *= value;
                    }
                    if (!live || i >= ecount) size[i] = in[i] = given[i] = 0.0f;
                }
                *reinterpret_cast<Held<float, EV>*>(&m.size[es][el]) = pack<float, EV>(size);
                *reinterpret_cast<Held<float, EV>*>(&m.in[es][el]) = pack<float, EV>(in);
                *reinterpret_cast<Held<float, EV>*>(&m.given[es][el]) = pack<float, EV>(given);
                *reinterpret_cast<Held<float, EV>*>(&m.slope[es][el]) = pack<float, EV>(slope);
                *reinterpret_cast<Held<float, EV>*>(&m.zslope[es][el]) = pack<float, EV>(zslope);
            }
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = i * kThreads + threadIdx.x, step = e / (2 * NP), which = e / NP % 2, n = e % NP;
                const float v = Element<T>::load(raw_bc[i]);
                if (step < kTile) (which ? m.c : m.b)[step][n] = make_float2(v, v);
            }
            const unsigned resets = q.reset ? __ballot_sync(0xffffffffu, flag) & 0xffu : 0u;
            __syncthreads();
            if (t > t0) {
                fetch(t - kTile);
                fetch_flag(t - kTile);
            }
            // ---- h through half a tile, then g back through it: the later half first. The state between the halves
            // is computed on the way, its way there again for the earlier half.
            Two between[4];
            auto state_of = [&](int i, const Two (&from)[4], Two (&to)[4]) {
                in_order();
                const Two by = two(*reinterpret_cast<const float2*>(&m.size[i][2 * pair]));
                const Two in = two(*reinterpret_cast<const float2*>(&m.in[i][2 * pair]));
                Two bn[4], e[4];
                twice(&m.b[i][n0], bn);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    bn[n] = in * bn[n];
                    e[n] = decay(by, rate[n]);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) to[n] = multiply_add(e[n], from[n], bn[n]);
                if (resets >> i & 1) {  // (a branch that all take alike: selects would cost as much as the products)
                    in_order();
#pragma unroll
                    for (int n = 0; n < 4; ++n) to[n] = bn[n];
                }
            };
            auto before_tile = [&](Two (&h)[4]) {
#pragma unroll
                for (int n = 0; n < 4; ++n) h[n] = two(m.before[n][threadIdx.x]);
            };
            auto half = [&](auto which, auto&& between_passes) {
                constexpr int FIRST = decltype(which)::value * kHalf;
                Two h[kHalf][4];
                if (FIRST) {
                    state_of(FIRST, between, h[0]);
                } else {
                    before_tile(between);
                    state_of(0, between, h[0]);
                }
#pragma unroll
                for (int i = 1; i < kHalf; ++i) state_of(FIRST + i, h[i - 1], h[i]);
                between_passes();
#pragma unroll
                for (int k = kHalf - 1; k >= 0; --k) {
                    const int i = FIRST + k;
                    if (k % 2) in_order();
                    const Two by = two(*reinterpret_cast<const float2*>(&m.size[i][2 * pair]));
                    const Two in = two(*reinterpret_cast<const float2*>(&m.in[i][2 * pair]));
                    const Two given = two(*reinterpret_cast<const float2*>(&m.given[i][2 * pair]));
                    Two bn[4], cn[4];
                    twice(&m.b[i][n0], bn);
                    twice(&m.c[i][n0], cn);
                    Two of_h, of_b, of_a, e[4];
                        float db[4], dc[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        e[n] = decay(by, rate[n]);
                        g[n] = multiply_add(given, cn[n], g[n]);
                        of_h = multiply_add(h[k][n], cn[n], of_h);
                        of_b = multiply_add(g[n], bn[n], of_b);
                        db[n] = (in * g[n]).sum();
                        dc[n] = (given * h[k][n]).sum();
                    }
                    if (resets >> i & 1) {
                        in_order();
#pragma unroll
                        for (int n = 0; n < 4; ++n) g[n] = Two();
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const Two from = k ? h[k ? k - 1 : 0][n] : between[n];
                            g[n] = g[n] * e[n];
                            const Two through = g[n] * from;
                            of_a = multiply_add(through, rate[n], of_a);
                            da[n] = multiply_add(through, by, da[n]);
                        }
                    }
                    m.channel_sums[k][0][along][Shape::channel_at(pair, along)] = of_h.get();
                    m.channel_sums[k][1][along][Shape::channel_at(pair, along)] = of_b.get();
                    m.channel_sums[k][2][along][Shape::channel_at(pair, along)] = of_a.get();
                    m.state_sums[k][0][along][Shape::state_at(pair, along)] = make_float4(db[0], db[1], db[2], db[3]);
                    m.state_sums[k][1][along][Shape::state_at(pair, along)] = make_float4(dc[0], dc[1], dc[2], dc[3]);
                }
            };
            auto leave = [&](auto which) {
                constexpr int FIRST = decltype(which)::value * kHalf;
            // ---- the sums over states, and the gradients of u, delta and z
            if (es / kHalf == FIRST / kHalf) {
                const int at = t + es;
                float sum[3][EV] = {};
#pragma unroll
                for (int k = 0; k < 3; ++k) {
#pragma unroll
                    for (int l = 0; l < LN; ++l) {
                        const float* from = reinterpret_cast<const float*>(m.channel_sums[es % kHalf][k][l]) + 2 * Shape::channel_at(el / 2, l) + (EV == 1 ? el % 2 : 0);
                        float v[EV];
                        unpack<float, EV>(load_held<float, EV>(from), v);
#pragma unroll
                        for (int i = 0; i < EV; ++i) sum[k][i] += v[i];
                    }
                }
                if (ecount > 0 && at < t1) {
                    const bool live = at < end;
                    float size[EV], given[EV];
                    unpack<float, EV>(load_held<float, EV>(&m.size[es][el]), size);
                    unpack<float, EV>(load_held<float, EV>(&m.given[es][el]), given);
                    float slope[EV], zslope[EV];
                    unpack<float, EV>(load_held<float, EV>(&m.slope[es][el]), slope);
                    unpack<float, EV>(load_held<float, EV>(&m.zslope[es][el]), zslope);
                    float du[EV], ddelta[EV], dz[EV], of_u[EV];
                    unpack<T, EV>(raw_u, of_u);
#pragma unroll
                    for (int i = 0; i < EV; ++i) {
                        const float vu = of_u[i], skip = m.skip[el + i];
                        du[i] = live ? fmaf(skip, given[i], size[i] * sum[1][i]) : 0.0f;
                        ddelta[i] = live ? fmaf(kLn2, sum[2][i], vu * sum[1][i]) * slope[i] : 0.0f;
                        dz[i] = live ? zslope[i] * fmaf(skip, vu, sum[0][i]) : 0.0f;
                        dbias[i] += ddelta[i];
                        if (live) dd[i] = fmaf(given[i], vu, dd[i]);
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        if (k == 2 && !a.dz.data) continue;
                        const Track<void>& track = k == 0 ? a.du : k == 1 ? a.ddelta : a.dz;
                        T* to = const_cast<T*>(row_of(track, at));
                        const Held<T, EV> v = pack<T, EV>(k == 0 ? du : k == 1 ? ddelta : dz);
                        if (ecount == EV && a.paired) {
                            store_held<T, EV>(to, v);
                        } else {
#pragma unroll
                            for (int i = 0; i < EV; ++i) {
                                if (i < ecount) to[i] = reinterpret_cast<const T*>(&v)[i];
                            }
                        }
                    }
                }
            }
            // ---- the sums over channels: every thread has a part of four states'
            constexpr int SPLIT = Shape::SPLIT;
            const int quad = threadIdx.x / SPLIT, share = threadIdx.x % SPLIT, step = quad / (2 * LN), which_sum = quad / LN % 2, l = quad % LN;
            Two x, y;
#pragma unroll
            for (int p = 0; p < PARTS; p += SPLIT) {
                const float4 v = m.state_sums[step][which_sum][l][Shape::state_at(p + share, l)];
                x = x + Two(v.x, v.y);
                y = y + Two(v.z, v.w);
            }
            float2 vx = x.get(), vy = y.get();
#pragma unroll
            for (int o = SPLIT / 2; o >= 1; o >>= 1) {
                vx.x += __shfl_xor_sync(0xffffffffu, vx.x, o);
                vx.y += __shfl_xor_sync(0xffffffffu, vx.y, o);
                vy.x += __shfl_xor_sync(0xffffffffu, vy.x, o);
                vy.y += __shfl_xor_sync(0xffffffffu, vy.y, o);
            }
            if (share == 0 && t + FIRST + step < end && 4 * l < a.states) {
                const float sum[4] = {vx.x, vx.y, vy.x, vy.y};
                float* to = a.shared +
                    ((((static_cast<int64_t>(part) * a.groups + group) * q.sequences + s) * q.steps + t + FIRST + step) * 2 + which_sum) * a.states + 4 * l;
                if (a.states % 4 == 0) {  // the workspace starts on 256 bytes
                    *reinterpret_cast<float4*>(to) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                } else {
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        if (4 * l + n < a.states) to[n] = sum[n];
                    }
                }
            }
            };
            before_tile(between);
#pragma unroll
            for (int i = 0; i < kHalf; ++i) state_of(i, between, between);
            half(Constant<1>{}, [] {});
            __syncthreads();
            leave(Constant<1>{});
            half(Constant<0>{}, [] { __syncthreads(); });  // (what the later half left is read)
            if (t > t0) fetch_before(t - kTile);
            if (++since == 16 || t == t0) {
                flush(first);
                first = false;
                since = 0;
            }
            __syncthreads();
            leave(Constant<0>{});
        }
        // past the sequence's end
        for (int at = t0 + (end > t0 ? (end - t0 + kTile - 1) / kTile * kTile : 0) + es; at < t1; at += kTile) {
            for (int k = 0; k < 3; ++k) {
                if (k == 2 && !a.dz.data) continue;
                T* to = const_cast<T*>(row_of(k == 0 ? a.du : k == 1 ? a.ddelta : a.dz, at));
                for (int i = 0; i < ecount; ++i) to[i] = Element<T>::store(0.0f);
            }
        }
        if (chunk == 0 && a.dstate) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float2 v = g[n].get();
                float* to = a.dstate + (s * channels + c0) * a.states + n0 + n;
                if (n0 + n < a.states && has0) to[0] = v.x;
                if (n0 + n < a.states && has1) to[a.states] = v.y;
            }
        }
        __syncthreads();  // the next item's tile writes what this one's last still reads
    }
    if (first) flush(true);  // no step at all: zeros
    // the rows of threads, one step of a tile each, in their order
#pragma unroll
    for (int i = 0; i < EV; ++i) {
        m.size[es][el + i] = dd[i];
        m.in[es][el + i] = dbias[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < CB; i += kThreads) {
        if (part * CB + i >= a.per) continue;
        float of_d = 0.0f, of_bias = 0.0f;
#pragma unroll
        for (int r = 0; r < kTile; ++r) {
            of_d += m.size[r][i];
            of_bias += m.in[r][i];
        }
        const int c = group * a.per + part * CB + i;
        partial[static_cast<int64_t>(a.states) * channels + c] = of_d;
        partial[static_cast<int64_t>(a.states + 1) * channels + c] = of_bias;
    }
}

// da, dd and ddelta_bias from the workers' sums. Block (32, 16): 32 of the (states + 2) channels columns.
static __global__ void k_scan_parameters(Call a, float* da, float* dd, float* dbias) {
    wait_previous();
    release_next();
    __shared__ float sums[16][33];
    const int channels = a.q.channels;
    const int64_t columns = static_cast<int64_t>(a.states + 2) * channels, column = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
    float v = 0.0f;
    if (column < columns) {
#pragma unroll 4
        for (int r = threadIdx.y; r < a.workers; r += 16) v += a.partial[r * columns + column];
    }
    sums[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y != 0 || column >= columns) return;
#pragma unroll
    for (int r = 1; r < 16; ++r) v += sums[r][threadIdx.x];
    const int n = static_cast<int>(column / channels), c = static_cast<int>(column - static_cast<int64_t>(n) * channels);
    if (n < a.states) {
        da[static_cast<int64_t>(c) * a.states + n] = v;
    } else if (n == a.states) {
        if (dd) dd[c] = v;
    } else if (dbias) {
        dbias[c] = v;
    }
}

// dB and dC from the blocks' sums: one thread a (sequence, step, group, b or c, state).
template <typename T>
__global__ void __launch_bounds__(256) k_scan_shared(Call a) {
    wait_previous();
    release_next();
    const Sequences& q = a.q;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int width = 2 * a.states;
    const int64_t row = index / width;  // (group, sequence, step)
    const int e = static_cast<int>(index - row * width);
    const int64_t rows = q.sequences * q.steps;
    if (row >= rows * a.groups) return;
    const int group = static_cast<int>(row / rows);
    const int64_t at = row - group * rows, s = at / q.steps;
    const int t = static_cast<int>(at - s * q.steps), which = e / a.states, n = e - which * a.states;
    float v = 0.0f;
    if (t < q.live(s)) {
        const int64_t apart = a.groups * rows * width;
        for (int p = 0; p < a.group_blocks; ++p) v += a.shared[p * apart + index];
    }
    T* to = which ? static_cast<T*>(a.dc.data) + s * a.dc.sequence + t * a.dc.step + group * a.dc_group
                  : static_cast<T*>(a.db.data) + s * a.db.sequence + t * a.db.step + group * a.db_group;
    to[n] = Element<T>::store(v);
}

// ------------------------------------------------------------------ a single step
// LP lanes (a power of two) share a channel and hold V consecutive states of it each; a block takes kStepAhead
// sequences and goes through the channels of one group, a tile of kStepThreads / LP of them at a time, with the
// sequences' B and C in shared memory. Bound by the states' bytes, read once and written once: a thread has its
// channel's states of every sequence in flight together. Lane l of a channel does the elementwise part of the
// sequences l, l + LP, ... and gives D and D u to the others; the sums over its lanes end where they are used.
// 32,768 x 512 x 16 in bf16: 420 us, 83 % of the copy rate (every lane with its own elementwise part, B and C: 1,262).
constexpr int kStepAhead = 4;
constexpr int kStepThreads = 256;
template <typename T, int V, int LP>
__global__ void __launch_bounds__(kStepThreads) k_scan_step(Call a, float* state) {
    constexpr int HELD = V == 4 ? 4 : 2;                  // states of a lane at most: up to 64 over 16 or 32 lanes
    constexpr int TIMES = HELD / V;
    constexpr int OWN = LP >= kStepAhead ? 1 : kStepAhead / LP;  // sequences whose elementwise part a lane does
    wait_previous();
    release_next();
    __shared__ __align__(16) float bc[kStepAhead][2][kMostStates];
    const Sequences& q = a.q;
    const int channels = q.channels;
    // block = (turn * groups + group) * splits + split
    const int64_t at = static_cast<int64_t>(blockIdx.x) / a.splits;
    const int split = static_cast<int>(blockIdx.x - at * a.splits);
    const int64_t turn = at / a.groups;
    const int group = static_cast<int>(at - turn * a.groups);
    const int64_t s0 = turn * kStepAhead;
    const int count = static_cast<int>(min(int64_t{kStepAhead}, q.sequences - s0));
    for (int e = threadIdx.x; e < count * 2 * a.states; e += kStepThreads) {
        const int i = e / (2 * a.states), rest = e - i * 2 * a.states, which = rest / a.states, n = rest - which * a.states;
        const Track<void>& track = which ? a.c : a.b;
        const int64_t apart = which ? a.c_group : a.b_group;
        bc[i][which][n] = Element<T>::load(static_cast<const T*>(track.data)[(s0 + i) * track.sequence + group * apart + n]);
    }
    __syncthreads();
    const int lane = threadIdx.x % LP, n0 = lane * V;
    constexpr int TILE = kStepThreads / LP;
    for (int local = split * TILE + threadIdx.x / LP; local - static_cast<int>(threadIdx.x) / LP < a.per; local += a.splits * TILE) {
        const bool mine = local < a.per;
        const int c = group * a.per + (mine ? local : 0);
        Pack<float, V> h[kStepAhead][TIMES], rate[TIMES];
#pragma unroll
        for (int i = 0; i < kStepAhead; ++i) {
#pragma unroll
            for (int k = 0; k < TIMES; ++k) {
                const int n = n0 + k * LP * V;
                if (mine && i < count && n < a.states) h[i][k] = *reinterpret_cast<const Pack<float, V>*>(state + ((s0 + i) * channels + c) * a.states + n);
            }
        }
#pragma unroll
        for (int k = 0; k < TIMES; ++k) {
            const int n = n0 + k * LP * V;
            if (n < a.states) rate[k] = *reinterpret_cast<const Pack<float, V>*>(a.a + static_cast<int64_t>(c) * a.states + n);
        }
        // the elementwise part of this lane's own sequences
        float vu[OWN], size[OWN], gate[OWN];
        const float skip = a.d ? a.d[c] : 0.0f, bias = a.delta_bias ? a.delta_bias[c] : 0.0f;
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int i = lane + o * LP;
            vu[o] = size[o] = 0.0f;
            gate[o] = 1.0f;
            if (i >= count || i >= kStepAhead) continue;
            const int64_t s = s0 + i;
            vu[o] = Element<T>::load(static_cast<const T*>(a.u.data)[s * a.u.sequence + c]);
            size[o] = Element<T>::load(static_cast<const T*>(a.delta.data)[s * a.delta.sequence + c]) + bias;
            if (a.softplus) size[o] = softplus(size[o]);
            if (a.z.data) {
                const float w = Element<T>::load(static_cast<const T*>(a.z.data)[s * a.z.sequence + c]);
                gate[o] = w * sigmoid(w);
            }
        }
#pragma unroll
        for (int k = 0; k < TIMES; ++k) {
#pragma unroll
            for (int v = 0; v < V; ++v) rate[k].v[v] *= kLog2E;
        }
        float sum[kStepAhead];
#pragma unroll
        for (int i = 0; i < kStepAhead; ++i) {
            sum[i] = 0.0f;
            // (the lanes of a channel are neighbours in a warp: width LP)
            const float by = __shfl_sync(0xffffffffu, size[i / LP < OWN ? i / LP : 0], i % LP, LP);
            const float in = by * __shfl_sync(0xffffffffu, vu[i / LP < OWN ? i / LP : 0], i % LP, LP);
            if (i >= count) continue;
            const bool cut = q.reset != nullptr && q.reset[(s0 + i) * q.reset_sequence] != 0;
#pragma unroll
            for (int k = 0; k < TIMES; ++k) {
                const int n = n0 + k * LP * V;
                if (n >= a.states) continue;
                const Pack<float, V> b = *reinterpret_cast<const Pack<float, V>*>(&bc[i][0][n]), cc = *reinterpret_cast<const Pack<float, V>*>(&bc[i][1][n]);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float kept = cut ? 0.0f : decay(by, rate[k].v[v]), from = cut ? 0.0f : h[i][k].v[v];
                    h[i][k].v[v] = fmaf(kept, from, in * b.v[v]);
                    sum[i] = fmaf(h[i][k].v[v], cc.v[v], sum[i]);
                }
                if (mine) *reinterpret_cast<Pack<float, V>*>(state + ((s0 + i) * channels + c) * a.states + n) = h[i][k];
            }
        }
#pragma unroll
        for (int o = LP / 2; o >= 1; o >>= 1) {
#pragma unroll
            for (int i = 0; i < kStepAhead; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        }
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int i = lane + o * LP;
            float y = sum[0];
#pragma unroll
            for (int k = 1; k < kStepAhead; ++k) y = i == k ? sum[k] : y;
            if (mine && i < count && i < kStepAhead) {
                static_cast<T*>(a.y.data)[(s0 + i) * a.y.sequence + c] = Element<T>::store(fmaf(skip, vu[o], y) * gate[o]);
            }
        }
    }
}

// ------------------------------------------------------------------ host
// Lanes of a channel and states of a lane, for `states` states.
inline int padded(int64_t states) { return states <= 16 ? 16 : states <= 32 ? 32 : 64; }
inline int64_t tiles_of(int64_t steps) { return (steps + kTile - 1) / kTile; }

// The forward pass's chunks.
struct ForwardPlan {
    int channels, group_blocks, chunks, chunk;
    int64_t blocks;
    ForwardPlan(const t8b_sequences_t& q, int64_t groups, int64_t states) {
        channels = kThreads * kHeld / padded(states);
        group_blocks = static_cast<int>((q.channels / groups + channels - 1) / channels);
        const int64_t per_chunk = q.sequences * groups * group_blocks, steps = std::max<int64_t>(q.steps, 1);
        // cut where fewer than two blocks an SM would run; cutting takes every exponential twice
        int64_t want = 1;
        if (per_chunk < 3 * kSms) want = std::max<int64_t>(1, std::min<int64_t>(6 * kSms / std::max<int64_t>(per_chunk, 1), steps / 32));
        if (want < 3) want = 1;
        chunk = static_cast<int>(round_up((steps + want - 1) / want, kTile));
        chunks = static_cast<int>((steps + chunk - 1) / chunk);
        blocks = per_chunk * chunks;
    }
};
struct BackwardPlan {
    int channels, group_blocks, chunks, chunk, workers;
    int end_blocks;  // blocks of a group in k_scan_back_ends
    BackwardPlan(const t8b_sequences_t& q, int64_t groups, int64_t states) {
        channels = kThreads / 32 * 2 * (32 / (padded(states) / 4));
        group_blocks = static_cast<int>((q.channels / groups + channels - 1) / channels);
        end_blocks = static_cast<int>((q.channels / groups + kThreads * 16 / padded(states) - 1) / (kThreads * 16 / padded(states)));
        const int64_t across = groups * group_blocks, steps = std::max<int64_t>(q.steps, 1);
        const int64_t resident = std::max<int64_t>(1, 4 * kSms / across);
        // the least time by rounds of resident blocks; a cut takes a third more work
        int64_t best = 0, want = 1;
        for (int64_t parts = 1; parts <= std::max<int64_t>(1, steps / 64); parts = parts < 8 ? parts + 1 : parts + parts / 4) {
            const int64_t length = round_up((steps + parts - 1) / parts, kTile), count = (steps + length - 1) / length;
            const int64_t rounds = (q.sequences * count + resident - 1) / resident;
            const int64_t cost = rounds * length * (count > 1 ? 4 : 3);
            if (best == 0 || cost < best) {
                best = cost;
                want = parts;
            }
            if (q.sequences * count > 4 * resident) break;
        }
        chunk = static_cast<int>(round_up((steps + want - 1) / want, kTile));
        chunks = static_cast<int>((steps + chunk - 1) / chunk);
        workers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(resident, q.sequences * chunks)));
    }
};

template <typename T>
void launch_forward(const Call& given, const ForwardPlan& plan, int64_t states, cudaStream_t stream) {
    Call a = given;
    a.chunks = plan.chunks;
    a.chunk = plan.chunk;
    a.group_blocks = plan.group_blocks;
    auto go = [&](auto main, auto ends) {
        const unsigned grid = static_cast<unsigned>(plan.blocks);
        if (a.chunks > 1) {
            launch_chain("k_scan_ends", ends, grid, kThreads, 0, stream, true, a);
            launch_chain("k_scan_join", k_scan_join, blocks(a.q.sequences * states * a.q.channels, 256), 256, 0, stream, true, a, false);
        }
        launch_chain("k_scan_forward", main, grid, kThreads, 0, stream, true, a);
    };
    switch (padded(states)) {
        case 16: go(k_scan_forward<T, 1, false>, k_scan_forward<T, 1, true>); break;
        case 32: go(k_scan_forward<T, 2, false>, k_scan_forward<T, 2, true>); break;
        default: go(k_scan_forward<T, 4, false>, k_scan_forward<T, 4, true>); break;
    }
}

template <typename T, int LN>
void launch_backward_tiles(const Call& a, cudaStream_t stream) {
    constexpr size_t bytes = sizeof(typename Backward<T, LN>::Shared);
    static uint64_t configured = 0;
    allow_smem(k_scan_backward<T, LN>, bytes, configured);
    launch_chain("k_scan_backward", k_scan_backward<T, LN>, dim3(a.groups * a.group_blocks, a.workers), kThreads, bytes, stream, true, a);
}

template <typename T>
void launch_backward(const Call& given, const BackwardPlan& plan, float* da, float* dd, float* dbias, cudaStream_t stream) {
    Call a = given;
    a.chunks = plan.chunks;
    a.chunk = plan.chunk;
    a.workers = plan.workers;
    const int width = padded(a.states);
    if (a.chunks > 1) {
        a.group_blocks = plan.end_blocks;
        const int64_t grid = a.q.sequences * a.chunks * a.groups * a.group_blocks;
        auto ends = width == 16 ? k_scan_back_ends<T, 16, 1> : width == 32 ? k_scan_back_ends<T, 16, 2> : k_scan_back_ends<T, 16, 4>;
        launch_chain("k_scan_back_ends", ends, static_cast<unsigned>(grid), kThreads, 0, stream, true, a);
        launch_chain("k_scan_join", k_scan_join, blocks(a.q.sequences * a.states * a.q.channels, 256), 256, 0, stream, true, a, true);
    }
    a.group_blocks = plan.group_blocks;
    switch (width) {
        case 16: launch_backward_tiles<T, 4>(a, stream); break;
        case 32: launch_backward_tiles<T, 8>(a, stream); break;
        default: launch_backward_tiles<T, 16>(a, stream); break;
    }
    launch_chain("k_scan_parameters", k_scan_parameters, blocks(static_cast<int64_t>(a.states + 2) * a.q.channels, 32), dim3(32, 16), 0, stream,
                 true, a, da, dd, dbias);
    const int64_t outputs = a.groups * a.q.sequences * a.q.steps * 2 * a.states;
    launch_chain("k_scan_shared", k_scan_shared<T>, static_cast<unsigned>((outputs + 255) / 256), 256, 0, stream, true, a);
}

template <typename T>
void launch_step(const Call& given, float* state, bool wide, cudaStream_t stream) {
    Call a = given;
    const int packs = wide ? a.states / 4 : a.states;
    int lanes = 1;
    while (lanes < packs && lanes < 32) lanes *= 2;
    const int64_t turns = (a.q.sequences + kStepAhead - 1) / kStepAhead, tiles = (a.per + kStepThreads / lanes - 1) / (kStepThreads / lanes);
    // as many blocks as are resident at once, four an SM, where the sequences alone do not make them
    a.splits = static_cast<int>(std::max<int64_t>(1, std::min(tiles, 4 * kSms / std::max<int64_t>(1, turns * a.groups))));
    const int64_t grid = turns * a.groups * a.splits;
    if (grid > std::numeric_limits<int32_t>::max()) raise(T8B_EINVAL, "selective scan step: too many elements for one call");
    auto go = [&](auto kernel) { launch_chain("k_scan_step", kernel, static_cast<unsigned>(grid), kStepThreads, 0, stream, true, a, state); };
    if (wide) {
        switch (lanes) {
            case 1: go(k_scan_step<T, 4, 1>); break;
            case 2: go(k_scan_step<T, 4, 2>); break;
            case 4: go(k_scan_step<T, 4, 4>); break;
            case 8: go(k_scan_step<T, 4, 8>); break;
            default: go(k_scan_step<T, 4, 16>); break;
        }
    } else {
        switch (lanes) {
            case 1: go(k_scan_step<T, 1, 1>); break;
            case 2: go(k_scan_step<T, 1, 2>); break;
            case 4: go(k_scan_step<T, 1, 4>); break;
            case 8: go(k_scan_step<T, 1, 8>); break;
            case 16: go(k_scan_step<T, 1, 16>); break;
            default: go(k_scan_step<T, 1, 32>); break;
        }
    }
}

}  // namespace scan
}  // namespace op
}  // namespace t8b
