// Causal convolution with one short filter a channel, over sequences with resets and lengths.
//
//   p_t = b + sum_(j < K) w[K - 1 - j] x_(t-j),   y_t = act(p_t)
//   dp_t = dy_t act'(p_t),   dx_t = sum_(j < K) w[K - 1 - j] dp_(t+j),   dw[K - 1 - j] = sum dp_t x_(t-j),   db = sum dp_t
//
// where a term whose two steps lie on different sides of a reset is left out. Bound by memory: x (and
// dy) once in, y (or dx) once out. A thread takes V consecutive channels of a run of steps and keeps
// the last K - 1 rows in registers, so a row is read once but for the K - 1 rows around a run, which
// neighbouring threads hold in L1 or L2. Rows come through a ring in shared memory that a thread fills
// (cp.async) and reads alone: two groups of rows are in flight while one is worked on, and no thread waits for
// another. 65,536 x 1,024 with 4 taps and silu in bf16: forward 68 us (62 % of the copy rate), backward 129 (48 %);
// rows loaded into registers took 109 and 341. What is left is latency and instructions: 22 and 16 warps an SM at 55 %
// of their issue slots.
#include "ops_memory.cuh"

namespace t8b {
namespace op {
namespace {

constexpr int kThreads = 128;
constexpr int kRun = 32;      // steps of a thread's run
constexpr int kBackRun = 64;  // backward: the longer, the fewer steps are computed twice around its ends
constexpr int kGroup = 4;  // rows that are taken together
constexpr int kSms = 148;
constexpr int kPartialRows = 16;

struct Conv {
    Sequences q;
    Track<void> x, dy, y;  // y: y, or dx
    const void* weight;
    const void* bias;
    const void* state;
    const void* final_gradient;
    void* final_state;
    void* dstate;
    float* partial;  // [workers][width + 1][channels]: sums of dw and db
    int parameter_type, activation, runs, packs;
    int lanes;  // neighbouring threads of one run: a power of two, at most a warp
};

// V channels as (V + 1) / 2 pairs.
template <int V, int K>
__device__ __forceinline__ void load_filter(const Conv& a, int c, Two (&w)[K][(V + 1) / 2], Two (&b)[(V + 1) / 2]) {
    float f[K + 1][V + 1] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) {
        f[K][v] = a.bias ? load_any(a.bias, a.parameter_type, c + v) : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) f[k][v] = load_any(a.weight, a.parameter_type, static_cast<size_t>(c + v) * K + k);
    }
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) {
        b[i] = Two(f[K][2 * i], f[K][2 * i + 1]);
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = Two(f[k][2 * i], f[k][2 * i + 1]);
    }
}
template <int H, int N>
__device__ __forceinline__ void clear(Two (&v)[N][H]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
        for (int i = 0; i < H; ++i) v[k][i] = Two();
    }
}
template <int H, int N>
__device__ __forceinline__ void shift(Two (&window)[N][H], const Two (&x)[H]) {
#pragma unroll
    for (int k = 0; k + 1 < N; ++k) {
#pragma unroll
        for (int i = 0; i < H; ++i) window[k][i] = window[k + 1][i];
    }
#pragma unroll
    for (int i = 0; i < H; ++i) window[N - 1][i] = x[i];
}
template <int ACT>
__device__ __forceinline__ Two activate_two(const Two& v) {
    const float2 f = v.get();
    return Two(activate<ACT>(f.x), activate<ACT>(f.y));
}
template <int ACT>
__device__ __forceinline__ Two slope_of(const Two& v) {
    const float2 f = v.get();
    float value, x, y;
    activate_slope<ACT>(f.x, value, x);
    activate_slope<ACT>(f.y, value, y);
    return Two(x, y);
}
// The rows of a run one after the other, V elements of each, through this thread's slots of the ring: two
// groups of kGroup rows, `kThreads` packs apart. Rows at and past `end` are zeros.
template <typename T, int V>
struct Ring {
    Held<T, V>* slots;
    const T* from;  // the next row to fetch
    int64_t step;
    int next, end;
    __device__ __forceinline__ Ring(Held<T, V>* slots_, const T* base, int64_t step_, int t0, int end_)
        : slots(slots_), from(base + t0 * step_), step(step_), next(t0), end(end_) {}
    __device__ __forceinline__ void fetch(int half) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i, ++next, from += step) {
            Held<T, V>* to = slots + (half * kGroup + i) * kThreads;
            if (next >= end) {
                *to = Held<T, V>{};
            } else if constexpr (V * sizeof(T) >= 4) {
                copy_async<V * sizeof(T)>(to, from);
            } else {
                *to = load_held<T, V>(from);
            }
        }
    }
    __device__ __forceinline__ void take(int half, Held<T, V> (&rows)[kGroup]) const {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) rows[i] = slots[(half * kGroup + i) * kThreads];
    }
};
// Which of the 32 steps from t0 on (those before `end`) are resets, a bit each: `lanes` threads find them together.
__device__ __forceinline__ uint32_t resets_of(const Sequences& q, int64_t s, int t0, int end, int lanes) {
    if (q.reset == nullptr) return 0;
    uint32_t bits = 0;
    for (int i = threadIdx.x & (lanes - 1); i < 32; i += lanes) {
        if (t0 + i < end && q.resets(s, t0 + i)) bits |= 1u << i;
    }
    for (int o = lanes / 2; o >= 1; o >>= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, o);
    return bits;
}
template <int H, int K>
__device__ __forceinline__ void filter(const Two (&w)[K][H], const Two (&b)[H], const Two (&window)[K - 1][H], const Two (&row)[H], Two (&p)[H]) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
        p[i] = multiply_add(w[K - 1][i], row[i], b[i]);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) p[i] = multiply_add(w[k][i], window[k][i], p[i]);
    }
}
// The K - 1 rows before step t0, as step t0 may see them (a reset at t0 itself is the caller's), and
// how many steps of its round they reach back, at most K.
template <typename T, int V, int K>
__device__ __forceinline__ int load_window(const Conv& a, const T* x, int64_t s, int c, int t0, Two (&window)[K - 1][(V + 1) / 2]) {
    constexpr int H = (V + 1) / 2;
    const Sequences& q = a.q;
    int since = K;
    clear<H, K - 1>(window);
    Held<T, V> raw[K - 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int t = t0 - (K - 1) + k;
        raw[k] = Held<T, V>{};
        if (t >= 0) {
            raw[k] = load_held<T, V>(x + t * a.x.step);
        } else if (a.state) {
            raw[k] = load_held<T, V>(static_cast<const T*>(a.state) + (s * (K - 1) + (K - 1 + t)) * q.channels + c);
        }
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int t = t0 - (K - 1) + k;
        if (t >= 0) {
            ++since;
            if (q.resets(s, t)) {
                clear<H, K - 1>(window);
                since = 0;
            }
        }
        Two row[H];
        unpack<T, V>(raw[k], row);
        shift<H, K - 1>(window, row);
    }
    return since;
}

// One thread: a pack of channels, a run of steps of a sequence.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads, 6) k_conv_forward(Conv a) {
    constexpr int H = (V + 1) / 2;
    __shared__ Held<T, V> ring[2 * kGroup][kThreads];
    wait_previous();
    release_next();
    const Sequences& q = a.q;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int across = (a.packs + a.lanes - 1) / a.lanes * a.lanes;
    const int64_t item = index / across;
    const int column = static_cast<int>(index - item * across), c = column * V;
    const bool inside = item < q.sequences * a.runs;
    const int64_t run = inside ? item / q.sequences : 0, s = inside ? item - run * q.sequences : 0;
    const int t0 = static_cast<int>(run) * kRun, t1 = min(q.steps, t0 + kRun), last = q.live(s), end = min(t1, last);
    const uint32_t resets = resets_of(q, s, t0, end, a.lanes);
    if (!inside || column >= a.packs) return;
    const T* x = static_cast<const T*>(a.x.data) + s * a.x.sequence + c;
    T* y = static_cast<T*>(a.y.data) + s * a.y.sequence + c + t0 * a.y.step;
    T* final_state = a.final_state ? static_cast<T*>(a.final_state) + s * (K - 1) * q.channels + c : nullptr;
    const bool none = t0 == 0 && last == 0;  // no step: the final state is the initial one
    Two window[K - 1][H];
    int t = t0;
    if (end > t0) {
        Ring<T, V> rows(&ring[0][threadIdx.x], x, a.x.step, t0, end);
        rows.fetch(0);
        copies_commit();
        rows.fetch(1);
        copies_commit();
        load_window<T, V, K>(a, x, s, c, t0, window);
        Two w[K][H], b[H];
        load_filter<V, K>(a, c, w, b);
        with_activation(a.activation, [&](auto act) {
            for (int half = 0; t < end; half ^= 1) {
                Held<T, V> now[kGroup];
                copies_wait<1>();
                rows.take(half, now);
                rows.fetch(half);
                copies_commit();
                auto step = [&](int i) {
                    Two row[H], p[H];
                    unpack<T, V>(now[i], row);
                    filter<H, K>(w, b, window, row, p);
#pragma unroll
                    for (int h = 0; h < H; ++h) p[h] = activate_two<decltype(act)::value>(p[h]);
                    *reinterpret_cast<Held<T, V>*>(y) = pack<T, V>(p);
                    y += a.y.step;
                    shift<H, K - 1>(window, row);
                };
                if (t + kGroup <= end && (resets >> (t - t0) & ((1u << kGroup) - 1)) == 0) {
#pragma unroll
                    for (int i = 0; i < kGroup; ++i) step(i);
                } else {
#pragma unroll
                    for (int i = 0; i < kGroup; ++i) {
                        if (t + i >= end) continue;
                        if (resets >> (t - t0 + i) & 1) clear<H, K - 1>(window);
                        step(i);
                    }
                }
                t += kGroup;
            }
        });
        copies_wait<0>();
    } else if (none && final_state) {
        load_window<T, V, K>(a, x, s, c, t0, window);
    }
    if (final_state && (none || (end > t0 && end == last))) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Held<T, V>*>(final_state + k * q.channels) = pack<T, V>(window[k]);
    }
    for (t = max(t0, end); t < t1; ++t, y += a.y.step) *reinterpret_cast<Held<T, V>*>(y) = Held<T, V>{};
}

// Block (x, y): x packs of channels, y runs at a time; every thread goes through the runs that are a
// multiple of the launch's workers apart and keeps its channels' sums of dw and db. A run's dx takes
// dp of the K - 1 steps behind it too, which are computed again.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 3) k_conv_backward(Conv a) {
    constexpr int H = (V + 1) / 2;
    constexpr int WIDTH = (K + 1) * 2 * H + 1;
    // the ring of x and dy, and at the end the sums of the block's threads
    constexpr int RING = 4 * kGroup * kThreads * sizeof(Held<T, V>), SUMS = kThreads * WIDTH * sizeof(float);
    __shared__ __align__(16) unsigned char memory[RING > SUMS ? RING : SUMS];
    auto* ring = reinterpret_cast<Held<T, V>*>(memory) + threadIdx.y * blockDim.x + threadIdx.x;
    wait_previous();
    release_next();
    const Sequences& q = a.q;
    const int column = blockIdx.x * blockDim.x + threadIdx.x;
    const int c = column * V;
    const bool mine = column < a.packs;
    const int cc = mine ? c : 0;
    Two dw[K][H], db[1][H], w[K][H], b[H];
    clear<H, K>(dw);
    clear<H, 1>(db);
    load_filter<V, K>(a, cc, w, b);
    const int64_t items = q.sequences * a.runs;
    // every thread of a warp makes as many turns: the resets are found together
    for (int64_t turn = static_cast<int64_t>(blockIdx.y) * blockDim.y; turn < items; turn += static_cast<int64_t>(gridDim.y) * blockDim.y) {
        const int64_t item = min(turn + threadIdx.y, items - 1);
        const bool working = mine && turn + threadIdx.y < items;
        const int64_t run = item / q.sequences, s = item - run * q.sequences;
        const int t0 = static_cast<int>(run) * kBackRun, t1 = min(q.steps, t0 + kBackRun), last = q.live(s), far = min(t1 + K - 1, last);
        static_assert(kBackRun == 64, "two words of resets, and one for the steps behind the run");
        const uint64_t resets = resets_of(q, s, t0, far, a.lanes) | static_cast<uint64_t>(resets_of(q, s, t0 + 32, far, a.lanes)) << 32;
        const uint32_t behind = resets_of(q, s, t0 + kBackRun, far, a.lanes);
        if (!working) continue;
        const T* x = static_cast<const T*>(a.x.data) + s * a.x.sequence + c;
        const T* dy = static_cast<const T*>(a.dy.data) + s * a.dy.sequence + c;
        T* dx = a.y.data ? static_cast<T*>(a.y.data) + s * a.y.sequence + c : nullptr;
        T* dstate = a.dstate ? static_cast<T*>(a.dstate) + s * (K - 1) * q.channels + c : nullptr;
        const T* given = a.final_gradient ? static_cast<const T*>(a.final_gradient) + s * (K - 1) * q.channels + c : nullptr;
        // pending[j]: the gradient so far of the row j before the current one; the oldest is complete
        // once the current step has added to it
        Two pending[K][H], window[K - 1][H];
        clear<H, K>(pending);
        if (last > t0) {
            Ring<T, V> rows_x(ring, x, a.x.step, t0, far), rows_dy(ring + 2 * kGroup * kThreads, dy, a.dy.step, t0, far);
            rows_x.fetch(0);
            rows_dy.fetch(0);
            copies_commit();
            rows_x.fetch(1);
            rows_dy.fetch(1);
            copies_commit();
            int since = load_window<T, V, K>(a, x, s, c, t0, window);
            T* to = dx ? dx + (t0 - (K - 1)) * a.y.step : nullptr;
            with_activation(a.activation, [&](auto act) {
                int half = 0;
                for (int t = t0; t < t1 + K - 1; t += kGroup, half ^= 1) {
                    Held<T, V> now_x[kGroup], now_dy[kGroup];
                    copies_wait<1>();
                    rows_x.take(half, now_x);
                    rows_dy.take(half, now_dy);
                    rows_x.fetch(half);
                    rows_dy.fetch(half);
                    copies_commit();
                    const uint32_t begins = t - t0 < kBackRun ? static_cast<uint32_t>(resets >> (t - t0)) : behind >> (t - t0 - kBackRun);
                    auto step = [&](auto whole, int i) {
                        constexpr bool WHOLE = decltype(whole)::value != 0;  // within the run, and no reset near
                        const int at = t + i;
                        Two row[H], p[H], pre[H];
                        unpack<T, V>(now_x[i], row);
                        unpack<T, V>(now_dy[i], p);
                        if (!WHOLE) {
                            since = min(since + 1, K);
                            if (begins >> i & 1) {
                                clear<H, K - 1>(window);
                                since = 0;
                            }
                        }
                        filter<H, K>(w, b, window, row, pre);
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            p[h] = p[h] * slope_of<decltype(act)::value>(pre[h]);
                            if (!WHOLE && at >= last) p[h] = Two();  // behind the sequence nothing is added any more
                        }
#pragma unroll
                        for (int j = K - 1; j >= 1; --j) {
#pragma unroll
                            for (int h = 0; h < H; ++h) {
                                pending[j][h] = multiply_add(w[K - 1 - j][h], WHOLE || since >= j ? p[h] : Two(), pending[j - 1][h]);
                            }
                        }
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            pending[0][h] = w[K - 1][h] * p[h];
                            const Two own = WHOLE || at < t1 ? p[h] : Two();
                            db[0][h] = db[0][h] + own;
                            dw[K - 1][h] = multiply_add(own, row[h], dw[K - 1][h]);
#pragma unroll
                            for (int k = 0; k < K - 1; ++k) dw[k][h] = multiply_add(own, window[k][h], dw[k][h]);
                        }
                        if (!WHOLE && at == last - 1 && given) {  // the final state's entry K - 2 - j is row last - 1 - j
#pragma unroll
                            for (int j = 0; j < K - 1; ++j) {
                                if (since < j) continue;
                                Two v[H];
                                unpack<T, V>(load_held<T, V>(given + (K - 2 - j) * q.channels), v);
#pragma unroll
                                for (int h = 0; h < H; ++h) pending[j][h] = pending[j][h] + v[h];
                            }
                        }
                        const int done = at - (K - 1);
                        if (WHOLE || (done >= t0 && done < t1)) {
                            if (dx) *reinterpret_cast<Held<T, V>*>(to) = pack<T, V>(pending[K - 1]);
                        } else if (done < 0 && t0 == 0 && dstate) {
                            *reinterpret_cast<Held<T, V>*>(dstate + (K - 1 + done) * q.channels) = pack<T, V>(pending[K - 1]);
                        }
                        if (dx) to += a.y.step;
                        shift<H, K - 1>(window, row);
                    };
                    const bool whole = since >= K - 1 && t >= t0 + K - 1 && t + kGroup <= t1 && t + kGroup < last && (begins & ((1u << kGroup) - 1)) == 0;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < kGroup; ++i) {
                            in_order();
                            step(Constant<1>{}, i);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < kGroup; ++i) {
                            in_order();
                            step(Constant<0>{}, i);
                        }
                    }
                }
            });
            copies_wait<0>();
            continue;
        }
        if (t0 == 0 && dstate) {  // no step: the final state is the initial one
#pragma unroll
            for (int k = 0; k < K - 1; ++k) {
                *reinterpret_cast<Held<T, V>*>(dstate + k * q.channels) = given ? load_held<T, V>(given + k * q.channels) : pack<T, V>(pending[k]);
            }
        }
        if (dx) {
            const Two zero[H];
            for (int t = t0; t < t1; ++t) *reinterpret_cast<Held<T, V>*>(dx + t * a.y.step) = pack<T, V>(zero);
        }
    }
    if (a.partial == nullptr) return;
    // the block's rows of threads meet in shared memory, in their order
    __syncthreads();
    float* slot = reinterpret_cast<float*>(memory) + (threadIdx.y * blockDim.x + threadIdx.x) * WIDTH;
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int k = 0; k <= K; ++k) {
            const float2 f = k < K ? dw[k < K ? k : 0][h].get() : db[0][h].get();
            slot[(k * H + h) * 2] = f.x;
            slot[(k * H + h) * 2 + 1] = f.y;
        }
    }
    __syncthreads();
    if (threadIdx.y != 0 || !mine) return;
    float* out = a.partial + static_cast<size_t>(blockIdx.y) * (K + 1) * q.channels + c;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float sum = 0.0f;
            for (int r = 0; r < blockDim.y; ++r) sum += slot[r * blockDim.x * WIDTH + k * 2 * H + v];
            out[static_cast<size_t>(k) * q.channels + v] = sum;
        }
    }
}

// dw and db from the blocks' sums, in a fixed order. Block (32, kPartialRows): 32 of the (width + 1) channels columns.
__global__ void k_conv_parameters(const float* partial, int count, int channels, int width, void* dw, void* db, int type) {
    wait_previous();
    release_next();
    __shared__ float sums[kPartialRows][33];
    const int columns = (width + 1) * channels;
    const int column = blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (column < columns) {
#pragma unroll 4
        for (int r = threadIdx.y; r < count; r += kPartialRows) v += partial[static_cast<size_t>(r) * columns + column];
    }
    sums[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y != 0 || column >= columns) return;
#pragma unroll
    for (int r = 1; r < kPartialRows; ++r) v += sums[r][threadIdx.x];
    const int k = column / channels, c = column - k * channels;
    if (k == width) {
        if (db) store_any(db, type, c, v);
    } else if (dw) {
        store_any(dw, type, static_cast<size_t>(c) * width + k, v);
    }
}

// One thread: a pack of channels of a sequence, one step.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) k_conv_step(Conv a) {
    wait_previous();
    release_next();
    const Sequences& q = a.q;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t s = index / a.packs;
    const int c = static_cast<int>(index - s * a.packs) * V;
    if (s >= q.sequences) return;
    T* state = static_cast<T*>(a.final_state) + s * (K - 1) * q.channels + c;
    const Held<T, V> raw = load_held<T, V>(static_cast<const T*>(a.x.data) + s * a.x.sequence + c);
    Held<T, V> held[K - 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) held[k] = load_held<T, V>(state + k * q.channels);
    const bool cut = q.reset != nullptr && q.reset[s * q.reset_sequence] != 0;
    constexpr int H = (V + 1) / 2;
    Two w[K][H], p[H], row[H];
    load_filter<V, K>(a, c, w, p);
    if (cut) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) held[k] = Held<T, V>{};
    }
    unpack<T, V>(raw, row);
#pragma unroll
    for (int h = 0; h < H; ++h) p[h] = multiply_add(w[K - 1][h], row[h], p[h]);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        unpack<T, V>(held[k], row);
#pragma unroll
        for (int h = 0; h < H; ++h) p[h] = multiply_add(w[k][h], row[h], p[h]);
    }
    with_activation(a.activation, [&](auto act) {
#pragma unroll
        for (int h = 0; h < H; ++h) p[h] = activate_two<decltype(act)::value>(p[h]);
    });
    *reinterpret_cast<Held<T, V>*>(static_cast<T*>(a.y.data) + s * a.y.sequence + c) = pack<T, V>(p);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Held<T, V>*>(state + k * q.channels) = k + 1 < K - 1 ? held[k + 1 < K - 1 ? k + 1 : 0] : raw;
}

// ------------------------------------------------------------------ dispatch
template <typename Body>
void with_width(int width, Body&& body) {
    switch (width) {
        case 2: body(Constant<2>{}); break;
        case 3: body(Constant<3>{}); break;
        default: body(Constant<4>{}); break;
    }
}

// How the backward pass is laid out: threads along packs, rows of threads, blocks along runs.
struct Layout {
    int across, rows, columns, workers;
    Layout(int64_t items, int packs) {
        across = kThreads;
        while (across > 1 && across / 2 >= packs) across /= 2;
        rows = kThreads / across;
        columns = (packs + across - 1) / across;
        // four blocks an SM are resident; more workers leave more sums to join
        workers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((items + rows - 1) / rows, 4 * kSms / std::min(columns, 4 * kSms))));
    }
};
// Neighbouring threads of one run in the forward pass.
int lanes_of(int packs) {
    int lanes = 32;
    while (lanes > 1 && lanes / 2 >= packs) lanes /= 2;
    return lanes;
}
int64_t runs_of(int64_t steps, int run) { return std::max<int64_t>(1, (steps + run - 1) / run); }

// Consecutive channels of a thread where every row and state starts on a pack's boundary. (8 of 16 bits take fewer
// instructions but twice the registers: 65,536 x 1,024 in bf16 forward 84 us against 72.)
constexpr int kPack = 4;

void check_call(const char* what, const t8b_sequences_t* q, bool step, int type, const void* weight, const void* bias, int parameter_type,
                int width, int activation) {
    check_sequences(what, q, step);
    const std::string name(what);
    if (!is_type(type) || !is_type(parameter_type)) raise(T8B_EINVAL, name + ": unknown type");
    if (parameter_type != T8B_F32 && parameter_type != type) raise(T8B_EINVAL, name + ": weight and bias are fp32 or of x's type");
    if (width < 2 || width > 4) raise(T8B_EINVAL, name + ": a width of 2 to 4");
    if (activation < T8B_LINEAR || activation > T8B_TANH) raise(T8B_EINVAL, name + ": unknown activation");
    if (weight == nullptr) raise(T8B_EINVAL, name + ": weight is null");
    for (const void* p : {weight, bias}) check_elements(what, p, type_size(parameter_type));
}

}  // namespace
}  // namespace op
}  // namespace t8b

using namespace t8b;
using namespace t8b::op;

extern "C" int t8b_causal_conv_forward(const t8b_sequences_t* q, int type, t8b_track_t x, const void* weight, const void* bias,
                                       int parameter_type, int width, int activation, const void* state, t8b_track_t y,
                                       void* final_state, void* stream) {
    return guarded([&] {
        check_call("causal conv", q, false, type, weight, bias, parameter_type, width, activation);
        const size_t size = type_size(type);
        check_track("causal conv x", *q, false, x, q->channels, size, false);
        check_track("causal conv y", *q, false, y, q->channels, size, true);
        for (const void* p : {state, static_cast<const void*>(final_state)}) check_elements("causal conv state", p, size);
        if (q->sequences == 0) return;
        const int64_t held = q->sequences * (width - 1) * q->channels;
        Overlaps o{"causal conv"};
        o.input(span_of(*q, false, x, q->channels, size));
        o.input(span_of(state, held, size));
        o.output(span_of(*q, false, y, q->channels, size));
        o.output(span_of(final_state, held, size));
        Conv a{};
        a.q = Sequences(*q);
        a.x = Track<void>(x);
        a.y = Track<void>(y);
        a.weight = weight;
        a.bias = bias;
        a.state = state;
        a.final_state = final_state;
        a.parameter_type = parameter_type;
        a.activation = activation;
        a.runs = static_cast<int>(runs_of(q->steps, kRun));
        with_type(type, [&](auto element) {
            using T = decltype(element);
            constexpr int V = kPack;
            const bool wide = q->channels % V == 0 && rows_aligned(*q, false, x, size, V * size) && rows_aligned(*q, false, y, size, V * size) &&
                aligned(state, V * size) && aligned(final_state, V * size);
            a.packs = static_cast<int>(wide ? q->channels / V : q->channels);
            a.lanes = lanes_of(a.packs);
            const int64_t grid = (q->sequences * a.runs * ((a.packs + a.lanes - 1) / a.lanes * a.lanes) + kThreads - 1) / kThreads;
            if (grid > std::numeric_limits<int32_t>::max()) raise(T8B_EINVAL, "causal conv: too many elements for one call");
            with_width(width, [&](auto k) {
                constexpr int K = decltype(k)::value;
                launch_chain("k_conv_forward", wide ? k_conv_forward<T, V, K> : k_conv_forward<T, 1, K>, static_cast<unsigned>(grid), kThreads, 0,
                             static_cast<cudaStream_t>(stream), true, a);
            });
        });
        check(cudaGetLastError(), "causal conv launch");
    });
}

extern "C" size_t t8b_causal_conv_workspace(const t8b_sequences_t* q, int width) {
    if (q == nullptr || !countable(*q) || q->sequences < 1 || width < 2 || width > 4) return 0;
    const int64_t items = q->sequences * runs_of(q->steps, kBackRun);
    const Layout wide(items, static_cast<int>((q->channels + kPack - 1) / kPack)), single(items, static_cast<int>(q->channels));
    return sizeof(float) * static_cast<size_t>(std::max(wide.workers, single.workers)) * (width + 1) * q->channels;
}

extern "C" int t8b_causal_conv_backward(const t8b_sequences_t* q, int type, t8b_track_t dy, t8b_track_t x, const void* weight,
                                        const void* bias, int parameter_type, int width, int activation, const void* state,
                                        const void* final_gradient, t8b_track_t dx, void* dweight, void* dbias, void* dstate,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_call("causal conv", q, false, type, weight, bias, parameter_type, width, activation);
        const size_t size = type_size(type);
        check_track("causal conv dy", *q, false, dy, q->channels, size, false);
        check_track("causal conv x", *q, false, x, q->channels, size, false);
        if (dx.data) check_track("causal conv dx", *q, false, dx, q->channels, size, true);
        for (const void* p : {state, final_gradient, static_cast<const void*>(dstate)}) check_elements("causal conv state", p, size);
        for (const void* p : {dweight, dbias}) check_elements("causal conv parameters", p, type_size(parameter_type));
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const bool parameters = dweight != nullptr || dbias != nullptr;
        if (q->sequences == 0) {
            if (dweight) check(cudaMemsetAsync(dweight, 0, q->channels * width * type_size(parameter_type), st), "clear dweight");
            if (dbias) check(cudaMemsetAsync(dbias, 0, q->channels * type_size(parameter_type), st), "clear dbias");
            return;
        }
        const int64_t held = q->sequences * (width - 1) * q->channels;
        Overlaps o{"causal conv"};
        o.input(span_of(*q, false, dy, q->channels, size));
        o.input(span_of(*q, false, x, q->channels, size));
        o.input(span_of(state, held, size));
        o.input(span_of(final_gradient, held, size));
        o.output(span_of(*q, false, dx, q->channels, size));
        o.output(span_of(dstate, held, size));
        if (parameters && (workspace == nullptr || workspace_bytes < t8b_causal_conv_workspace(q, width) || !aligned(workspace, 16))) {
            raise(T8B_EINVAL, "causal conv: the workspace is missing, unaligned or smaller than t8b_causal_conv_workspace");
        }
        Conv a{};
        a.q = Sequences(*q);
        a.x = Track<void>(x);
        a.dy = Track<void>(dy);
        a.y = Track<void>(dx);
        a.weight = weight;
        a.bias = bias;
        a.state = state;
        a.final_gradient = final_gradient;
        a.dstate = dstate;
        a.partial = parameters ? static_cast<float*>(workspace) : nullptr;
        a.parameter_type = parameter_type;
        a.activation = activation;
        a.runs = static_cast<int>(runs_of(q->steps, kBackRun));
        with_type(type, [&](auto element) {
            using T = decltype(element);
            constexpr int V = kPack;
            bool wide = q->channels % V == 0;
            for (const t8b_track_t* t : {&dy, &x, &dx}) wide = wide && rows_aligned(*q, false, *t, size, V * size);
            for (const void* p : {state, final_gradient, static_cast<const void*>(dstate)}) wide = wide && aligned(p, V * size);
            a.packs = static_cast<int>(wide ? q->channels / V : q->channels);
            const Layout l(q->sequences * a.runs, a.packs);
            a.lanes = std::min(l.across, 32);
            with_width(width, [&](auto k) {
                constexpr int K = decltype(k)::value;
                launch_chain("k_conv_backward", wide ? k_conv_backward<T, V, K> : k_conv_backward<T, 1, K>, dim3(l.columns, l.workers),
                             dim3(l.across, l.rows), 0, st, true, a);
            });
            if (parameters) {
                launch_chain("k_conv_parameters", k_conv_parameters, blocks((width + 1) * q->channels, 32), dim3(32, kPartialRows), 0, st, true,
                             static_cast<const float*>(workspace), l.workers, static_cast<int>(q->channels), width, dweight, dbias, parameter_type);
            }
        });
        check(cudaGetLastError(), "causal conv launch");
    });
}

extern "C" int t8b_causal_conv_step(const t8b_sequences_t* q, int type, t8b_track_t x, const void* weight, const void* bias,
                                    int parameter_type, int width, int activation, void* state, t8b_track_t y, void* stream) {
    return guarded([&] {
        check_call("causal conv step", q, true, type, weight, bias, parameter_type, width, activation);
        const size_t size = type_size(type);
        check_track("causal conv step x", *q, true, x, q->channels, size, false);
        check_track("causal conv step y", *q, true, y, q->channels, size, true);
        check_elements("causal conv step state", state, size);
        if (q->sequences == 0) return;
        if (state == nullptr) raise(T8B_EINVAL, "causal conv step: state is null");
        Overlaps o{"causal conv step"};
        o.input(span_of(*q, true, x, q->channels, size));
        o.output(span_of(*q, true, y, q->channels, size));
        o.output(span_of(state, q->sequences * (width - 1) * q->channels, size));
        Conv a{};
        a.q = Sequences(*q);
        a.x = Track<void>(x);
        a.y = Track<void>(y);
        a.weight = weight;
        a.bias = bias;
        a.final_state = state;
        a.parameter_type = parameter_type;
        a.activation = activation;
        with_type(type, [&](auto element) {
            using T = decltype(element);
            constexpr int V = kPack;
            const bool wide = q->channels % V == 0 && rows_aligned(*q, true, x, size, V * size) && rows_aligned(*q, true, y, size, V * size) &&
                aligned(state, V * size);
            a.packs = static_cast<int>(wide ? q->channels / V : q->channels);
            const int64_t grid = (q->sequences * a.packs + kThreads - 1) / kThreads;
            if (grid > std::numeric_limits<int32_t>::max()) raise(T8B_EINVAL, "causal conv step: too many elements for one call");
            with_width(width, [&](auto k) {
                constexpr int K = decltype(k)::value;
                launch_chain("k_conv_step", wide ? k_conv_step<T, V, K> : k_conv_step<T, 1, K>, static_cast<unsigned>(grid), kThreads, 0,
                             static_cast<cudaStream_t>(stream), true, a);
            });
        });
        check(cudaGetLastError(), "causal conv step launch");
    });
}
