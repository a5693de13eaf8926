// Causal convolution with one short filter a channel, over sequences with resets and lengths.
//
//   p_t = b + sum_(j < K) w[K - 1 - j] x_(t-j),   y_t = act(p_t)
//   dp_t = dy_t act'(p_t),   dx_t = sum_(j < K) w[K - 1 - j] dp_(t+j),   dw[K - 1 - j] = sum dp_t x_(t-j),   db = sum dp_t
//
// where a term whose two steps lie on different sides of a reset is left out. Bound by memory: x (and
// dy) once in, y (or dx) once out. A thread takes V consecutive channels of a run of steps and keeps
// the last K - 1 rows in registers, so a row is read once but for the K - 1 rows around a run, which
// neighbouring threads hold in L1 or L2; the rows of the next turn are in flight while one is worked on.
#include "ops_memory.cuh"

namespace t8b {
namespace op {
namespace {

constexpr int kThreads = 128;
constexpr int kRun = 32;       // steps of a thread's run
constexpr int kAhead = 4;      // rows in flight
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
};

template <int V, int K>
__device__ __forceinline__ void load_filter(const Conv& a, int c, float (&w)[K][V], float (&b)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        b[v] = a.bias ? load_any(a.bias, a.parameter_type, c + v) : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][v] = load_any(a.weight, a.parameter_type, static_cast<size_t>(c + v) * K + k);
    }
}
template <int V, int N>
__device__ __forceinline__ void clear(float (&v)[N][V]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] = 0.0f;
    }
}
template <int V, int N>
__device__ __forceinline__ void shift(float (&window)[N][V], const float (&x)[V]) {
#pragma unroll
    for (int k = 0; k + 1 < N; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) window[k][i] = window[k + 1][i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) window[N - 1][i] = x[i];
}
// The K - 1 rows before step t0, as step t0 may see them (a reset at t0 itself is the caller's), and
// how many steps of its round they reach back, at most K.
template <typename T, int V, int K>
__device__ __forceinline__ int load_window(const Conv& a, const T* x, int64_t s, int c, int t0, float (&window)[K - 1][V]) {
    const Sequences& q = a.q;
    int since = K;
    clear<V, K - 1>(window);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int t = t0 - (K - 1) + k;
        if (t >= 0) {
            if (q.resets(s, t)) {
                clear<V, K - 1>(window);
                since = 0;
            } else {
                ++since;
            }
            float row[V];
            unpack<T, V>(load_pack<T, V>(x + t * a.x.step), row);
            shift<V, K - 1>(window, row);
        } else {
            float row[V];
#pragma unroll
            for (int i = 0; i < V; ++i) row[i] = 0.0f;
            if (a.state) {
                const T* at = static_cast<const T*>(a.state) + (s * (K - 1) + (K - 1 + t)) * q.channels + c;
                unpack<T, V>(load_pack<T, V>(at), row);
            }
            shift<V, K - 1>(window, row);
        }
    }
    return since;
}

// One thread: a pack of channels, a run of steps of a sequence.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) k_conv_forward(Conv a) {
    wait_previous();
    release_next();
    const Sequences& q = a.q;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const int64_t item = index / a.packs;
    const int c = static_cast<int>(index - item * a.packs) * V;
    if (item >= q.sequences * a.runs) return;
    const int64_t s = item % q.sequences;
    const int t0 = static_cast<int>(item / q.sequences) * kRun, t1 = min(q.steps, t0 + kRun), last = q.live(s), end = min(t1, last);
    const T* x = static_cast<const T*>(a.x.data) + s * a.x.sequence + c;
    T* y = static_cast<T*>(a.y.data) + s * a.y.sequence + c;
    T* final_state = a.final_state ? static_cast<T*>(a.final_state) + s * (K - 1) * q.channels + c : nullptr;
    float window[K - 1][V];
    auto keep = [&]() {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Pack<T, V>*>(final_state + k * q.channels) = pack<T, V>(window[k]);
    };
    if (end > t0 || (t0 == 0 && last == 0 && final_state)) load_window<T, V, K>(a, x, s, c, t0, window);
    if (t0 == 0 && last == 0 && final_state) keep();
    if (end > t0) {
        float w[K][V], b[V];
        load_filter<V, K>(a, c, w, b);
        Pack<T, V> next[kAhead];
        bool flag[kAhead];
        auto fetch = [&](int t) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (t + i < end) {
                    next[i] = load_pack<T, V>(x + (t + i) * a.x.step);
                    flag[i] = q.resets(s, t + i);
                }
            }
        };
        fetch(t0);
        for (int t = t0; t < end; t += kAhead) {
            float row[kAhead][V];
            bool cut[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                unpack<T, V>(next[i], row[i]);
                cut[i] = flag[i];
            }
            fetch(t + kAhead);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (t + i >= end) break;
                if (cut[i]) clear<V, K - 1>(window);
                float p[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    p[v] = fmaf(w[K - 1][v], row[i][v], b[v]);
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) p[v] = fmaf(w[k][v], window[k][v], p[v]);
                }
                with_activation(a.activation, [&](auto act) {
#pragma unroll
                    for (int v = 0; v < V; ++v) p[v] = activate<decltype(act)::value>(p[v]);
                });
                *reinterpret_cast<Pack<T, V>*>(y + (t + i) * a.y.step) = pack<T, V>(p);
                shift<V, K - 1>(window, row[i]);
            }
        }
        if (end == last && final_state) keep();
    }
    Pack<T, V> zero;
#pragma unroll
    for (int v = 0; v < V; ++v) zero.v[v] = Element<T>::store(0.0f);
    for (int t = max(t0, end); t < t1; ++t) *reinterpret_cast<Pack<T, V>*>(y + t * a.y.step) = zero;
}

// Block (x, y): x packs of channels, y runs at a time; every thread goes through the runs that are a
// multiple of the launch's workers apart and keeps its channels' sums of dw and db. A run's dx takes
// dp of the K - 1 steps behind it too, which are computed again.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) k_conv_backward(Conv a) {
    wait_previous();
    release_next();
    const Sequences& q = a.q;
    const int column = blockIdx.x * blockDim.x + threadIdx.x;
    const int c = column * V;
    const bool mine = column < a.packs;
    float dw[K][V], db[1][V];
    clear<V, K>(dw);
    clear<V, 1>(db);
    if (mine) {
        float w[K][V], b[V];
        load_filter<V, K>(a, c, w, b);
        const int64_t items = q.sequences * a.runs;
        for (int64_t item = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; item < items;
             item += static_cast<int64_t>(gridDim.y) * blockDim.y) {
            const int64_t s = item % q.sequences;
            const int t0 = static_cast<int>(item / q.sequences) * kRun, t1 = min(q.steps, t0 + kRun), last = q.live(s);
            const T* x = static_cast<const T*>(a.x.data) + s * a.x.sequence + c;
            const T* dy = static_cast<const T*>(a.dy.data) + s * a.dy.sequence + c;
            T* dx = static_cast<T*>(a.y.data) + s * a.y.sequence + c;
            T* dstate = a.dstate ? static_cast<T*>(a.dstate) + s * (K - 1) * q.channels + c : nullptr;
            const T* given = a.final_gradient ? static_cast<const T*>(a.final_gradient) + s * (K - 1) * q.channels + c : nullptr;
            // pending[j]: the gradient so far of the row j before the current one; the oldest is complete
            // once the current step has added to it
            float pending[K][V], window[K - 1][V];
            clear<V, K>(pending);
            const int end = min(t1, last), far = min(t1 + K - 1, last);
            auto write = [&](int row, const float(&v)[V]) {
                if (row >= t0 && row < t1) {
                    if (dx) *reinterpret_cast<Pack<T, V>*>(dx + row * a.y.step) = pack<T, V>(v);
                } else if (row < 0 && t0 == 0 && dstate) {
                    *reinterpret_cast<Pack<T, V>*>(dstate + (K - 1 + row) * q.channels) = pack<T, V>(v);
                }
            };
            auto add_final = [&](int since) {  // after step last - 1: row last - 1 - j is entry K - 2 - j
                if (!given) return;
#pragma unroll
                for (int j = 0; j < K - 1; ++j) {
                    float v[V];
                    unpack<T, V>(load_pack<T, V>(given + (K - 2 - j) * q.channels), v);
#pragma unroll
                    for (int i = 0; i < V; ++i) pending[j][i] += since >= j ? v[i] : 0.0f;
                }
            };
            if (end > t0) {
                int since = load_window<T, V, K>(a, x, s, c, t0, window);
                Pack<T, V> next_x[kAhead], next_dy[kAhead];
                bool flag[kAhead];
                auto fetch = [&](int t) {
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        if (t + i < far) {
                            next_x[i] = load_pack<T, V>(x + (t + i) * a.x.step);
                            next_dy[i] = load_pack<T, V>(dy + (t + i) * a.dy.step);
                            flag[i] = q.resets(s, t + i);
                        }
                    }
                };
                fetch(t0);
                for (int t = t0; t < far; t += kAhead) {
                    float row[kAhead][V], g[kAhead][V];
                    bool cut[kAhead];
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        unpack<T, V>(next_x[i], row[i]);
                        unpack<T, V>(next_dy[i], g[i]);
                        cut[i] = flag[i];
                    }
                    fetch(t + kAhead);
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        const int at = t + i;
                        if (at >= far) break;
                        if (cut[i]) {
                            clear<V, K - 1>(window);
                            since = 0;
                        } else {
                            since = min(since + 1, K);
                        }
                        float p[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            p[v] = fmaf(w[K - 1][v], row[i][v], b[v]);
#pragma unroll
                            for (int k = 0; k < K - 1; ++k) p[v] = fmaf(w[k][v], window[k][v], p[v]);
                        }
                        with_activation(a.activation, [&](auto act) {
#pragma unroll
                            for (int v = 0; v < V; ++v) {
                                float value, slope;
                                activate_slope<decltype(act)::value>(p[v], value, slope);
                                p[v] = g[i][v] * slope;
                            }
                        });
#pragma unroll
                        for (int j = K - 1; j >= 1; --j) {
#pragma unroll
                            for (int v = 0; v < V; ++v) pending[j][v] = pending[j - 1][v] + (since >= j ? w[K - 1 - j][v] * p[v] : 0.0f);
                        }
#pragma unroll
                        for (int v = 0; v < V; ++v) pending[0][v] = w[K - 1][v] * p[v];
                        if (at < t1) {
#pragma unroll
                            for (int v = 0; v < V; ++v) {
                                db[0][v] += p[v];
                                dw[K - 1][v] = fmaf(p[v], row[i][v], dw[K - 1][v]);
#pragma unroll
                                for (int k = 0; k < K - 1; ++k) dw[k][v] = fmaf(p[v], window[k][v], dw[k][v]);
                            }
                        }
                        if (at == last - 1) add_final(since);
                        write(at - (K - 1), pending[K - 1]);
                        shift<V, K - 1>(window, row[i]);
                    }
                }
                // what ends with the sequence (a later run writes its rows itself)
                if (far == last) {
#pragma unroll
                    for (int j = K - 2; j >= 0; --j) write(far - 1 - j, pending[j]);
                }
            } else if (t0 == 0 && dstate) {  // no step: the final state is the initial one
                if (given) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Pack<T, V>*>(dstate + k * q.channels) = load_pack<T, V>(given + k * q.channels);
                } else {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Pack<T, V>*>(dstate + k * q.channels) = pack<T, V>(pending[k]);
                }
            }
            float zero[1][V];
            clear<V, 1>(zero);
            for (int t = max(t0, end); t < t1; ++t) write(t, zero[0]);
        }
    }
    if (a.partial == nullptr) return;
    // the block's rows of threads meet in shared memory, in their order
    __shared__ float joined[kThreads][(K + 1) * V + 1];
    float* slot = joined[threadIdx.y * blockDim.x + threadIdx.x];
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < K; ++k) slot[k * V + v] = dw[k][v];
        slot[K * V + v] = db[0][v];
    }
    __syncthreads();
    if (threadIdx.y != 0 || !mine) return;
    float* out = a.partial + static_cast<size_t>(blockIdx.y) * (K + 1) * q.channels + c;
#pragma unroll
    for (int i = 0; i < (K + 1) * V; ++i) {
        float sum = slot[i];
        for (int r = 1; r < blockDim.y; ++r) sum += slot[r * blockDim.x * ((K + 1) * V + 1) + i];
        out[static_cast<size_t>(i / V) * q.channels + i % V] = sum;
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
    const Pack<T, V> raw = load_pack<T, V>(static_cast<const T*>(a.x.data) + s * a.x.sequence + c);
    Pack<T, V> held[K - 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) held[k] = load_pack<T, V>(state + k * q.channels);
    const bool cut = q.reset != nullptr && q.reset[s * q.reset_sequence] != 0;
    float w[K][V], p[V], row[V];
    load_filter<V, K>(a, c, w, p);
    if (cut) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
#pragma unroll
            for (int v = 0; v < V; ++v) held[k].v[v] = Element<T>::store(0.0f);
        }
    }
    unpack<T, V>(raw, row);
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = fmaf(w[K - 1][v], row[v], p[v]);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        unpack<T, V>(held[k], row);
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] = fmaf(w[k][v], row[v], p[v]);
    }
    with_activation(a.activation, [&](auto act) {
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] = activate<decltype(act)::value>(p[v]);
    });
    *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.y.data) + s * a.y.sequence + c) = pack<T, V>(p);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Pack<T, V>*>(state + k * q.channels) = k + 1 < K - 1 ? held[k + 1 < K - 1 ? k + 1 : 0] : raw;
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
int64_t runs_of(int64_t steps) { return std::max<int64_t>(1, (steps + kRun - 1) / kRun); }

// V consecutive channels a thread where every row and state starts on a pack's boundary.
template <typename T>
constexpr int forward_pack() { return sizeof(T) == 2 ? 8 : 4; }
constexpr int kBackwardPack = 4;

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
        a.runs = static_cast<int>(runs_of(q->steps));
        with_type(type, [&](auto element) {
            using T = decltype(element);
            constexpr int V = forward_pack<T>();
            const bool wide = q->channels % V == 0 && rows_aligned(*q, false, x, size, V * size) && rows_aligned(*q, false, y, size, V * size) &&
                aligned(state, V * size) && aligned(final_state, V * size);
            a.packs = static_cast<int>(wide ? q->channels / V : q->channels);
            const int64_t grid = (q->sequences * a.runs * a.packs + kThreads - 1) / kThreads;
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
    if (q == nullptr || q->sequences < 1 || q->channels < 1 || q->steps < 0 || width < 2 || width > 4) return 0;
    const int64_t items = q->sequences * runs_of(q->steps);
    const Layout wide(items, static_cast<int>((q->channels + kBackwardPack - 1) / kBackwardPack)), single(items, static_cast<int>(q->channels));
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
        a.runs = static_cast<int>(runs_of(q->steps));
        with_type(type, [&](auto element) {
            using T = decltype(element);
            constexpr int V = kBackwardPack;
            bool wide = q->channels % V == 0;
            for (const t8b_track_t* t : {&dy, &x, &dx}) wide = wide && rows_aligned(*q, false, *t, size, V * size);
            for (const void* p : {state, final_gradient, static_cast<const void*>(dstate)}) wide = wide && aligned(p, V * size);
            a.packs = static_cast<int>(wide ? q->channels / V : q->channels);
            const Layout l(q->sequences * a.runs, a.packs);
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
            constexpr int V = forward_pack<T>();
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
