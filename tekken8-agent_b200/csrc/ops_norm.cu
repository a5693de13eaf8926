// Layer norm over the last axis, forward and backward.
//
//   y = (x - mean) rstd w + b,   mean = sum(x) / n,   rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//   dx = rstd (g - sum(g)/n - xhat sum(g xhat)/n) + residual gradient,   g = dy w,  xhat = (x - mean) rstd
//   dw = sum over rows of dy xhat,   db = sum over rows of dy
//
// Bound by memory: a pass reads x (and dy) once and writes y (or dx) once. A row of up to 128, 256,
// 512 or 1,024 elements belongs to 8, 16 or 32 lanes of a warp and lies in their registers, 16 or 32
// elements a lane; a longer one (to 8,192) to one block, 32 elements a thread. The statistics are two
// passes over those registers (the mean, then the squares of the differences), so no row is read
// twice and no variance is a difference of large sums. The grid is persistent: a lane keeps its columns' parameters, and in
// the backward pass its columns' sums of dw and db, in registers over all the rows its warp takes;
// the blocks' sums are joined in a fixed order by k_norm_parameters, so results repeat bit for bit.
// Rows of more than 8,192 elements go through the k_wide_* kernels, which read a row again from L2.
#include <algorithm>
#include <atomic>

#include "ops.cuh"

namespace t8b {
namespace op {
namespace {

constexpr int kWarps = 8;          // warps of a block of the forms that give a row to lanes of one warp
constexpr int kThreads = 32 * kWarps;  // and the most threads of a block that shares a row
constexpr int kMostColumns = 32 * kThreads;
constexpr int kWideThreads = 512;  // threads of a block in the forms for rows beyond that
constexpr int kPartialRows = 16;   // rows of threads in k_norm_parameters
// How a row of n elements is shared: by 8, 16 or 32 lanes that hold 16 elements each, by 32 lanes that
// hold 32 (kLong), or by a block whose threads hold 32 (0). The more a thread holds, the fewer
// instructions and barriers an element costs; at 16 elements two blocks of the backward pass are
// resident, at 32 one. 65,536 x 768 in bf16, 32 lanes by 32 against a block by 16: forward 37 / 57 us,
// backward 65 / 79; 8,192 x 8,192, a block by 32 against by 16: 49 / 73, 89 / 96.
constexpr int kLong = 64;
constexpr int group_of(int64_t n) { return n <= 128 ? 8 : n <= 256 ? 16 : n <= 512 ? 32 : n <= 1024 ? kLong : 0; }
__host__ __device__ constexpr int lanes_of(int group) { return group == kLong ? 32 : group; }
__host__ __device__ constexpr int held_of(int group) { return group == kLong || group == 0 ? 32 : 16; }
// Resident blocks: as many as the registers allow (a thread holds w, b and a row forward; w, dw, db and
// two rows backward).
__host__ __device__ constexpr int resident_blocks(int group, bool backward) { return backward && held_of(group) == 32 ? 1 : 2; }

struct Norm {
    const void* x;
    const void* dy;
    const void* residual;
    const void* weight;
    const void* bias;
    void* y;  // y, or dx
    float* mean;
    float* rstd;
    float* partial;  // [2][grid][n]: each block's sums of dw and db
    int64_t rows, x_stride, y_stride, dy_stride, residual_stride;
    int n, parameter_type;
    int shift;  // SHIFT: every matrix's row stride, modulo V
    float epsilon;
};

// Sums over the row's threads: G lanes of a warp, or (G = 0) the block with one barrier (shared
// values alternate between two buffers, so the barrier of the next sum protects those of this one).
template <int G, int COUNT>
__device__ __forceinline__ void row_sum(float (&v)[COUNT], float (*shared)[kWideThreads / 32][2], int& turn) {
#pragma unroll
    for (int o = (G ? G : 32) / 2; o >= 1; o >>= 1) {
#pragma unroll
        for (int k = 0; k < COUNT; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
    if (G) return;
    const int warps = blockDim.x >> 5;
    auto& buffer = shared[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int k = 0; k < COUNT; ++k) buffer[threadIdx.x >> 5][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < COUNT; ++k) v[k] = 0.0f;
    for (int w = 0; w < warps; ++w) {
        const float2 one = *reinterpret_cast<const float2*>(buffer[w]);
        v[0] += one.x;
        if (COUNT == 2) v[COUNT - 1] += one.y;
    }
}

// Thread t of a row's G threads holds the elements of columns (i G + t) V + j - s, i < NV, j < V; what
// of them is not in the row is 0. s is 0 where every row starts on a pack's boundary; with SHIFT it is
// how many elements the row's start lies past one (rows of an odd length: the same for every row that
// a thread takes, since they lie a multiple of V rows apart), so packs are aligned and the first and
// last of a row are shared with its neighbours.
//
// Rows come through a ring of stages in shared memory that a thread fills (cp.async, the same 16 or 8
// bytes that it will read) and reads alone, so the ring needs no barrier and a warp has its next rows
// in flight while it works on one (262,144 x 512 in bf16, when the ring came in: backward 297 -> 205 us,
// forward 123 -> 88; the backward pass takes 133 now). Single elements (V = 1) are read when they are used: 4-byte copies take as
// many instructions as the elements (65,536 x 151 in fp32, backward: 55 us against 37).
template <typename T, int V, int NV, bool SHIFT>
struct Rows {
    static constexpr int kPack = V * sizeof(T);
    static constexpr bool kRing = V > 1;
    const T* from;         // the next row to fetch (or, without a ring, to get)
    int64_t step;          // elements to the row after it
    int first, apart, n;   // this thread's first column, and columns to its next pack
    int at[NV];            // its packs: elements from `from`,
    uint32_t bytes[NV];    // and what to copy of them (the copy fills the rest with 0)

    __device__ __forceinline__ Rows(const void* base, int64_t stride, int64_t row, int64_t rows_apart, int first_column, int apart_, int columns)
        : from(static_cast<const T*>(base) + row * stride), step(rows_apart * stride), first(first_column), apart(apart_), n(columns) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = first + i * apart;
            at[i] = c < n ? c : SHIFT ? first % V : 0;  // a pack past the row copies nothing, from an aligned place
            if (SHIFT && c >= n && at[i] > 0) at[i] -= V;
            bytes[i] = c >= n ? 0 : SHIFT && c + V > n ? (n - c) * sizeof(T) : kPack;
        }
    }
    // slot: this thread's first pack in a stage, consecutive packs `pitch` bytes apart
    __device__ __forceinline__ void fetch(uint32_t slot, int pitch) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (kPack == 16) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot + i * pitch), "l"(from + at[i]), "r"(bytes[i]) : "memory");
            } else if constexpr (kRing) {
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(slot + i * pitch), "l"(from + at[i]), "r"(bytes[i]) : "memory");
            }
        }
        from += step;
    }
    // A pair of a pack that starts at column c: what lies before the row is not its own.
    __device__ __forceinline__ Two own(float2 f, int i, int j) const {
        if (SHIFT && i == 0) {
            if (first + 2 * j < 0) f.x = 0.0f;
            if (first + 2 * j + 1 < 0) f.y = 0.0f;
        }
        return Two(f.x, f.y);
    }
    __device__ __forceinline__ void get(const unsigned char* slot, int pitch, Two (&v)[NV * V / 2]) {
        if constexpr (kRing) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if constexpr (sizeof(T) == 2) {
                    const Pack<uint32_t, V / 2> p = *reinterpret_cast<const Pack<uint32_t, V / 2>*>(slot + i * pitch);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) v[i * (V / 2) + j] = own(Element<T>::unpack(p.v[j]), i, j);
                } else {
                    const Pack<float, V> p = *reinterpret_cast<const Pack<float, V>*>(slot + i * pitch);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) v[i * (V / 2) + j] = own(make_float2(p.v[2 * j], p.v[2 * j + 1]), i, j);
                }
            }
        } else {
            T raw[NV];
            float f[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {  // the loads first, all in flight
                raw[i] = Element<T>::store(0.0f);
                if (first + i * apart < n) raw[i] = from[first + i * apart];
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) f[i] = Element<T>::load(raw[i]);
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) v[i] = Two(f[2 * i], f[2 * i + 1]);
            from += step;
        }
    }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void ring_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
// Stages of a ring of `bytes` a thread and a stage: two blocks of 256 threads fit an SM, and more
// than two rows ahead gained nothing (262,144 x 512 forward in bf16: 88 us, with three 99).
constexpr int ring_stages(int bytes) { return bytes == 0 || 384 / bytes < 3 ? 2 : 3; }

// to: the row
template <typename T, int V, int NV, bool SHIFT>
__device__ __forceinline__ void store_row(T* to, int first, int apart, int n, const Two (&v)[NV * V / 2]) {
    if constexpr (V == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float2 f = v[i / 2].get();
            if (first + i * apart < n) to[first + i * apart] = Element<T>::store(i % 2 ? f.y : f.x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = first + i * apart;
            if (c >= n) continue;
            if (SHIFT && (c < 0 || c + V > n)) {  // shared with a neighbouring row
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 f = v[(i * V + j) / 2].get();
                    if (c + j >= 0 && c + j < n) to[c + j] = Element<T>::store(j % 2 ? f.y : f.x);
                }
                continue;
            }
            if constexpr (sizeof(T) == 2) {
                Pack<uint32_t, V / 2> p;
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float2 f = v[i * (V / 2) + j].get();
                    p.v[j] = Element<T>::pack(f.x, f.y);
                }
                *reinterpret_cast<Pack<uint32_t, V / 2>*>(to + c) = p;
            } else {
                Pack<float, V> p;
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float2 f = v[i * (V / 2) + j].get();
                    p.v[2 * j] = f.x;
                    p.v[2 * j + 1] = f.y;
                }
                *reinterpret_cast<Pack<float, V>*>(to + c) = p;
            }
        }
    }
}
template <int V, int NV>
__device__ __forceinline__ void load_parameter(const void* p, int type, float missing, int first, int apart, int n,
                                               Two (&v)[NV * V / 2]) {
    float f[NV * V];
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
        const int c = first + (i / V) * apart + i % V;
        f[i] = p != nullptr && c >= 0 && c < n ? load_any(p, type, c) : missing;
    }
#pragma unroll
    for (int i = 0; i < NV * V / 2; ++i) v[i] = Two(f[2 * i], f[2 * i + 1]);
}

template <typename TX, int V, int NV>
struct ForwardRing {
    static constexpr int kBytes = V > 1 ? NV * V * static_cast<int>(sizeof(TX)) : 0;  // of a thread and a stage
    static constexpr int kStages = ring_stages(kBytes);
};
template <typename TX, typename TY, int V, int NV>
struct BackwardRing {
    static constexpr int kX = ForwardRing<TX, V, NV>::kBytes, kDy = ForwardRing<TY, V, NV>::kBytes;
    static constexpr int kBytes = 2 * kX + kDy;
    static constexpr int kStages = ring_stages(kBytes);
};

// Where this thread stands: thread t of the `group` that shares a row, on the block's rows first,
// first + step and so on, `mine` of them; the warp goes on for `turns` rows (a row of fewer than 32
// lanes may end before its warp does: the sums take every lane).
template <int G>
struct Seat {
    static constexpr bool kWarp = G != 0;
    static constexpr int kPerWarp = kWarp ? 32 / (kWarp ? G : 1) : 1;
    int group, t, row, rows, mine, turns;
    int64_t first, step;
    __device__ __forceinline__ explicit Seat(int64_t total)
        : group(kWarp ? G : blockDim.x), t(kWarp ? threadIdx.x % (kWarp ? G : 1) : threadIdx.x),
          row(kWarp ? threadIdx.x / (kWarp ? G : 1) : 0), rows(kWarp ? blockDim.x / (kWarp ? G : 1) : 1) {
        first = static_cast<int64_t>(blockIdx.x) * rows + row;
        step = static_cast<int64_t>(gridDim.x) * rows;
        mine = count(first, total);
        turns = count(first - row % kPerWarp, total);
    }
    __device__ __forceinline__ int count(int64_t from, int64_t total) const {
        return from < total ? static_cast<int>((total - from + step - 1) / step) : 0;
    }
};

template <typename TX, typename TY, int V, bool SHIFT, int G>
__global__ void __launch_bounds__(kThreads, resident_blocks(G, false)) k_norm_forward(Norm a) {
    constexpr int HELD = held_of(G), LANES = lanes_of(G);
    constexpr int NV = HELD / V;
    using Ring = ForwardRing<TX, V, NV>;
    constexpr int S = Ring::kStages;
    wait_previous();
    release_next();
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ __align__(8) float shared[2][kWideThreads / 32][2];
    int turn = 0;
    const Seat<LANES> seat(a.rows);
    const int at = seat.t * V - (SHIFT ? static_cast<int>(seat.first % V * a.shift % V) : 0), apart = seat.group * V;
    Rows<TX, V, NV, SHIFT> x(a.x, a.x_stride, seat.first, seat.step, at, apart, a.n);
    const int pitch = blockDim.x * V * static_cast<int>(sizeof(TX)), stage_bytes = blockDim.x * Ring::kBytes;
    const unsigned char* mine = ring + threadIdx.x * V * sizeof(TX);
    const uint32_t slot = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
    if (Ring::kBytes) {
#pragma unroll
        for (int k = 0; k < S - 1; ++k) {
            if (k < seat.mine) x.fetch(slot + k * stage_bytes, pitch);
            ring_commit();
        }
    }
    Two w[HELD / 2], b[HELD / 2];
    load_parameter<V, NV>(a.weight, a.parameter_type, 1.0f, at, apart, a.n, w);
    load_parameter<V, NV>(a.bias, a.parameter_type, 0.0f, at, apart, a.n, b);
    const float scale = 1.0f / static_cast<float>(a.n);
    const bool whole = !SHIFT && a.n == seat.group * HELD;  // every thread holds as many elements as it can
    TY* y = static_cast<TY*>(a.y) + seat.first * a.y_stride;
    const int64_t y_step = seat.step * a.y_stride;
    const auto outside = [&](int e) {  // whether held element e is not the row's
        const int c = at + (e / V) * apart;
        return SHIFT ? c + e % V < 0 || c + e % V >= a.n : c >= a.n;
    };
    float* to_mean = a.mean ? a.mean + seat.first : nullptr;
    float* to_rstd = a.rstd ? a.rstd + seat.first : nullptr;
    int stage = 0;
    for (int k = 0; k < seat.turns; ++k, y += y_step) {
        const bool live = k < seat.mine;
        Two v[HELD / 2];
        if (Ring::kBytes) {
            if (k + S - 1 < seat.mine) x.fetch(slot + (stage == 0 ? S - 1 : stage - 1) * stage_bytes, pitch);
            ring_commit();
            ring_wait<S - 1>();
        }
        if (Ring::kBytes || live) x.get(mine + stage * stage_bytes, pitch, v);
        stage = stage == S - 1 ? 0 : stage + 1;
        Two total;
#pragma unroll
        for (int i = 0; i < HELD / 2; ++i) total = total + v[i];
        float sum[1] = {total.sum()};
        row_sum<LANES>(sum, shared, turn);
        const float mean = sum[0] * scale;
        const Two off(-mean, -mean);
        Two squared;
        if (whole) {
#pragma unroll
            for (int i = 0; i < HELD / 2; ++i) {
                v[i] = v[i] + off;
                squared = multiply_add(v[i], v[i], squared);
            }
        } else {
#pragma unroll
            for (int i = 0; i < HELD / 2; ++i) {
                float2 d = (v[i] + off).get();
                if (outside(2 * i)) d.x = 0.0f;
                if (outside(2 * i + 1)) d.y = 0.0f;
                v[i] = Two(d.x, d.y);
                squared = multiply_add(v[i], v[i], squared);
            }
        }
        float squares[1] = {squared.sum()};
        row_sum<LANES>(squares, shared, turn);
        const float rstd = rsqrtf(squares[0] * scale + a.epsilon);
        const Two scaled(rstd, rstd);
#pragma unroll
        for (int i = 0; i < HELD / 2; ++i) v[i] = multiply_add(v[i] * scaled, w[i], b[i]);
        if (!live) continue;
        store_row<TY, V, NV, SHIFT>(y, at, apart, a.n, v);
        if (seat.t == 0) {
            if (to_mean) to_mean[k * seat.step] = mean;
            if (to_rstd) to_rstd[k * seat.step] = rstd;
        }
    }
    ring_wait<0>();
}

template <typename TX, typename TY, int V, bool SHIFT, int G>
__global__ void __launch_bounds__(kThreads, resident_blocks(G, true)) k_norm_backward(Norm a) {
    constexpr int HELD = held_of(G), LANES = lanes_of(G);
    constexpr int NV = HELD / V;
    using Ring = BackwardRing<TX, TY, V, NV>;
    constexpr int S = Ring::kStages;
    wait_previous();
    release_next();
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ __align__(8) float shared[2][kWideThreads / 32][2];
    int turn = 0;
    const Seat<LANES> seat(a.rows);
    const int at = seat.t * V - (SHIFT ? static_cast<int>(seat.first % V * a.shift % V) : 0), apart = seat.group * V;
    Rows<TX, V, NV, SHIFT> x(a.x, a.x_stride, seat.first, seat.step, at, apart, a.n);
    Rows<TX, V, NV, SHIFT> residual(a.residual, a.residual_stride, seat.first, seat.step, at, apart, a.n);
    Rows<TY, V, NV, SHIFT> dy(a.dy, a.dy_stride, seat.first, seat.step, at, apart, a.n);
    const int x_pitch = blockDim.x * V * static_cast<int>(sizeof(TX)), dy_pitch = blockDim.x * V * static_cast<int>(sizeof(TY));
    const int stage_bytes = blockDim.x * Ring::kBytes;
    // a stage: x, residual, dy
    const unsigned char* mine_x = ring + threadIdx.x * V * sizeof(TX);
    const unsigned char* mine_dy = ring + 2 * blockDim.x * Ring::kX + threadIdx.x * V * sizeof(TY);
    const int residual_at = blockDim.x * Ring::kX;
    const uint32_t slot_x = static_cast<uint32_t>(__cvta_generic_to_shared(mine_x));
    const uint32_t slot_dy = static_cast<uint32_t>(__cvta_generic_to_shared(mine_dy));
    auto fetch = [&](int stage, bool any) {
        if (!Ring::kBytes) return;
        if (any) {
            x.fetch(slot_x + stage * stage_bytes, x_pitch);
            dy.fetch(slot_dy + stage * stage_bytes, dy_pitch);
            if (a.residual) residual.fetch(slot_x + residual_at + stage * stage_bytes, x_pitch);
        }
        ring_commit();
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) fetch(k, k < seat.mine);
    // the statistics of this row and the next two
    const float* from_mean = a.mean + seat.first;
    const float* from_rstd = a.rstd + seat.first;
    float means[2] = {0.0f, 0.0f}, rstds[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (k < seat.mine) {
            means[k] = from_mean[k * seat.step];
            rstds[k] = from_rstd[k * seat.step];
        }
    }
    from_mean += 2 * seat.step;
    from_rstd += 2 * seat.step;
    Two w[HELD / 2], dw[HELD / 2], db[HELD / 2];
    load_parameter<V, NV>(a.weight, a.parameter_type, 1.0f, at, apart, a.n, w);
    const float scale = 1.0f / static_cast<float>(a.n);
    TX* dx = static_cast<TX*>(a.y) + seat.first * a.y_stride;
    const int64_t dx_step = seat.step * a.y_stride;
    int stage = 0;
    for (int k = 0; k < seat.turns; ++k, dx += dx_step) {
        const bool live = k < seat.mine;
        fetch(stage == 0 ? S - 1 : stage - 1, k + S - 1 < seat.mine);
        const float mean = means[0], rstd = rstds[0];
        means[0] = means[1];
        rstds[0] = rstds[1];
        if (k + 2 < seat.mine) {
            means[1] = *from_mean;
            rstds[1] = *from_rstd;
            from_mean += seat.step;
            from_rstd += seat.step;
        }
        if (Ring::kBytes) ring_wait<S - 1>();
        Two v[HELD / 2], g[HELD / 2];
        if (live) {
            x.get(mine_x + stage * stage_bytes, x_pitch, v);
            dy.get(mine_dy + stage * stage_bytes, dy_pitch, g);
        }
        Two of_g, of_gx;
        {
            const Two off(-mean, -mean), scaled(rstd, rstd);
#pragma unroll
            for (int i = 0; i < HELD / 2; ++i) {
                // Beyond the row x and dy are 0 and add 0 to every sum. sum(g xhat) is rstd times sum(g
                // (x - mean)): a product with xhat would be 0 * inf there where mean * rstd overflows.
                const Two given = g[i];
                v[i] = v[i] + off;
                db[i] = db[i] + given;
                g[i] = given * w[i];
                of_g = of_g + g[i];
                of_gx = multiply_add(g[i], v[i], of_gx);
                v[i] = v[i] * scaled;
                if (live) dw[i] = multiply_add(given, v[i], dw[i]);
            }
        }
        float sum[2] = {of_g.sum(), of_gx.sum() * rstd};
        row_sum<LANES>(sum, shared, turn);
        if (live) {
            const float c0 = -rstd * (sum[0] * scale), c1 = -rstd * (sum[1] * scale);
            const Two of_one(c0, c0), of_x(c1, c1), of_dy(rstd, rstd);
#pragma unroll
            for (int i = 0; i < HELD / 2; ++i) v[i] = multiply_add(g[i], of_dy, multiply_add(v[i], of_x, of_one));
            if (a.residual) {
                residual.get(mine_x + residual_at + stage * stage_bytes, x_pitch, g);
#pragma unroll
                for (int i = 0; i < HELD / 2; ++i) v[i] = v[i] + g[i];
            }
            store_row<TX, V, NV, SHIFT>(dx, at, apart, a.n, v);
        }
        stage = stage == S - 1 ? 0 : stage + 1;
    }
    ring_wait<0>();
    if (a.partial == nullptr) return;
    float* out = a.partial + static_cast<size_t>(blockIdx.x) * a.n;
    if (G) {
        // the rows' sums meet in shared memory, over the ring: [rows of the block][group HELD]
        float* joined = reinterpret_cast<float*>(ring);
        const int width = LANES * HELD;
#pragma unroll
        for (int which = 0; which < 2; ++which, out += static_cast<size_t>(gridDim.x) * a.n) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const float2 pair = (which ? db[i / 2] : dw[i / 2]).get();
                const int c = at + (i / V) * apart + i % V;
                if (c >= 0 && c < a.n) joined[seat.row * width + c] = i % 2 ? pair.y : pair.x;
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
                float v = 0.0f;
                for (int k = 0; k < seat.rows; ++k) v += joined[k * width + c];
                out[c] = v;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = at + (i / V) * apart + i % V;
            const float2 w2 = dw[i / 2].get(), b2 = db[i / 2].get();
            if (c >= 0 && c < a.n) {
                out[c] = i % 2 ? w2.y : w2.x;
                out[static_cast<size_t>(gridDim.x) * a.n + c] = i % 2 ? b2.y : b2.x;
            }
        }
    }
}

// dw and db from the blocks' sums, in a fixed order. Block (32, kPartialRows): 32 columns.
__global__ void k_norm_parameters(const float* partial, int count, int n, void* dw, void* db, int type) {
    wait_previous();
    release_next();
    __shared__ float sums[kPartialRows][33];
    void* out = blockIdx.y ? db : dw;
    if (out == nullptr) return;
    const int c = blockIdx.x * 32 + threadIdx.x;
    const float* p = partial + static_cast<size_t>(blockIdx.y) * count * n;
    float v = 0.0f;
    if (c < n) {
#pragma unroll 4
        for (int r = threadIdx.y; r < count; r += kPartialRows) v += p[static_cast<size_t>(r) * n + c];
    }
    sums[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y != 0 || c >= n) return;
#pragma unroll
    for (int r = 1; r < kPartialRows; ++r) v += sums[r][threadIdx.x];
    store_any(out, type, c, v);
}

// ------------------------------------------------------------------ rows beyond 8,192 elements
__device__ __forceinline__ float block_sum(float v, float (*shared)[kWideThreads / 32][2], int& turn) {
    float s[1] = {v};
    row_sum<0>(s, shared, turn);
    return s[0];
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kWideThreads) k_wide_forward(Norm a) {
    __shared__ __align__(8) float shared[2][kWideThreads / 32][2];
    int turn = 0;
    const float scale = 1.0f / static_cast<float>(a.n);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
        TY* y = static_cast<TY*>(a.y) + row * a.y_stride;
        float v = 0.0f;
        for (int c = threadIdx.x; c < a.n; c += kWideThreads) v += Element<TX>::load(x[c]);
        const float mean = block_sum(v, shared, turn) * scale;
        v = 0.0f;
        for (int c = threadIdx.x; c < a.n; c += kWideThreads) {
            const float d = Element<TX>::load(x[c]) - mean;
            v += d * d;
        }
        const float rstd = rsqrtf(block_sum(v, shared, turn) * scale + a.epsilon);
        for (int c = threadIdx.x; c < a.n; c += kWideThreads) {
            const float w = a.weight ? load_any(a.weight, a.parameter_type, c) : 1.0f;
            const float b = a.bias ? load_any(a.bias, a.parameter_type, c) : 0.0f;
            y[c] = Element<TY>::store((Element<TX>::load(x[c]) - mean) * rstd * w + b);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// dx alone; k_wide_columns sums the parameters' gradients.
template <typename TX, typename TY>
__global__ void __launch_bounds__(kWideThreads) k_wide_backward(Norm a) {
    __shared__ __align__(8) float shared[2][kWideThreads / 32][2];
    int turn = 0;
    const float scale = 1.0f / static_cast<float>(a.n);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
        const TY* dy = static_cast<const TY*>(a.dy) + row * a.dy_stride;
        const TX* residual = a.residual ? static_cast<const TX*>(a.residual) + row * a.residual_stride : nullptr;
        TX* dx = static_cast<TX*>(a.y) + row * a.y_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum[2] = {0.0f, 0.0f};
        for (int c = threadIdx.x; c < a.n; c += kWideThreads) {
            const float w = a.weight ? load_any(a.weight, a.parameter_type, c) : 1.0f;
            const float g = Element<TY>::load(dy[c]) * w;
            sum[0] += g;
            sum[1] += g * ((Element<TX>::load(x[c]) - mean) * rstd);
        }
        row_sum<0>(sum, shared, turn);
        const float of_g = sum[0] * scale, of_gx = sum[1] * scale;
        for (int c = threadIdx.x; c < a.n; c += kWideThreads) {
            const float w = a.weight ? load_any(a.weight, a.parameter_type, c) : 1.0f;
            const float g = Element<TY>::load(dy[c]) * w;
            const float h = (Element<TX>::load(x[c]) - mean) * rstd;
            float v = rstd * (g - of_g - h * of_gx);
            if (residual) v += Element<TX>::load(residual[c]);
            dx[c] = Element<TX>::store(v);
        }
    }
}

// Grid (column blocks, row parts): one thread a column, one part of the rows a block row.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256) k_wide_columns(Norm a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.n) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = Element<TY>::load(static_cast<const TY*>(a.dy)[row * a.dy_stride + c]);
        dw += g * ((Element<TX>::load(static_cast<const TX*>(a.x)[row * a.x_stride + c]) - a.mean[row]) * a.rstd[row]);
        db += g;
    }
    a.partial[static_cast<size_t>(blockIdx.y) * a.n + c] = dw;
    a.partial[(static_cast<size_t>(gridDim.y) + blockIdx.y) * a.n + c] = db;
}

// ------------------------------------------------------------------ dispatch
int multiprocessors() {
    static std::atomic<int> counts[64];
    int device = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    int count = counts[device & 63].load(std::memory_order_relaxed);
    if (count == 0) {
        check(cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device), "SM count");
        counts[device & 63].store(count, std::memory_order_relaxed);
    }
    return count;
}

// Threads and rows in flight of a block, and the grid: what is resident at once, and no more than
// there are rows to take; `n` counts what a row's threads have to hold, shift included.
int threads_of(int64_t n) { return group_of(n) ? kThreads : static_cast<int>(round_up((n + 31) / 32, 32)); }
int blocks_of(int64_t rows, int64_t n, bool backward, int sms) {
    const int group = group_of(n);
    const int64_t in_flight = group ? kThreads / lanes_of(group) : 1;
    const int64_t resident = sms * resident_blocks(group, backward) * (kThreads / threads_of(n));
    const int64_t want = (rows + in_flight - 1) / in_flight;
    // a block's next row is a multiple of 8 rows on, whatever V is
    return static_cast<int>(std::max<int64_t>(1, want <= resident ? want : in_flight == 1 ? resident / 8 * 8 : resident));
}
constexpr int kWideBlocks = 64;

// The blocks whose sums of dw and db a backward pass leaves.
template <typename TX, typename TY, int V, bool SHIFT, int G>
int launch_norm(const Norm& a, bool backward, int sms, cudaStream_t stream) {
    const int64_t held = a.n + (SHIFT ? V - 1 : 0);
    const int threads = threads_of(held), grid = blocks_of(a.rows, held, backward, sms);
    if (backward) {
        using Ring = BackwardRing<TX, TY, V, held_of(G) / V>;
        constexpr int kJoined = G ? kThreads * held_of(G) * 4 : 0;
        static uint64_t configured = 0;
        allow_smem(k_norm_backward<TX, TY, V, SHIFT, G>, std::max(Ring::kStages * Ring::kBytes * kThreads, kJoined), configured);
        launch_chain("k_norm_backward", k_norm_backward<TX, TY, V, SHIFT, G>, grid, threads,
                     std::max(Ring::kStages * Ring::kBytes * threads, kJoined), stream, true, a);
    } else {
        using Ring = ForwardRing<TX, V, held_of(G) / V>;
        static uint64_t configured = 0;
        allow_smem(k_norm_forward<TX, TY, V, SHIFT, G>, Ring::kStages * Ring::kBytes * kThreads, configured);
        launch_chain("k_norm_forward", k_norm_forward<TX, TY, V, SHIFT, G>, grid, threads, Ring::kStages * Ring::kBytes * threads,
                     stream, true, a);
    }
    return grid;
}

template <typename TX, typename TY, int V, bool SHIFT>
int run(const Norm& a, bool backward, int sms, cudaStream_t stream) {
    const int group = group_of(a.n + (SHIFT ? V - 1 : 0));
    if constexpr (!SHIFT) {
        if (group == 8) return launch_norm<TX, TY, V, SHIFT, 8>(a, backward, sms, stream);
        if (group == 16) return launch_norm<TX, TY, V, SHIFT, 16>(a, backward, sms, stream);
    }
    switch (group) {
        case 32: return launch_norm<TX, TY, V, SHIFT, 32>(a, backward, sms, stream);
        case kLong: return launch_norm<TX, TY, V, SHIFT, kLong>(a, backward, sms, stream);
        default: return launch_norm<TX, TY, V, SHIFT, 0>(a, backward, sms, stream);
    }
}

template <typename TX, typename TY>
int norm(const Norm& given, bool backward, cudaStream_t stream) {
    Norm a = given;
    const int sms = multiprocessors();
    if (a.n > kMostColumns) {
        const int grid = static_cast<int>(std::min<int64_t>(a.rows, sms * 4)), parts = static_cast<int>(std::min<int64_t>(a.rows, kWideBlocks));
        if (!backward) {
            launch("k_norm_forward", k_wide_forward<TX, TY>, grid, kWideThreads, 0, stream, a);
            return grid;
        }
        if (a.partial) launch("k_norm_columns", k_wide_columns<TX, TY>, dim3(blocks(a.n, 256), parts), 256, 0, stream, a);
        launch("k_norm_backward", k_wide_backward<TX, TY>, grid, kWideThreads, 0, stream, a);
        return parts;
    }
    // 16 bytes a lane of the wider type where every matrix starts on its vector's boundary: as they
    // lie where every row does too; shifted where the rows' starts differ from it alike in all of them
    // and rows are longer than 256; single elements otherwise. Shifted against single, us, bf16:
    // 20,000 x 3,001 forward 71 / 95, backward 111 / 155; 40,000 x 801 44 / 39, 56 / 66; 100,000 x 333 48 / 53,
    // 71 / 67; 65,536 x 151 17.6 / 15.2, 27.7 / 24.6; fp32: 100,000 x 333 47 / 59, 70 / 76.
    constexpr int V = 16 / (sizeof(TX) > sizeof(TY) ? sizeof(TX) : sizeof(TY));
    const size_t ys = backward ? sizeof(TX) : sizeof(TY);
    const bool bases = aligned(a.x, V * sizeof(TX)) && aligned(a.dy, V * sizeof(TY)) && aligned(a.residual, V * sizeof(TX)) && aligned(a.y, V * ys);
    if (a.rows == 1) a.x_stride = a.y_stride = a.dy_stride = a.residual_stride = 0;
    a.shift = static_cast<int>(a.x_stride % V);
    const bool alike = a.y_stride % V == a.shift && (a.dy == nullptr || a.dy_stride % V == a.shift) &&
        (a.residual == nullptr || a.residual_stride % V == a.shift);
    if (bases && alike && a.shift == 0 && a.n % V == 0) return run<TX, TY, V, false>(a, backward, sms, stream);
    if (bases && alike && a.n > 256 && a.n + V - 1 <= kMostColumns) return run<TX, TY, V, true>(a, backward, sms, stream);
    return run<TX, TY, 1, false>(a, backward, sms, stream);
}

template <typename TX>
int norm_y(const Norm& a, int y_type, bool backward, cudaStream_t stream) {
    if (y_type == T8B_F32) return norm<TX, float>(a, backward, stream);
    if (y_type == T8B_BF16) return norm<TX, bf16>(a, backward, stream);
    return norm<TX, f16>(a, backward, stream);
}

int dispatch(const Norm& a, int x_type, int y_type, bool backward, cudaStream_t stream) {
    if (x_type == T8B_F32) return norm_y<float>(a, y_type, backward, stream);
    if (x_type == T8B_BF16) return norm_y<bf16>(a, y_type, backward, stream);
    return norm_y<f16>(a, y_type, backward, stream);
}

void check_sizes(int64_t rows, int64_t n) {
    if (rows < 0 || rows > (1ll << 32)) raise(T8B_EINVAL, "layer norm: rows from 0 to 4294967296");
    if (n < 1 || n > (1 << 24)) raise(T8B_EINVAL, "layer norm: rows have 1 to 16777216 elements");
}

}  // namespace
}  // namespace op
}  // namespace t8b

using namespace t8b;
using namespace t8b::op;

extern "C" int t8b_layer_norm_forward(const void* x, int x_type, int64_t x_stride, const void* weight, const void* bias,
                                      int parameter_type, float epsilon, int64_t rows, int64_t n, void* y, int y_type,
                                      int64_t y_stride, float* mean, float* rstd, void* stream) {
    return guarded([&] {
        check_sizes(rows, n);
        if (!is_type(x_type) || !is_type(y_type) || !is_type(parameter_type)) raise(T8B_EINVAL, "layer norm: unknown type");
        if (!(epsilon >= 0.0f) || epsilon > std::numeric_limits<float>::max()) {
            raise(T8B_EINVAL, "layer norm: epsilon must be finite and not negative");
        }
        check_matrix("layer norm x", x, rows, n, x_stride, type_size(x_type));
        check_matrix("layer norm y", y, rows, n, y_stride, type_size(y_type));
        for (const void* vector : {weight, bias}) check_elements("layer norm parameters", vector, type_size(parameter_type));
        for (const float* vector : {mean, rstd}) check_elements("layer norm mean and rstd", vector, sizeof(float));
        if (rows == 0) return;
        const Span to(y, rows, n, y_stride, type_size(y_type)), from(x, rows, n, x_stride, type_size(x_type));
        if (to.overlaps(from) && !(x == y && x_stride == y_stride && x_type == y_type && n <= kMostColumns)) {
            raise(T8B_EINVAL, "layer norm: y may be x itself in rows of up to 8192 elements, and overlap it in no other way");
        }
        Norm a{};
        a.x = x;
        a.weight = weight;
        a.bias = bias;
        a.y = y;
        a.mean = mean;
        a.rstd = rstd;
        a.rows = rows;
        a.x_stride = x_stride;
        a.y_stride = y_stride;
        a.n = static_cast<int>(n);
        a.parameter_type = parameter_type;
        a.epsilon = epsilon;
        dispatch(a, x_type, y_type, false, static_cast<cudaStream_t>(stream));
        check(cudaGetLastError(), "layer norm launch");
    });
}

extern "C" size_t t8b_layer_norm_workspace(int64_t rows, int64_t n) {
    if (rows < 1 || n < 1) return 0;
    // the most blocks of any form, on any device of up to 256 multiprocessors, so that it needs none to answer
    int most = kWideBlocks;
    if (n <= kMostColumns) most = std::max(blocks_of(rows, n, true, 256), blocks_of(rows, n + 7, true, 256));
    return static_cast<size_t>(2) * most * static_cast<size_t>(n) * sizeof(float);
}

extern "C" int t8b_layer_norm_backward(const void* dy, int y_type, int64_t dy_stride, const void* x, int x_type,
                                       int64_t x_stride, const void* weight, int parameter_type, const float* mean,
                                       const float* rstd, const void* residual_gradient, int64_t residual_stride,
                                       int64_t rows, int64_t n, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(rows, n);
        if (!is_type(x_type) || !is_type(y_type) || !is_type(parameter_type)) raise(T8B_EINVAL, "layer norm: unknown type");
        const size_t xs = type_size(x_type), ys = type_size(y_type);
        check_matrix("layer norm dy", dy, rows, n, dy_stride, ys);
        check_matrix("layer norm x", x, rows, n, x_stride, xs);
        check_matrix("layer norm dx", dx, rows, n, dx_stride, xs);
        if (residual_gradient) check_matrix("layer norm residual gradient", residual_gradient, rows, n, residual_stride, xs);
        for (const void* vector : {weight, static_cast<const void*>(dweight), static_cast<const void*>(dbias)}) {
            check_elements("layer norm parameters", vector, type_size(parameter_type));
        }
        for (const float* vector : {mean, rstd}) check_elements("layer norm mean and rstd", vector, sizeof(float));
        if (rows > 0 && (mean == nullptr || rstd == nullptr)) raise(T8B_EINVAL, "layer norm: mean and rstd are null");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const bool parameters = dweight != nullptr || dbias != nullptr;
        if (rows == 0) {
            if (dweight) check(cudaMemsetAsync(dweight, 0, n * type_size(parameter_type), st), "clear dweight");
            if (dbias) check(cudaMemsetAsync(dbias, 0, n * type_size(parameter_type), st), "clear dbias");
            return;
        }
        const Span to(dx, rows, n, dx_stride, xs);
        if (to.overlaps(Span(x, rows, n, x_stride, xs)) || to.overlaps(Span(dy, rows, n, dy_stride, ys)) ||
            to.overlaps(Span(residual_gradient, rows, n, residual_stride, xs))) {
            raise(T8B_EINVAL, "layer norm: dx overlaps an input");
        }
        if (parameters && (workspace == nullptr || workspace_bytes < t8b_layer_norm_workspace(rows, n) || !aligned(workspace, 16))) {
            raise(T8B_EINVAL, "layer norm: the workspace is missing, unaligned or smaller than t8b_layer_norm_workspace");
        }
        Norm a{};
        a.x = x;
        a.dy = dy;
        a.residual = residual_gradient;
        a.weight = weight;
        a.y = dx;
        a.mean = const_cast<float*>(mean);
        a.rstd = const_cast<float*>(rstd);
        a.partial = parameters ? static_cast<float*>(workspace) : nullptr;
        a.rows = rows;
        a.x_stride = x_stride;
        a.y_stride = dx_stride;
        a.dy_stride = dy_stride;
        a.residual_stride = residual_stride;
        a.n = static_cast<int>(n);
        a.parameter_type = parameter_type;
        const int count = dispatch(a, x_type, y_type, true, st);
        if (parameters) {
            launch_chain("k_norm_parameters", k_norm_parameters, dim3(blocks(n, 32), 2), dim3(32, kPartialRows), 0, st, true,
                         static_cast<const float*>(workspace), count, a.n, dweight, dbias,
                         parameter_type);
        }
        check(cudaGetLastError(), "layer norm launch");
    });
}
