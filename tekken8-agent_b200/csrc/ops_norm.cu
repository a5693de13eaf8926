// Layer norm over the last axis, forward and backward.
//
//   y = (x - mean) rstd w + b,   mean = sum(x) / n,   rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//   dx = rstd (g - sum(g)/n - xhat sum(g xhat)/n) + residual gradient,   g = dy w,  xhat = (x - mean) rstd
//   dw = sum over rows of dy xhat,   db = sum over rows of dy
//
// Bound by memory: a pass reads x (and dy) once and writes y (or dx) once. A row of up to 512
// elements belongs to one warp and lies in its registers, 16 elements a lane; a longer one (to
// 8,192) to one block, 16 elements a thread. The statistics are two passes over those registers
// (the mean, then the squares of the differences), so no row is read twice and no variance is a
// difference of large sums. The grid is persistent: a lane keeps its columns' parameters, and in
// the backward pass its columns' sums of dw and db, in registers over all the rows its warp takes;
// the blocks' sums are joined in a fixed order by k_norm_parameters, so results repeat bit for bit.
// Rows of more than 8,192 elements go through the k_wide_* kernels, which read a row again from L2.
#include <algorithm>

#include "ops.cuh"

namespace t8b {
namespace op {
namespace {

constexpr int kHeld = 16;        // elements of a row that one thread holds
constexpr int kWarps = 8;        // warps (rows in flight) of a block in the warp form
constexpr int kBlockMax = 512;   // threads of a block in the block form
constexpr int kPartialRows = 16; // rows of threads in k_norm_parameters

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
    float epsilon;
};

// Sums a (and b) over the row's threads: a warp, or the block with one barrier (shared values
// alternate between two buffers, so the barrier of the next sum protects those of this one).
template <bool WARP, int COUNT>
__device__ __forceinline__ void row_sum(float (&v)[COUNT], float (*shared)[kBlockMax / 32][2], int& turn) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
#pragma unroll
        for (int k = 0; k < COUNT; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
    if (WARP) return;
    const int warps = blockDim.x >> 5;
    auto& buffer = shared[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int k = 0; k < COUNT; ++k) buffer[threadIdx.x >> 5][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
        float sum = 0.0f;
        for (int w = 0; w < warps; ++w) sum += buffer[w][k];
        v[k] = sum;
    }
}

// Thread t of a row's G threads holds elements (i G + t) V + j, i < NV, j < V.
template <typename T, int V, int NV>
__device__ __forceinline__ void load_row(const T* row, int t, int group, int n, float (&v)[NV * V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * group + t) * V;
        Pack<T, V> p;
        const bool in = c < n;
        if (in) p = *reinterpret_cast<const Pack<T, V>*>(row + c);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i * V + j] = in ? Element<T>::load(p.v[j]) : 0.0f;
    }
}
template <typename T, int V, int NV>
__device__ __forceinline__ void store_row(T* row, int t, int group, int n, const float (&v)[NV * V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * group + t) * V;
        if (c < n) {
            Pack<T, V> p;
#pragma unroll
            for (int j = 0; j < V; ++j) p.v[j] = Element<T>::store(v[i * V + j]);
            *reinterpret_cast<Pack<T, V>*>(row + c) = p;
        }
    }
}
template <int V, int NV>
__device__ __forceinline__ void load_parameter(const void* p, int type, float missing, int t, int group, int n,
                                               float (&v)[NV * V]) {
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
        const int c = ((i / V) * group + t) * V + i % V;
        v[i] = p != nullptr && c < n ? load_any(p, type, c) : missing;
    }
}

template <typename TX, typename TY, int V, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarps : kBlockMax) k_norm_forward(Norm a) {
    __shared__ float shared[2][kBlockMax / 32][2];
    int turn = 0;
    const int group = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
    float w[NV * V], b[NV * V];
    load_parameter<V, NV>(a.weight, a.parameter_type, 1.0f, t, group, a.n, w);
    load_parameter<V, NV>(a.bias, a.parameter_type, 0.0f, t, group, a.n, b);
    const float scale = 1.0f / static_cast<float>(a.n);
    for (int64_t row = first; row < a.rows; row += step) {
        float v[NV * V];
        load_row<TX, V, NV>(static_cast<const TX*>(a.x) + row * a.x_stride, t, group, a.n, v);
        float sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV * V; ++i) sum[0] += v[i];
        row_sum<WARP>(sum, shared, turn);
        const float mean = sum[0] * scale;
        float squares[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV * V; ++i) {
            const int c = ((i / V) * group + t) * V;
            v[i] = v[i] - mean;
            if (c < a.n) squares[0] += v[i] * v[i];
        }
        row_sum<WARP>(squares, shared, turn);
        const float rstd = rsqrtf(squares[0] * scale + a.epsilon);
#pragma unroll
        for (int i = 0; i < NV * V; ++i) v[i] = v[i] * rstd * w[i] + b[i];
        store_row<TY, V, NV>(static_cast<TY*>(a.y) + row * a.y_stride, t, group, a.n, v);
        if (t == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

template <typename TX, typename TY, int V, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarps : kBlockMax) k_norm_backward(Norm a) {
    __shared__ float shared[2][kBlockMax / 32][2];
    __shared__ float joined[WARP ? kWarps : 1][WARP ? 32 * NV * V : 1];
    int turn = 0;
    const int group = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * kWarps : gridDim.x;
    float w[NV * V], dw[NV * V], db[NV * V];
    load_parameter<V, NV>(a.weight, a.parameter_type, 1.0f, t, group, a.n, w);
#pragma unroll
    for (int i = 0; i < NV * V; ++i) dw[i] = db[i] = 0.0f;
    const float scale = 1.0f / static_cast<float>(a.n);
    for (int64_t row = first; row < a.rows; row += step) {
        float x[NV * V], g[NV * V];
        load_row<TX, V, NV>(static_cast<const TX*>(a.x) + row * a.x_stride, t, group, a.n, x);
        load_row<TY, V, NV>(static_cast<const TY*>(a.dy) + row * a.dy_stride, t, group, a.n, g);
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV * V; ++i) {
            x[i] = (x[i] - mean) * rstd;  // beyond the row g is 0, and so is every use of x
            dw[i] += g[i] * x[i];
            db[i] += g[i];
            g[i] *= w[i];
            sum[0] += g[i];
            sum[1] += g[i] * x[i];
        }
        row_sum<WARP>(sum, shared, turn);
        const float of_g = sum[0] * scale, of_gx = sum[1] * scale;
#pragma unroll
        for (int i = 0; i < NV * V; ++i) x[i] = rstd * (g[i] - of_g - x[i] * of_gx);
        if (a.residual) {
            load_row<TX, V, NV>(static_cast<const TX*>(a.residual) + row * a.residual_stride, t, group, a.n, g);
#pragma unroll
            for (int i = 0; i < NV * V; ++i) x[i] += g[i];
        }
        store_row<TX, V, NV>(static_cast<TX*>(a.y) + row * a.y_stride, t, group, a.n, x);
    }
    if (a.partial == nullptr) return;
    float* out = a.partial + static_cast<size_t>(blockIdx.x) * a.n;
#pragma unroll
    for (int which = 0; which < 2; ++which, out += static_cast<size_t>(gridDim.x) * a.n) {
        if (WARP) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV * V; ++i) joined[threadIdx.x >> 5][((i / V) * 32 + t) * V + i % V] = which ? db[i] : dw[i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.n; c += 32 * kWarps) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) v += joined[k][c];
                out[c] = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV * V; ++i) {
                const int c = ((i / V) * group + t) * V + i % V;
                if (c < a.n) out[c] = which ? db[i] : dw[i];
            }
        }
    }
}

// dw and db from the blocks' sums, in a fixed order. Block (32, kPartialRows): 32 columns.
__global__ void k_norm_parameters(const float* partial, int count, int n, void* dw, void* db, int type) {
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
__device__ __forceinline__ float block_sum(float v, float (*shared)[kBlockMax / 32][2], int& turn) {
    float s[1] = {v};
    row_sum<false>(s, shared, turn);
    return s[0];
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kBlockMax) k_wide_forward(Norm a) {
    __shared__ float shared[2][kBlockMax / 32][2];
    int turn = 0;
    const float scale = 1.0f / static_cast<float>(a.n);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
        TY* y = static_cast<TY*>(a.y) + row * a.y_stride;
        float v = 0.0f;
        for (int c = threadIdx.x; c < a.n; c += kBlockMax) v += Element<TX>::load(x[c]);
        const float mean = block_sum(v, shared, turn) * scale;
        v = 0.0f;
        for (int c = threadIdx.x; c < a.n; c += kBlockMax) {
            const float d = Element<TX>::load(x[c]) - mean;
            v += d * d;
        }
        const float rstd = rsqrtf(block_sum(v, shared, turn) * scale + a.epsilon);
        for (int c = threadIdx.x; c < a.n; c += kBlockMax) {
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
__global__ void __launch_bounds__(kBlockMax) k_wide_backward(Norm a) {
    __shared__ float shared[2][kBlockMax / 32][2];
    int turn = 0;
    const float scale = 1.0f / static_cast<float>(a.n);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
        const TY* dy = static_cast<const TY*>(a.dy) + row * a.dy_stride;
        const TX* residual = a.residual ? static_cast<const TX*>(a.residual) + row * a.residual_stride : nullptr;
        TX* dx = static_cast<TX*>(a.y) + row * a.y_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum[2] = {0.0f, 0.0f};
        for (int c = threadIdx.x; c < a.n; c += kBlockMax) {
            const float w = a.weight ? load_any(a.weight, a.parameter_type, c) : 1.0f;
            const float g = Element<TY>::load(dy[c]) * w;
            sum[0] += g;
            sum[1] += g * ((Element<TX>::load(x[c]) - mean) * rstd);
        }
        row_sum<false>(sum, shared, turn);
        const float of_g = sum[0] * scale, of_gx = sum[1] * scale;
        for (int c = threadIdx.x; c < a.n; c += kBlockMax) {
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
    int device = 0, count = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    check(cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device), "SM count");
    return count;
}

// Blocks of the backward pass: what is resident at once (two blocks of 8 warps an SM), and no more
// than there are rows to take. The workspace is sized by the same rule.
constexpr int kBackwardBlocksPerSm = 2;
int backward_blocks(int64_t rows, int64_t n, int sms) {
    if (n > kHeld * kBlockMax) return static_cast<int>(std::min<int64_t>(rows, 64));
    const int64_t want = n <= kHeld * 32 ? (rows + kWarps - 1) / kWarps : rows;
    const int64_t threads = n <= kHeld * 32 ? 32 * kWarps : round_up((n + kHeld - 1) / kHeld, 32);
    const int64_t resident = static_cast<int64_t>(sms) * std::max<int64_t>(1, kBackwardBlocksPerSm * 32 * kWarps / threads);
    return static_cast<int>(std::max<int64_t>(1, std::min(want, resident)));
}

template <typename TX, typename TY, int V>
void run(const Norm& a, bool backward, int sms, cudaStream_t stream) {
    constexpr int NV = kHeld / V;
    const bool warp = a.n <= kHeld * 32;
    const int threads = warp ? 32 * kWarps : static_cast<int>(round_up((a.n + kHeld - 1) / kHeld, 32));
    if (backward) {
        const int grid = backward_blocks(a.rows, a.n, sms);
        if (!warp) {
            launch("k_norm_backward", k_norm_backward<TX, TY, V, NV, false>, grid, threads, 0, stream, a);
        } else if (a.n <= kHeld * 16) {
            launch("k_norm_backward", k_norm_backward<TX, TY, V, NV / 2 ? NV / 2 : 1, true>, grid, threads, 0, stream, a);
        } else {
            launch("k_norm_backward", k_norm_backward<TX, TY, V, NV, true>, grid, threads, 0, stream, a);
        }
        return;
    }
    const int64_t want = warp ? (a.rows + kWarps - 1) / kWarps : a.rows;
    const int grid = static_cast<int>(std::min<int64_t>(want, static_cast<int64_t>(sms) * std::max(1, 1024 / threads)));
    if (!warp) {
        launch("k_norm_forward", k_norm_forward<TX, TY, V, NV, false>, grid, threads, 0, stream, a);
    } else if (a.n <= kHeld * 16) {
        launch("k_norm_forward", k_norm_forward<TX, TY, V, NV / 2 ? NV / 2 : 1, true>, grid, threads, 0, stream, a);
    } else {
        launch("k_norm_forward", k_norm_forward<TX, TY, V, NV, true>, grid, threads, 0, stream, a);
    }
}

template <typename TX, typename TY>
void norm(const Norm& a, bool backward, cudaStream_t stream) {
    const int sms = multiprocessors();
    if (a.n > kHeld * kBlockMax) {
        const int grid = static_cast<int>(std::min<int64_t>(a.rows, sms * 4));
        if (!backward) {
            launch("k_norm_forward", k_wide_forward<TX, TY>, grid, kBlockMax, 0, stream, a);
            return;
        }
        if (a.partial) {
            launch("k_norm_columns", k_wide_columns<TX, TY>, dim3(blocks(a.n, 256), backward_blocks(a.rows, a.n, sms)), 256, 0,
                   stream, a);
        }
        launch("k_norm_backward", k_wide_backward<TX, TY>, grid, kBlockMax, 0, stream, a);
        return;
    }
    // 16 bytes a lane of the wider type where every row of every matrix starts on its vector's
    // boundary, single elements otherwise
    constexpr int V = 16 / (sizeof(TX) > sizeof(TY) ? sizeof(TX) : sizeof(TY));
    const auto fits = [](const void* p, int64_t stride, size_t size) {
        return p == nullptr || (aligned(p, V * size) && stride % V == 0);
    };
    const bool wide = a.n % V == 0 && fits(a.x, a.x_stride, sizeof(TX)) && fits(a.dy, a.dy_stride, sizeof(TY)) &&
        fits(a.residual, a.residual_stride, sizeof(TX)) && fits(a.y, a.y_stride, backward ? sizeof(TX) : sizeof(TY));
    if (wide) {
        run<TX, TY, V>(a, backward, sms, stream);
    } else {
        run<TX, TY, 1>(a, backward, sms, stream);
    }
}

template <typename TX>
void norm_y(const Norm& a, int y_type, bool backward, cudaStream_t stream) {
    if (y_type == T8B_F32) {
        norm<TX, float>(a, backward, stream);
    } else if (y_type == T8B_BF16) {
        norm<TX, bf16>(a, backward, stream);
    } else {
        norm<TX, f16>(a, backward, stream);
    }
}

void dispatch(const Norm& a, int x_type, int y_type, bool backward, cudaStream_t stream) {
    if (x_type == T8B_F32) {
        norm_y<float>(a, y_type, backward, stream);
    } else if (x_type == T8B_BF16) {
        norm_y<bf16>(a, y_type, backward, stream);
    } else {
        norm_y<f16>(a, y_type, backward, stream);
    }
}

void check_sizes(int64_t rows, int64_t n) {
    if (rows < 0) raise(T8B_EINVAL, "layer norm: a negative number of rows");
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
        check_matrix("layer norm x", x, rows, n, x_stride);
        check_matrix("layer norm y", y, rows, n, y_stride);
        if (rows == 0) return;
        const Span to(y, rows, n, y_stride, type_size(y_type)), from(x, rows, n, x_stride, type_size(x_type));
        if (to.overlaps(from) && !(x == y && x_stride == y_stride && x_type == y_type && n <= kHeld * kBlockMax)) {
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
    // sized for any device of up to 256 multiprocessors, so that it needs none to answer
    return static_cast<size_t>(2) * backward_blocks(rows, n, 256) * static_cast<size_t>(n) * sizeof(float);
}

extern "C" int t8b_layer_norm_backward(const void* dy, int y_type, int64_t dy_stride, const void* x, int x_type,
                                       int64_t x_stride, const void* weight, int parameter_type, const float* mean,
                                       const float* rstd, const void* residual_gradient, int64_t residual_stride,
                                       int64_t rows, int64_t n, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_sizes(rows, n);
        if (!is_type(x_type) || !is_type(y_type) || !is_type(parameter_type)) raise(T8B_EINVAL, "layer norm: unknown type");
        check_matrix("layer norm dy", dy, rows, n, dy_stride);
        check_matrix("layer norm x", x, rows, n, x_stride);
        check_matrix("layer norm dx", dx, rows, n, dx_stride);
        if (residual_gradient) check_matrix("layer norm residual gradient", residual_gradient, rows, n, residual_stride);
        if (rows > 0 && (mean == nullptr || rstd == nullptr)) raise(T8B_EINVAL, "layer norm: mean and rstd are null");
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const bool parameters = dweight != nullptr || dbias != nullptr;
        if (rows == 0) {
            if (dweight) check(cudaMemsetAsync(dweight, 0, n * type_size(parameter_type), st), "clear dweight");
            if (dbias) check(cudaMemsetAsync(dbias, 0, n * type_size(parameter_type), st), "clear dbias");
            return;
        }
        const size_t xs = type_size(x_type), ys = type_size(y_type);
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
        dispatch(a, x_type, y_type, true, st);
        if (parameters) {
            launch("k_norm_parameters", k_norm_parameters, dim3(blocks(n, 32), 2), dim3(32, kPartialRows), 0, st,
                   static_cast<const float*>(workspace), backward_blocks(rows, n, multiprocessors()), a.n, dweight, dbias,
                   parameter_type);
        }
        check(cudaGetLastError(), "layer norm launch");
    });
}
