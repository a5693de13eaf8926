// The linear map and the gated projection for one element type (bf16 or f16): epilogues over the
// GEMM of ops_gemm.cuh, the elementwise half of the backward passes, and the host side that plans
// and queues a call. ops_bf16.cu and ops_f16.cu instantiate it; ops_linear.cu holds the C entries.
#pragma once

#include <algorithm>
#include <atomic>

#include "gemm_host.cuh"
#include "ops_gemm.cuh"

namespace t8b {
namespace op {

// The device's count of waits that ran out (ops_linear.cu).
unsigned* stall_count();

struct LinearCall {
    const void *x, *weight, *bias, *residual;
    void *y, *pre;
    int64_t x_stride, weight_stride, residual_stride, y_stride, pre_stride;
    int64_t rows, in, out;
    int bias_type, activation, y_type;
    bool gated;
    int what;  // the parts of the workspace it uses (T8B_WORKSPACE_*)
    unsigned char* workspace;
    cudaStream_t stream;
};
struct LinearGradCall {
    const void *dy, *x, *weight, *pre;
    void *dx, *dweight, *dbias;
    int64_t dy_stride, x_stride, weight_stride, pre_stride, dx_stride, dweight_stride;
    int64_t rows, in, out;
    int bias_type, activation;
    bool gated;
    int what;  // the parts of the workspace it uses (T8B_WORKSPACE_*)
    unsigned char* workspace;
    cudaStream_t stream;
};
template <typename E>
void linear_forward(const LinearCall& c);
template <typename E>
void linear_backward(const LinearGradCall& c);

// ------------------------------------------------------------------ planning
// A GEMM's tile (pairs of CTAs on 256 x 256 or 256 x 128, or one CTA on 128 x 64) and the number of
// parts its k blocks are split into.
struct GemmPlan {
    int bn, splits;
};
constexpr int kClusters = 74, kSms = 148;
constexpr int kMaxSplits = 64;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Cycles of the busiest CTA as the plan's cost: waves x (k blocks x cycles + the tile's latency), plus
// the pass that joins the parts (its traffic over the chip's, and `join_cycles`). The cycles are fits to
// measured products: a narrower tile costs nearly as many a k-block, because what the MMAs read from
// shared memory bounds them, and less latency. 65,536 x 512 x 512 took 42.7 / 54.0 / 88.2 us by
// 256 / 128 / 64 columns, 4,096 rows of it 12.4 / 10.5 / 12.2, 512 rows 10.8 / 10.5 / 8.4; its weight's
// gradient 41 us in 18 parts, 318 in one.
inline GemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, bool may_split, double join_cycles = 4000) {
    struct Form {
        int pair, bn;
        double block_cycles, tile_cycles;
    };
    static constexpr Form forms[] = {{1, 256, 600, 4400}, {1, 128, 570, 2400}, {0, 64, 540, 1400}};
    const int64_t k_blocks = ceil_div(k, tc::BK);
    GemmPlan best{256, 1};
    double least = 1e300;
    for (const Form& f : forms) {
        const int64_t tiles = ceil_div(m, f.pair ? 256 : 128) * ceil_div(n, f.bn);
        const int64_t workers = f.pair ? kClusters : kSms;
        const int64_t most = may_split ? std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, k_blocks / 4)) : 1;
        // the parts that fill one to four waves; more or fewer leave workers idle
        for (int64_t wave = 0; wave <= (most > 1 ? 4 : 0); ++wave) {
            const int64_t splits = wave == 0 ? 1 : std::min<int64_t>(most, std::max<int64_t>(1, wave * workers / tiles));
            const double waves = static_cast<double>(ceil_div(tiles * splits, workers));
            double cost = waves * (static_cast<double>(ceil_div(k_blocks, splits)) * f.block_cycles + f.tile_cycles);
            if (splits > 1) cost += join_cycles + static_cast<double>(splits) * m * n * 8.0 / 2500.0;
            if (cost < least) {
                least = cost;
                best = GemmPlan{f.bn, static_cast<int>(splits)};
            }
        }
    }
    return best;
}

// Whether a forward pass goes row by row (k_few_rows) and not by tiles. Up to 4 rows always. Up to 16 rows
// where the sums are short, the warps, one for each column of the output and group of 8 rows, are resident
// at once (beyond that they take a second turn), and a gate's second sums do not make up for it. Measured
// (bf16, us a call among others, by rows / by tiles): 512 -> 512: 1 row 2.2 / 5.6, 16 rows 4.9 / 5.7;
// 512 -> 2,816: 4 rows 3.7 / 5.8, 8 rows 5.6 / 5.8, 9 rows 6.9 / 5.8; 512 -> 1,408: 16 rows 5.5 / 5.8; 512 -> 1,792:
// 16 rows 8.8 / 5.9; 512 -> 8,192: 4 rows 6.4 / 7.6, 5 rows 10.0 / 7.7; gated 512 -> 1,408: 8 rows 6.3 / 6.5, 9
// rows 6.9 / 6.7, 16 rows 7.0 / 6.6; gated 256 -> 1,408: 16 rows 4.8 / 5.4; 2,048 -> 2,048: 4 rows 7.4 / 13.1, 8 rows
// 14.6 / 13.1; 4,096 -> 512: 4 rows 12.1 / 22.5, 8 rows 25.4 / 22.4. Rows off 16-byte boundaries cross earlier,
// 151 -> 512: 4 rows 5.1 / 6.1, 8 rows 8.4 / 6.2; they keep the rule, with which their call needs no workspace.
inline bool is_few(int64_t rows, int64_t in, int64_t out, bool gated) {
    const int64_t warps = out * ceil_div(rows, 8);
    return rows <= 4 || (rows <= 16 && in <= 512 && warps <= 2816 && (gated ? 2 : 1) * warps * in <= 2816 * 512);
}

// The gradients' products. The weight's sums over the rows and is split wherever that pays; the input's
// where few rows leave SMs idle behind a long sum over the columns: whole backward passes in us, one part
// / split, linear 64 x 512 x 1,408 10.9 / 9.0, 64 x 512 x 8,192 43 / 17.7, 2,048 x 512 x 8,192 63 / 41,
// gated 64 x 512 x 4,096 45 / 19.6. Never above 16,384 rows, where tiles of any width fill the chip.
// The other product runs beside it on the SMs it leaves, so its split has to save more: at the cost
// of a lone join 512 x 512 x 1,408 took 14.5 for 11.4.
inline GemmPlan weight_grad_plan(int64_t rows, int64_t in, int64_t columns) { return plan_gemm(columns, in, rows, true); }
inline GemmPlan input_grad_plan(int64_t rows, int64_t in, int64_t columns) {
    return plan_gemm(rows, in, columns, rows <= 16384, 8000);
}

// The parts of a split GEMM: fp32 [splits][rows to whole tiles][columns to whole pieces].
inline size_t split_rows(int64_t m) { return round_up(m, 256); }
inline size_t split_pitch(int64_t n) { return round_up(n, 4); }
inline size_t split_bytes(const GemmPlan& p, int64_t m, int64_t n) { return p.splits * split_rows(m) * split_pitch(n) * 4; }

// Row parts of the elementwise backward pass over dy's columns (each gives one row of partial column
// sums): with 256 columns a block, two blocks an SM, and no more resident, so that they spread evenly
// even where they start behind a kernel that leaves some SMs first (three where they find room: 460 us
// for the gated backward of 65,536 x 1,408 against 426).
constexpr int kGradRows = 8, kGradBlocks = 2;
constexpr size_t kGradSmem = 100 * 1024;
inline int grad_parts(int64_t rows, int64_t out) {
    const int64_t across = ceil_div(out, 256);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, kGradRows), kSms * kGradBlocks / across)));
}

// The workspace of a call, in this order and as far as `what` (T8B_WORKSPACE_* bits) says; each part
// starts on a 256-byte boundary.
struct Workspace {
    size_t x, weight, dz, sums, weight_parts, input_parts, bytes;
    size_t dz_pitch;
    Workspace(int64_t rows, int64_t in, int64_t out, bool gated, int what) {
        const int64_t columns = gated ? 2 * out : out;
        const size_t x_pitch = round_up(in, 8);
        dz_pitch = round_up(columns, 8);
        size_t at = 0;
        const auto take = [&](bool wanted, size_t size) {
            const size_t here = at;
            if (wanted) at += round_up(size, 256);
            return here;
        };
        const bool backward = (what & T8B_WORKSPACE_BACKWARD) != 0;
        x = take((what & T8B_WORKSPACE_X) != 0, rows * x_pitch * 2);
        weight = take((what & T8B_WORKSPACE_WEIGHT) != 0, columns * x_pitch * 2);
        dz = take(backward && (what & T8B_WORKSPACE_DZ) != 0, rows * dz_pitch * 2);
        sums = take(backward, static_cast<size_t>(grad_parts(rows, out)) * columns * 4);
        const GemmPlan one{0, 1}, of_weight = backward ? weight_grad_plan(rows, in, columns) : one;
        const GemmPlan of_input = backward ? input_grad_plan(rows, in, columns) : one;
        weight_parts = take(of_weight.splits > 1, split_bytes(of_weight, columns, in));
        input_parts = take(of_input.splits > 1, split_bytes(of_input, rows, in));
        bytes = at;
    }
};

// ------------------------------------------------------------------ epilogues
// 32 fp32 values as the packed 16-bit or fp32 pieces of a staging tile's row.
template <typename T, int BYTES>
__device__ __forceinline__ void stage32(unsigned char* tile, int row, int at, const float (&v)[32]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            *reinterpret_cast<float4*>(piece<BYTES>(tile, row, at / 4 + q)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            *reinterpret_cast<uint4*>(piece<BYTES>(tile, row, at / 8 + q)) =
                make_uint4(Element<T>::pack(v[8 * q], v[8 * q + 1]), Element<T>::pack(v[8 * q + 2], v[8 * q + 3]),
                           Element<T>::pack(v[8 * q + 4], v[8 * q + 5]), Element<T>::pack(v[8 * q + 6], v[8 * q + 7]));
        }
    }
}
template <typename T, int BYTES>
__device__ __forceinline__ void add32(unsigned char* tile, int row, int at, float (&v)[32]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float4 r = *reinterpret_cast<const float4*>(piece<BYTES>(tile, row, at / 4 + q));
            v[4 * q] += r.x;
            v[4 * q + 1] += r.y;
            v[4 * q + 2] += r.z;
            v[4 * q + 3] += r.w;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint4 r = *reinterpret_cast<const uint4*>(piece<BYTES>(tile, row, at / 8 + q));
            const uint32_t words[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = Element<T>::unpack(words[k]);
                v[8 * q + 2 * k] += f.x;
                v[8 * q + 2 * k + 1] += f.y;
            }
        }
    }
}
// 32 bias values through the warp's vector, one read a lane, then added to every row.
__device__ __forceinline__ float bias_at(const void* bias, int type, int c, int columns) {
    return bias != nullptr && c < columns ? load_any(bias, type, c) : 0.0f;
}
__device__ __forceinline__ void add_bias32(float* vector, float mine, int lane, float (&v)[32]) {
    __syncwarp();
    vector[lane] = mine;
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const float4 b = reinterpret_cast<const float4*>(vector)[q];
        v[4 * q] += b.x;
        v[4 * q + 1] += b.y;
        v[4 * q + 2] += b.z;
        v[4 * q + 3] += b.w;
    }
}

// y = activation(acc + bias) + residual in the type O, and acc + bias as `pre`; without FULL, acc
// alone (gradients, and the fp32 parts of a split GEMM). A group of epilogue warps takes half of the
// tile's columns in chunks of a 128-byte row (64 where a tile of 64 columns has no more): stores of
// 64-byte rows took 158 us where 128-byte rows take 130 (75,776 x 128 times 2,816 x 128, where stores
// are most of the work), one store for four warps' rows 147. A chunk's residual is fetched into the
// staging tile, the first one's while the MMAs run; y replaces it, then `pre`, read again from
// tensor memory.
template <typename E, typename O, int BN, bool FULL>
struct EpiLinear {
    static constexpr int kWide = sizeof(O) == 2 && BN >= 128 ? 64 : 32;  // columns of a chunk
    static constexpr int kBytes = kWide * sizeof(O);
    static constexpr int kPreBytes = kWide * 2;
    static constexpr int kColumns = BN / 2;  // of a group
    static constexpr int kChunks = kColumns / kWide;
    Tiled y, residual, pre;
    const void* bias;
    int bias_type, activation, has_residual, has_pre, split_rows;

    __device__ __forceinline__ int column(const Warp& w, int chunk) const { return w.tn * BN + w.group * kColumns + chunk * kWide; }
    __device__ __forceinline__ void fetch_chunk(Warp& w, int chunk) const {
        const int col = column(w, chunk);
        if (chunk >= kChunks || col >= y.columns) return;
        free_tile(w.lane);
        fetch<O, kBytes>(residual, w.tile, w.bar, w.row0, col, w.lane);
        w.in_flight = residual.tma;
    }
    __device__ __forceinline__ void begin(Warp& w) const {
        if (FULL && has_residual && w.row0 < y.rows) fetch_chunk(w, 0);
    }
    // 32 columns of acc + bias
    __device__ __forceinline__ void load(const Warp& w, int chunk, int at, float (&v)[32]) const {
        float b = 0.0f;
        if (FULL) b = bias_at(bias, bias_type, column(w, chunk) + at + w.lane, y.columns);
        tc::tmem_load32(w.taddr + w.group * kColumns + chunk * kWide + at, v);
        if (FULL && bias != nullptr) add_bias32(w.vector, b, w.lane, v);
    }
    __device__ __forceinline__ bool finish(Warp& w) const {
        if (w.row0 >= y.rows) return true;
        const int row0 = w.row0 + w.split * split_rows;
#pragma unroll 1
        for (int chunk = 0; chunk < kChunks; ++chunk) {
            const int col = column(w, chunk);
            if (col >= y.columns) break;
            if (FULL && has_residual) {
                if (residual.tma && !w.wait()) return false;
            } else {
                free_tile(w.lane);
            }
#pragma unroll
            for (int at = 0; at < kWide; at += 32) {
                float v[32];
                load(w, chunk, at, v);
                if (FULL) {
                    with_activation(activation, [&](auto act) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] = activate<decltype(act)::value>(v[k]);
                    });
                    if (has_residual) add32<O, kBytes>(w.tile, w.lane, at, v);
                }
                stage32<O, kBytes>(w.tile, w.lane, at, v);
            }
            send<O, kBytes>(y, w.tile, row0, col, w.lane);
            if (FULL && has_pre) {
                free_tile(w.lane);
#pragma unroll 1
                for (int at = 0; at < kWide; at += 32) {
                    float v[32];
                    load(w, chunk, at, v);
                    stage32<E, kPreBytes>(w.tile, w.lane, at, v);
                }
                send<E, kPreBytes>(pre, w.tile, row0, col, w.lane);
            }
            if (FULL && has_residual) fetch_chunk(w, chunk + 1);
        }
        return true;
    }
};

// h = activation(gate) up; the accumulator's first BN / 2 columns are the gate's, the others the
// up projection's of the same columns of h. A warp takes 64 columns of h (32 where a tile has no
// more) as one staging tile: h goes out through it, then gate and up, each read again from tensor
// memory, once the store before has read it.
template <typename E, int BN>
struct EpiGated {
    static constexpr int kHalf = BN / 2;
    static constexpr int kWide = kHalf >= 128 ? 64 : 32;  // columns of a warp
    static constexpr int kBytes = kWide * 2;
    Tiled h, gate, up;
    const void* bias;
    int bias_type, activation, has_pre;

    __device__ __forceinline__ void begin(Warp&) const {}
    // 32 columns of acc + bias of the gate (part 0) or the up projection (1), from column `at` of the warp's
    __device__ __forceinline__ void load(const Warp& w, int part, int at, float (&v)[32]) const {
        const int column = w.group * kWide + at;
        float b = 0.0f;
        if (bias != nullptr) {
            const int c = w.tn * kHalf + column + w.lane;
            if (c < h.columns) b = load_any(bias, bias_type, part * h.columns + c);
        }
        tc::tmem_load32(w.taddr + part * kHalf + column, v);
        if (bias != nullptr) add_bias32(w.vector, b, w.lane, v);
    }
    __device__ __forceinline__ bool finish(Warp& w) const {
        const int col = w.tn * kHalf + w.group * kWide;
        if (w.row0 >= h.rows || w.group * kWide >= kHalf || col >= h.columns) return true;
        free_tile(w.lane);
#pragma unroll 1
        for (int at = 0; at < kWide; at += 32) {
            float g[32], u[32];
            load(w, 0, at, g);
            with_activation(activation, [&](auto act) {
#pragma unroll
                for (int k = 0; k < 32; ++k) g[k] = activate<decltype(act)::value>(g[k]);
            });
            load(w, 1, at, u);
#pragma unroll
            for (int k = 0; k < 32; ++k) g[k] *= u[k];
            stage32<E, kBytes>(w.tile, w.lane, at, g);
        }
        send<E, kBytes>(h, w.tile, w.row0, col, w.lane);
        if (!has_pre) return true;
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
            free_tile(w.lane);
#pragma unroll
            for (int at = 0; at < kWide; at += 32) {
                float v[32];
                load(w, part, at, v);
                stage32<E, kBytes>(w.tile, w.lane, at, v);
            }
            send<E, kBytes>(part ? up : gate, w.tile, w.row0, col, w.lane);
        }
        return true;
    }
};

// ------------------------------------------------------------------ elementwise kernels
// Rows of `in` with any stride, copied to rows of `pitch` (a multiple of 8) elements: operands whose
// rows do not start on 16-byte boundaries, which TMA asks for. One 16-byte piece a thread; both
// operands of a product in one launch.
struct PackJob {
    const void* in;
    void* out;
    int64_t stride, rows, pitch;
    int columns;
};
template <typename E>
__global__ void k_pack(PackJob first, PackJob second, int after) {
    if (after == kInput) wait_previous();
    release_next();
    const int64_t pieces = first.rows * (first.pitch / 8), total = pieces + second.rows * (second.pitch / 8);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const PackJob& job = i < pieces ? first : second;
        const int64_t at = i < pieces ? i : i - pieces;
        const int64_t row = at / (job.pitch / 8);
        const int c = static_cast<int>(at - row * (job.pitch / 8)) * 8;
        const E* in = static_cast<const E*>(job.in) + row * job.stride + c;
        Pack<E, 8> p;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p.v[j] = Element<E>::store(0.0f);
            if (c + j < job.columns) p.v[j] = in[j];
        }
        *reinterpret_cast<Pack<E, 8>*>(static_cast<E*>(job.out) + row * job.pitch + c) = p;
    }
    if (after == kBeside) wait_previous();  // the next kernel's wait for this one covers both
}

// A forward pass of few rows: a warp per output column (or per gate and up column), its lanes over
// the row of the weight in 16-byte pieces (WIDE; single elements where rows are not aligned), R rows
// of x at a time. Bound by the latency of one pass over the weight, spread over every SM, where a
// tile of the tensor-core kernel would wait for its k blocks one after the other.
template <typename E>
struct FewRows {
    const E *x, *weight;
    const void *bias, *residual;
    void* y;
    E* pre;
    int64_t x_stride, weight_stride, residual_stride, y_stride, pre_stride;
    int rows, in, out, bias_type, activation, y_type;
};
constexpr int kFewWarps = 8;
template <typename E, bool GATED, int R, bool WIDE>
__global__ void __launch_bounds__(32 * kFewWarps) k_few_rows(FewRows<E> a) {
    wait_previous();
    release_next();
    constexpr int PARTS = GATED ? 2 : 1;
    const int lane = threadIdx.x & 31;
    const int row0 = blockIdx.y * R, live = min(R, a.rows - row0);
    for (int c = blockIdx.x * kFewWarps + (threadIdx.x >> 5); c < a.out; c += gridDim.x * kFewWarps) {
        const E* w[PARTS];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) w[p] = a.weight + (static_cast<int64_t>(p) * a.out + c) * a.weight_stride;
        const E* x = a.x + row0 * a.x_stride;
        float sum[PARTS][R];
        int done = 0;
        if (WIDE) {
            Two pair[PARTS][R];
            const int pieces = a.in / 8;
#pragma unroll 2
            for (int i = lane; i < pieces; i += 32) {
                Pack<uint32_t, 4> words[PARTS];
#pragma unroll
                for (int p = 0; p < PARTS; ++p) words[p] = *reinterpret_cast<const Pack<uint32_t, 4>*>(w[p] + i * 8);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r >= live) break;
                    const Pack<uint32_t, 4> row = *reinterpret_cast<const Pack<uint32_t, 4>*>(x + r * a.x_stride + i * 8);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 xv = Element<E>::unpack(row.v[j]);
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) {
                            const float2 wv = Element<E>::unpack(words[p].v[j]);
                            pair[p][r] = multiply_add(Two(xv.x, xv.y), Two(wv.x, wv.y), pair[p][r]);
                        }
                    }
                }
            }
            done = pieces * 8;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                for (int r = 0; r < R; ++r) sum[p][r] = pair[p][r].sum();
            }
        } else {
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                for (int r = 0; r < R; ++r) sum[p][r] = 0.0f;
            }
        }
#pragma unroll 4
        for (int i = done + lane; i < a.in; i += 32) {
            float wv[PARTS];
#pragma unroll
            for (int p = 0; p < PARTS; ++p) wv[p] = Element<E>::load(w[p][i]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r >= live) break;
                const float xv = Element<E>::load(x[r * a.x_stride + i]);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) sum[p][r] = fmaf(xv, wv[p], sum[p][r]);
            }
        }
        float mine[PARTS];  // lane r: row r's sums
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            mine[p] = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v = sum[p][r];
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane == r) mine[p] = v;
            }
            if (a.bias) mine[p] += load_any(a.bias, a.bias_type, static_cast<size_t>(p) * a.out + c);
        }
        if (lane >= live) continue;
        const int64_t row = row0 + lane;
        if (a.pre) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p) a.pre[row * a.pre_stride + static_cast<int64_t>(p) * a.out + c] = Element<E>::store(mine[p]);
        }
        float v = 0.0f;
        with_activation(a.activation, [&](auto act) { v = activate<decltype(act)::value>(mine[0]); });
        if (GATED) v *= mine[PARTS - 1];
        if (a.residual) v += load_any(a.residual, a.y_type, row * a.residual_stride + c);
        store_any(a.y, a.y_type, row * a.y_stride + c, v);
    }
}

// The elementwise half of a backward pass: dz (rows of `pitch` elements) from dy and pre, and this
// block row's column sums of dz in fp32, before dz is rounded. A thread holds V columns over its
// rows; block (32, kGradRows).
//   linear: dz = dy activation'(pre);  gated: dz = [dy up activation'(gate) | dy activation(gate)]
// dz is rounded to the operands' type because the tensor cores take both operands of a product in one
// 16-bit type; a second 16-bit part for what that leaves out would double both products, which are two thirds of
// a large pass. It is as large an error as the outputs' own rounding: dx and dweight of 65,536 x 512 x 512 are off by
// 2.35e-3 of their norm in bf16 where products of fp32 dz, rounded once, are off by 1.66e-3 (f16: 2.9e-4 and
// 2.1e-4). In f16 dz has that type's range too: gradients are scaled before the call, as for dy itself.
// Bound by memory: it reads dy and pre and writes dz once. With V = 8 a thread's next rows come
// through its own part of a ring in shared memory (cp.async, as in the layer norm's kernels).
constexpr int kGradStages = 4;
template <typename E, bool GATED, int V>
constexpr int grad_ring_bytes() { return V == 8 ? kGradStages * (GATED ? 3 : 2) * 16 * 32 * kGradRows : 0; }

template <typename E, bool GATED, int V>
__global__ void __launch_bounds__(32 * kGradRows, V == 8 ? kGradBlocks : 5)
    k_activation_grad(const E* dy, int64_t dy_stride, const E* pre, int64_t pre_stride, int64_t rows, int columns,
                      int activation, E* dz, int64_t pitch, float* sums) {
    wait_previous();
    release_next();  // operands may be packed beside it
    constexpr int PARTS = GATED ? 2 : 1;
    constexpr bool RING = V == 8;
    constexpr int kThreads = 32 * kGradRows;
    constexpr int kStage = (GATED ? 3 : 2) * 16 * kThreads;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ float joined[kGradRows][32 * V + 1];
    const int c = (blockIdx.x * 32 + threadIdx.x) * V;
    float sum[PARTS][V];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[p][j] = 0.0f;
    }
    if (c < columns) {
        with_activation(activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            constexpr bool READS = GATED || ACT != T8B_LINEAR;  // pre
            const int64_t first = static_cast<int64_t>(blockIdx.y) * kGradRows + threadIdx.y;
            const int64_t step = static_cast<int64_t>(gridDim.y) * kGradRows;
            const E* from_dy = dy + first * dy_stride + c;
            const E* from_pre = READS ? pre + first * pre_stride + c : nullptr;
            E* to = dz ? dz + first * pitch + c : nullptr;
            unsigned char* mine = ring + (threadIdx.y * 32 + threadIdx.x) * 16;
            const uint32_t slot = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
            auto copy = [&](uint32_t at, const E* from) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
            };
            auto fetch = [&](int stage, bool any) {
                if (any) {
                    const uint32_t at = slot + stage * kStage;
                    copy(at, from_dy);
                    if (READS) copy(at + 16 * kThreads, from_pre);
                    if (GATED) copy(at + 32 * kThreads, from_pre + columns);
                    from_dy += step * dy_stride;
                    if (READS) from_pre += step * pre_stride;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            if (RING) {
#pragma unroll
                for (int k = 0; k < kGradStages - 1; ++k) fetch(k, first + k * step < rows);
            }
            auto use = [&](const Pack<E, V>& d, const Pack<E, V>& z, const Pack<E, V>& u) {
                Pack<E, V> out, out_up;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float value, slope;
                    const float g = Element<E>::load(d.v[j]);
                    activate_slope<ACT>(Element<E>::load(z.v[j]), value, slope);
                    const float of_z = g * slope * (GATED ? Element<E>::load(u.v[j]) : 1.0f);
                    sum[0][j] += of_z;
                    out.v[j] = Element<E>::store(of_z);
                    if (GATED) {
                        const float of_u = g * value;
                        sum[PARTS - 1][j] += of_u;
                        out_up.v[j] = Element<E>::store(of_u);
                    }
                }
                if (to) {
                    *reinterpret_cast<Pack<E, V>*>(to) = out;
                    if (GATED) *reinterpret_cast<Pack<E, V>*>(to + columns) = out_up;
                    to += step * pitch;
                }
            };
            int stage = 0;
            int64_t row = first;
            if (!RING) {  // four rows' elements in flight
                constexpr int kBatch = 4;
                for (; row + (kBatch - 1) * step < rows; row += kBatch * step) {
                    Pack<E, V> d[kBatch], z[kBatch], u[kBatch];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        d[k] = *reinterpret_cast<const Pack<E, V>*>(from_dy);
                        z[k] = READS ? *reinterpret_cast<const Pack<E, V>*>(from_pre) : Pack<E, V>{};
                        u[k] = GATED ? *reinterpret_cast<const Pack<E, V>*>(from_pre + columns) : Pack<E, V>{};
                        from_dy += step * dy_stride;
                        if (READS) from_pre += step * pre_stride;
                    }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) use(d[k], z[k], u[k]);
                }
            }
            for (; row < rows; row += step) {
                Pack<E, V> d, z{}, u{};
                if (RING) {
                    fetch((stage + kGradStages - 1) % kGradStages, row + (kGradStages - 1) * step < rows);
                    asm volatile("cp.async.wait_group %0;" ::"n"(kGradStages - 1) : "memory");
                    const unsigned char* at = mine + stage * kStage;
                    d = *reinterpret_cast<const Pack<E, V>*>(at);
                    if (READS) z = *reinterpret_cast<const Pack<E, V>*>(at + 16 * kThreads);
                    if (GATED) u = *reinterpret_cast<const Pack<E, V>*>(at + 32 * kThreads);
                    stage = (stage + 1) % kGradStages;
                } else {
                    d = *reinterpret_cast<const Pack<E, V>*>(from_dy);
                    if (READS) z = *reinterpret_cast<const Pack<E, V>*>(from_pre);
                    if (GATED) u = *reinterpret_cast<const Pack<E, V>*>(from_pre + columns);
                    from_dy += step * dy_stride;
                    if (READS) from_pre += step * pre_stride;
                }
                use(d, z, u);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        });
    }
    if (sums == nullptr) return;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) joined[threadIdx.y][threadIdx.x * V + j] = sum[p][j];
        __syncthreads();
        for (int k = threadIdx.y * 32 + threadIdx.x; k < 32 * V; k += kThreads) {
            const int column = blockIdx.x * 32 * V + k;
            if (column >= columns) continue;
            float v = 0.0f;
#pragma unroll
            for (int r = 0; r < kGradRows; ++r) v += joined[r][k];
            sums[static_cast<size_t>(blockIdx.y) * columns * PARTS + p * columns + column] = v;
        }
    }
}

// What the last pass of a backward adds up, in a fixed order: the parts of split gradients (rounded
// once), four columns a thread, and the block rows' column sums of dz (dbias), 32 columns a block. The
// first blocks join the weight's gradient, the next the input's, the others the bias's. Block (32, 8).
struct Join {
    const float* parts;
    size_t part_elements;
    int splits, pitch, rows, columns;
    void* out;
    int64_t stride;
    unsigned blocks;
};
struct Totals {
    Join weight, input;
    const float* sums;
    int sums_rows, bias_columns;
    void* dbias;
    int bias_type;
};
template <typename E>
__global__ void __launch_bounds__(256) k_totals(Totals a) {
    wait_previous();
    release_next();
    const unsigned joins = a.weight.blocks + a.input.blocks;
    if (blockIdx.x < joins) {
        const bool first = blockIdx.x < a.weight.blocks;
        const Join& join = first ? a.weight : a.input;
        const unsigned block = first ? blockIdx.x : blockIdx.x - a.weight.blocks;
        const int64_t i = static_cast<int64_t>(block) * 256 + threadIdx.y * 32 + threadIdx.x;
        const int pieces = join.pitch / 4;
        if (i >= static_cast<int64_t>(join.rows) * pieces) return;
        const int row = static_cast<int>(i / pieces), c = static_cast<int>(i % pieces) * 4;
        const float* p = join.parts + static_cast<size_t>(row) * join.pitch + c;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int s = 0; s < join.splits; ++s, p += join.part_elements) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        E* to = static_cast<E*>(join.out) + static_cast<int64_t>(row) * join.stride + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j < join.columns) to[j] = Element<E>::store(v[j]);
        }
        return;
    }
    __shared__ float joined[8][33];
    const int c = (blockIdx.x - joins) * 32 + threadIdx.x;
    float v = 0.0f;
    if (c < a.bias_columns) {
#pragma unroll 8
        for (int r = threadIdx.y; r < a.sums_rows; r += 8) v += a.sums[static_cast<size_t>(r) * a.bias_columns + c];
    }
    joined[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y != 0 || c >= a.bias_columns) return;
#pragma unroll
    for (int r = 1; r < 8; ++r) v += joined[r][threadIdx.x];
    store_any(a.dbias, a.bias_type, c, v);
}

// ------------------------------------------------------------------ host side
template <typename T>
CUtensorMap tensor_map(const void* base, uint64_t inner, uint64_t outer, uint64_t pitch, uint32_t box_inner, uint32_t box_outer,
                       CUtensorMapSwizzle swizzle) {
    constexpr CUtensorMapDataType type = Element<T>::kType == T8B_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
        : Element<T>::kType == T8B_BF16                               ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap map;
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {pitch * sizeof(T)};
    const cuuint32_t box[2] = {box_inner, box_outer};
    const cuuint32_t element[2] = {1, 1};
    const CUresult r = tensor_map_encoder()(&map, type, 2, const_cast<void*>(base), dims, strides, box, element,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) raise(T8B_ECUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(static_cast<int>(r)));
    return map;
}

// Rows that TMA can address: 16-byte starts, and a row stride below its 2^40 bytes.
inline bool tma_rows(const void* p, int64_t rows, int64_t stride, size_t size) {
    return aligned(p, 16) && (rows <= 1 || ((stride * size) % 16 == 0 && stride * size < (1ull << 40)));
}
inline int64_t tma_pitch(int64_t rows, int64_t columns, int64_t stride, size_t size) {
    return rows <= 1 ? round_up(columns, 16 / size) : stride;
}

template <typename T, int BYTES>
Tiled tiled(const void* data, int64_t rows, int64_t columns, int64_t stride) {
    Tiled t{};
    t.data = const_cast<void*>(data);
    t.stride = stride;
    t.rows = static_cast<int>(rows);
    t.columns = static_cast<int>(columns);
    t.tma = data != nullptr && tma_rows(data, rows, stride, sizeof(T));
    if (t.tma) {
        t.map = tensor_map<T>(data, columns, rows, tma_pitch(rows, columns, stride, sizeof(T)), BYTES / sizeof(T), 32,
                              BYTES == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    }
    return t;
}

// A GEMM operand: row-major [rows][k] (K-major) or [k][rows] (MN-major), rows on 16-byte boundaries.
struct Matrix {
    const void* data;
    int64_t rows, k, pitch;
};

template <typename E, int CG, int BN, bool A_MN, bool B_MN, class Epi>
void launch_gemm(const char* label, const Matrix& a, const Matrix& b, int64_t columns, int second, int splits, int after,
                 const Epi& epi, cudaStream_t stream) {
    using P = Plan<CG, BN>;
    auto kernel = k_gemm<E, CG, BN, A_MN, B_MN, Epi>;
    static uint64_t configured = 0;
    allow_smem(kernel, P::kSmemBytes, configured);
    Shape s{};
    s.tiles_m = static_cast<int>(ceil_div(a.rows, tc::BM * CG));
    s.tiles_n = static_cast<int>(ceil_div(columns, second ? BN / 2 : BN));
    s.k_blocks = static_cast<int>(ceil_div(a.k, tc::BK));
    s.splits = splits;
    s.second = second;
    s.after = after;
    s.stalls = stall_count();
    const auto k_major = [](const Matrix& m, uint32_t box) {
        return tensor_map<E>(m.data, m.k, m.rows, tma_pitch(m.rows, m.k, m.pitch, 2), tc::BK, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const auto mn_major = [](const Matrix& m) {
        return tensor_map<E>(m.data, m.rows, m.k, tma_pitch(m.k, m.rows, m.pitch, 2), 64, tc::BK, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const CUtensorMap map_a = A_MN ? mn_major(a) : k_major(a, tc::BM);
    const CUtensorMap map_b = B_MN ? mn_major(b) : k_major(b, second ? BN / 2 : BN / CG);
    const int64_t work = static_cast<int64_t>(s.tiles_m) * s.tiles_n * s.splits;
    const int grid = static_cast<int>(std::min<int64_t>(work, CG == 2 ? kClusters : kSms)) * CG;
    launch_chain(label, kernel, grid, kGemmThreads, P::kSmemBytes, stream, true, map_a, map_b, s, epi);
}

// A matrix as a GEMM operand: where its rows do not suit TMA, a copy in the workspace, which pack()
// makes.
template <typename E>
Matrix operand(const void* data, int64_t rows, int64_t columns, int64_t stride, unsigned char* copy, PackJob& job) {
    if (tma_rows(data, rows, stride, sizeof(E))) return Matrix{data, rows, columns, tma_pitch(rows, columns, stride, sizeof(E))};
    job = PackJob{data, copy, stride, rows, static_cast<int64_t>(round_up(columns, 8)), static_cast<int>(columns)};
    return Matrix{copy, rows, columns, job.pitch};
}
template <typename E>
void pack(const PackJob (&jobs)[2], int after, cudaStream_t stream) {
    const int64_t pieces = (jobs[0].rows * jobs[0].pitch + jobs[1].rows * jobs[1].pitch) / 8;
    if (pieces == 0) return;
    launch_chain("k_pack", k_pack<E>, static_cast<unsigned>(std::min<int64_t>(ceil_div(pieces, 256), kSms * 16)), 256, 0, stream,
                 true, jobs[0], jobs[1], after);
}
// [rows][k] read along its rows' other axis: the same storage as an MN-major operand.
inline Matrix transposed(const Matrix& m) { return Matrix{m.data, m.k, m.rows, m.pitch}; }

template <typename E, typename O, int CG, int BN>
void forward_tile(const LinearCall& c, const Matrix& x, const Matrix& w) {
    using Epi = EpiLinear<E, O, BN, true>;
    Epi epi{};
    epi.y = tiled<O, Epi::kBytes>(c.y, c.rows, c.out, c.y_stride);
    if (c.residual) epi.residual = tiled<O, Epi::kBytes>(c.residual, c.rows, c.out, c.residual_stride);
    if (c.pre) epi.pre = tiled<E, Epi::kPreBytes>(c.pre, c.rows, c.out, c.pre_stride);
    epi.residual.rows = static_cast<int>(c.rows);
    epi.residual.columns = static_cast<int>(c.out);
    epi.bias = c.bias;
    epi.bias_type = c.bias_type;
    epi.activation = c.activation;
    epi.has_residual = c.residual != nullptr;
    epi.has_pre = c.pre != nullptr;
    launch_gemm<E, CG, BN, false, false>("k_linear", x, w, c.out, 0, 1, kInput, epi, c.stream);
}
template <typename E, int CG, int BN>
void gated_tile(const LinearCall& c, const Matrix& x, const Matrix& w) {
    using Epi = EpiGated<E, BN>;
    Epi epi{};
    epi.h = tiled<E, Epi::kBytes>(c.y, c.rows, c.out, c.y_stride);
    if (c.pre) {
        epi.gate = tiled<E, Epi::kBytes>(c.pre, c.rows, c.out, c.pre_stride);
        epi.up = tiled<E, Epi::kBytes>(static_cast<E*>(c.pre) + c.out, c.rows, c.out, c.pre_stride);
    }
    epi.bias = c.bias;
    epi.bias_type = c.bias_type;
    epi.activation = c.activation;
    epi.has_pre = c.pre != nullptr;
    launch_gemm<E, CG, BN, false, false>("k_gated", x, w, c.out, static_cast<int>(c.out), 1, kInput, epi, c.stream);
}

template <typename E, bool GATED, int R>
void few_rows(const LinearCall& c) {
    FewRows<E> a{};
    a.x = static_cast<const E*>(c.x);
    a.weight = static_cast<const E*>(c.weight);
    a.bias = c.bias;
    a.residual = c.residual;
    a.y = c.y;
    a.pre = static_cast<E*>(c.pre);
    a.x_stride = c.x_stride;
    a.weight_stride = c.weight_stride;
    a.residual_stride = c.residual_stride;
    a.y_stride = c.y_stride;
    a.pre_stride = c.pre_stride;
    a.rows = static_cast<int>(c.rows);
    a.in = static_cast<int>(c.in);
    a.out = static_cast<int>(c.out);
    a.bias_type = c.bias_type;
    a.activation = c.activation;
    a.y_type = c.y_type;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(c.out, kFewWarps), kSms * 8)), static_cast<unsigned>(ceil_div(c.rows, R)));
    const bool wide = aligned(c.x, 16) && aligned(c.weight, 16) && (c.rows == 1 || c.x_stride % 8 == 0) &&
        (c.weight_stride % 8 == 0 || (c.out == 1 && !GATED));
    if (wide) {
        launch_chain("k_few_rows", k_few_rows<E, GATED, R, true>, grid, 32 * kFewWarps, 0, c.stream, true, a);
    } else {
        launch_chain("k_few_rows", k_few_rows<E, GATED, R, false>, grid, 32 * kFewWarps, 0, c.stream, true, a);
    }
    check(cudaGetLastError(), "few rows");
}
template <typename E, bool GATED>
void few_rows(const LinearCall& c) {
    if (c.rows == 1) {
        few_rows<E, GATED, 1>(c);
    } else if (c.rows <= 4) {
        few_rows<E, GATED, 4>(c);
    } else {
        few_rows<E, GATED, 8>(c);
    }
}

template <typename E>
void linear_forward(const LinearCall& c) {
    const int64_t columns = c.gated ? 2 * c.out : c.out;
    if (is_few(c.rows, c.in, c.out, c.gated)) {
        c.gated ? few_rows<E, true>(c) : few_rows<E, false>(c);
        return;
    }
    const Workspace at(c.rows, c.in, c.out, c.gated, c.what);
    PackJob jobs[2]{};
    const Matrix x = operand<E>(c.x, c.rows, c.in, c.x_stride, c.workspace + at.x, jobs[0]);
    const Matrix w = operand<E>(c.weight, columns, c.in, c.weight_stride, c.workspace + at.weight, jobs[1]);
    pack<E>(jobs, kInput, c.stream);
    const GemmPlan p = plan_gemm(c.rows, columns, c.in, false);
    if (c.gated) {
        if (p.bn == 256) {
            gated_tile<E, 2, 256>(c, x, w);
        } else if (p.bn == 128) {
            gated_tile<E, 2, 128>(c, x, w);
        } else {
            gated_tile<E, 1, 64>(c, x, w);
        }
    } else if (c.y_type == T8B_F32) {
        if (p.bn == 256) {
            forward_tile<E, float, 2, 256>(c, x, w);
        } else if (p.bn == 128) {
            forward_tile<E, float, 2, 128>(c, x, w);
        } else {
            forward_tile<E, float, 1, 64>(c, x, w);
        }
    } else {
        if (p.bn == 256) {
            forward_tile<E, E, 2, 256>(c, x, w);
        } else if (p.bn == 128) {
            forward_tile<E, E, 2, 128>(c, x, w);
        } else {
            forward_tile<E, E, 1, 64>(c, x, w);
        }
    }
}

// out [a.rows][b.rows] = A . B^T without bias or activation, in E; the parts of a split k go to
// `parts`, and what is left to do to `join`.
template <typename E, int CG, int BN, bool A_MN>
void product_tile(const char* label, const Matrix& a, const Matrix& b, int splits, int after, void* out, int64_t stride,
                  float* parts, Join& join, cudaStream_t stream) {
    if (splits == 1) {
        using Epi = EpiLinear<E, E, BN, false>;
        Epi epi{};
        epi.y = tiled<E, Epi::kBytes>(out, a.rows, b.rows, stride);
        launch_gemm<E, CG, BN, A_MN, true>(label, a, b, b.rows, 0, 1, after, epi, stream);
        return;
    }
    using Epi = EpiLinear<E, float, BN, false>;
    Epi epi{};
    const int64_t rows = split_rows(a.rows), pitch = split_pitch(b.rows);
    epi.y = tiled<float, Epi::kBytes>(parts, rows * splits, b.rows, pitch);
    epi.split_rows = static_cast<int>(rows);
    launch_gemm<E, CG, BN, A_MN, true>(label, a, b, b.rows, 0, splits, after, epi, stream);
    join.parts = parts;
    join.part_elements = static_cast<size_t>(rows) * pitch;
    join.splits = splits;
    join.pitch = static_cast<int>(pitch);
    join.rows = static_cast<int>(a.rows);
    join.columns = static_cast<int>(b.rows);
    join.out = out;
    join.stride = stride;
    join.blocks = blocks(a.rows * (pitch / 4), 256);
}
template <typename E, bool A_MN>
void product(const char* label, const Matrix& a, const Matrix& b, const GemmPlan& p, int after, void* out, int64_t stride,
             float* parts, Join& join, cudaStream_t stream) {
    if (p.bn == 256) {
        product_tile<E, 2, 256, A_MN>(label, a, b, p.splits, after, out, stride, parts, join, stream);
    } else if (p.bn == 128) {
        product_tile<E, 2, 128, A_MN>(label, a, b, p.splits, after, out, stride, parts, join, stream);
    } else {
        product_tile<E, 1, 64, A_MN>(label, a, b, p.splits, after, out, stride, parts, join, stream);
    }
}

template <typename E, bool GATED, int V>
void activation_grad(const LinearGradCall& c, E* dz, int64_t pitch, float* sums) {
    const int columns = static_cast<int>(c.out);
    const dim3 grid(blocks(columns, 32 * V), grad_parts(c.rows, c.out));
    constexpr size_t kRing = V == 8 ? kGradSmem : 0;
    static_assert(grad_ring_bytes<E, GATED, V>() <= kRing, "ring");
    static uint64_t configured = 0;
    allow_smem(k_activation_grad<E, GATED, V>, kRing, configured);
    launch_chain("k_activation_grad", k_activation_grad<E, GATED, V>, grid, dim3(32, kGradRows), kRing, c.stream, true,
           static_cast<const E*>(c.dy), c.dy_stride, static_cast<const E*>(c.pre), c.pre_stride, c.rows, columns, c.activation, dz,
           pitch, sums);
    check(cudaGetLastError(), "activation gradient");
}

template <typename E>
void linear_backward(const LinearGradCall& c) {
    const int64_t columns = c.gated ? 2 * c.out : c.out;
    const Workspace at(c.rows, c.in, c.out, c.gated, c.what);
    // dz is dy itself where there is neither a gate nor an activation and its rows suit TMA
    E* dz_out = (c.what & T8B_WORKSPACE_DZ) != 0 ? reinterpret_cast<E*>(c.workspace + at.dz) : nullptr;
    float* sums = c.dbias ? reinterpret_cast<float*>(c.workspace + at.sums) : nullptr;
    Matrix dz{c.dy, c.rows, columns, tma_pitch(c.rows, columns, c.dy_stride, sizeof(E))};
    if (dz_out) dz = Matrix{dz_out, c.rows, columns, static_cast<int64_t>(at.dz_pitch)};
    if (dz_out || sums) {
        // eight columns a thread where every row of dy, pre and dz starts on a 16-byte boundary
        const bool wide = c.out % 8 == 0 && aligned(c.dy, 16) && c.dy_stride % 8 == 0 &&
            (c.pre == nullptr || (aligned(c.pre, 16) && c.pre_stride % 8 == 0));
        const int64_t pitch = static_cast<int64_t>(at.dz_pitch);
        if (c.gated) {
            wide ? activation_grad<E, true, 8>(c, dz_out, pitch, sums) : activation_grad<E, true, 1>(c, dz_out, pitch, sums);
        } else {
            wide ? activation_grad<E, false, 8>(c, dz_out, pitch, sums) : activation_grad<E, false, 1>(c, dz_out, pitch, sums);
        }
    }
    // operands are packed first, so that the two products are neighbours in the chain
    PackJob jobs[2]{};
    Matrix w{}, x{};
    if (c.dx) w = operand<E>(c.weight, columns, c.in, c.weight_stride, c.workspace + at.weight, jobs[0]);
    if (c.dweight) x = operand<E>(c.x, c.rows, c.in, c.x_stride, c.workspace + at.x, jobs[1]);
    pack<E>(jobs, dz_out || sums ? kBeside : kInput, c.stream);
    int after = kInput;
    Totals totals{};
    if (c.dx) {
        product<E, false>("k_input_grad", dz, transposed(w), input_grad_plan(c.rows, c.in, columns), after, c.dx, c.dx_stride,
                          reinterpret_cast<float*>(c.workspace + at.input_parts), totals.input, c.stream);
        after = kBeside;
    }
    if (c.dweight) {
        product<E, true>("k_weight_grad", transposed(dz), transposed(x), weight_grad_plan(c.rows, c.in, columns), after, c.dweight,
                         c.dweight_stride, reinterpret_cast<float*>(c.workspace + at.weight_parts), totals.weight, c.stream);
    }
    unsigned grid = totals.weight.blocks + totals.input.blocks;
    if (sums) {
        totals.sums = sums;
        totals.sums_rows = grad_parts(c.rows, c.out);
        totals.bias_columns = static_cast<int>(columns);
        totals.dbias = c.dbias;
        totals.bias_type = c.bias_type;
        grid += blocks(columns, 32);
    }
    if (grid > 0) launch_chain("k_totals", k_totals<E>, grid, dim3(32, 8), 0, c.stream, true, totals);
    check(cudaGetLastError(), "linear backward");
}

}  // namespace op
}  // namespace t8b
