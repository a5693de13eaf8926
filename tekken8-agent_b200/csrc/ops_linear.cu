// C entries of the linear map and the gated projection: argument checks, and the count of waits
// that ran out.
#include <mutex>

#include "ops_linear.cuh"

namespace t8b {
namespace op {

extern template void linear_forward<bf16>(const LinearCall&);
extern template void linear_forward<f16>(const LinearCall&);
extern template void linear_backward<bf16>(const LinearGradCall&);
extern template void linear_backward<f16>(const LinearGradCall&);

// Only ever counted up: a reader that cleared it could lose a stall counted after its read.
__device__ unsigned g_stalls;

unsigned* stall_count() {
    static std::atomic<unsigned*> counts[64];
    int device = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    std::atomic<unsigned*>& count = counts[device & 63];
    unsigned* p = count.load(std::memory_order_acquire);
    if (p == nullptr) {
        check(cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_stalls), "stall count");
        count.store(p, std::memory_order_release);
    }
    return p;
}

namespace {

constexpr int64_t kMostRows = (1ll << 31) - 1024, kMostColumns = 1 << 22;

void check_sizes(const char* what, int64_t rows, int64_t in, int64_t out) {
    if (rows < 0 || rows > kMostRows) raise(T8B_EINVAL, std::string(what) + ": rows out of range");
    if (in < 1 || in > kMostColumns || out < 1 || out > kMostColumns) {
        raise(T8B_EINVAL, std::string(what) + ": features must be from 1 to 4194304");
    }
}

void check_types(const char* what, int type, bool bias, int bias_type, int y_type, int activation) {
    if (type != T8B_BF16 && type != T8B_F16) raise(T8B_EINVAL, std::string(what) + ": operands are bf16 or f16");
    if (bias && bias_type != T8B_F32 && bias_type != type) raise(T8B_EINVAL, std::string(what) + ": the bias is fp32 or of the operands' type");
    if (y_type != T8B_F32 && y_type != type) raise(T8B_EINVAL, std::string(what) + ": the output is fp32 or of the operands' type");
    if (activation < T8B_LINEAR || activation > T8B_TANH) raise(T8B_EINVAL, std::string(what) + ": unknown activation");
}

void check_workspace(const char* what, const void* workspace, size_t have, size_t need) {
    if (need > 0 && (workspace == nullptr || have < need || !aligned(workspace, 256))) {
        raise(T8B_EINVAL, std::string(what) + ": the workspace is missing, not 256-byte aligned or below " + std::to_string(need) + " bytes");
    }
}

void forward(const char* what, int type, LinearCall& c, void* workspace, size_t workspace_bytes) {
    check_sizes(what, c.rows, c.in, c.out);
    check_types(what, type, c.bias != nullptr, c.bias_type, c.y_type, c.activation);
    const int64_t columns = c.gated ? 2 * c.out : c.out;
    const size_t ys = type_size(c.y_type);
    check_matrix(what, c.x, c.rows, c.in, c.x_stride, 2);
    check_matrix(what, c.weight, columns, c.in, c.weight_stride, 2);
    check_matrix(what, c.y, c.rows, c.out, c.y_stride, ys);
    if (c.residual) check_matrix(what, c.residual, c.rows, c.out, c.residual_stride, ys);
    if (c.pre) check_matrix(what, c.pre, c.rows, columns, c.pre_stride, 2);
    if (c.bias) check_elements(what, c.bias, type_size(c.bias_type));
    if (c.rows == 0) return;
    const Span x(c.x, c.rows, c.in, c.x_stride, 2), w(c.weight, columns, c.in, c.weight_stride, 2);
    const Span y(c.y, c.rows, c.out, c.y_stride, ys), pre(c.pre, c.rows, columns, c.pre_stride, 2);
    const Span residual(c.residual, c.rows, c.out, c.residual_stride, ys);
    const Span bias(c.bias, 1, columns, columns, type_size(c.bias_type));
    const bool in_place = c.residual == c.y && c.residual_stride == c.y_stride;
    if (y.overlaps(x) || y.overlaps(w) || y.overlaps(pre) || y.overlaps(bias) || (y.overlaps(residual) && !in_place) ||
        pre.overlaps(x) || pre.overlaps(w) || pre.overlaps(residual) || pre.overlaps(bias)) {
        raise(T8B_EINVAL, std::string(what) + ": an output overlaps another argument");
    }
    if (!is_few(c.rows, c.in, c.out, c.gated)) {
        if (!tma_rows(c.x, c.rows, c.x_stride, 2)) c.what |= T8B_WORKSPACE_X;
        if (!tma_rows(c.weight, columns, c.weight_stride, 2)) c.what |= T8B_WORKSPACE_WEIGHT;
    }
    check_workspace(what, workspace, workspace_bytes, Workspace(c.rows, c.in, c.out, c.gated, c.what).bytes);
    c.workspace = static_cast<unsigned char*>(workspace);
    if (type == T8B_BF16) {
        linear_forward<bf16>(c);
    } else {
        linear_forward<f16>(c);
    }
}

void backward(const char* what, int type, LinearGradCall& c, void* workspace, size_t workspace_bytes) {
    check_sizes(what, c.rows, c.in, c.out);
    check_types(what, type, c.dbias != nullptr, c.bias_type, type, c.activation);
    const int64_t columns = c.gated ? 2 * c.out : c.out;
    check_matrix(what, c.dy, c.rows, c.out, c.dy_stride, 2);
    const bool reads_pre = c.gated || c.activation != T8B_LINEAR;
    if (reads_pre) {
        check_matrix(what, c.pre, c.rows, columns, c.pre_stride, 2);
    } else {
        c.pre = nullptr;
    }
    if (c.dx) check_matrix(what, c.weight, columns, c.in, c.weight_stride, 2);
    if (c.dx) check_matrix(what, c.dx, c.rows, c.in, c.dx_stride, 2);
    if (c.dweight) check_matrix(what, c.x, c.rows, c.in, c.x_stride, 2);
    if (c.dweight) check_matrix(what, c.dweight, columns, c.in, c.dweight_stride, 2);
    if (c.dbias) check_elements(what, c.dbias, type_size(c.bias_type));
    if (c.rows == 0) {
        if (c.dweight) {
            check(cudaMemset2DAsync(c.dweight, c.dweight_stride * 2, 0, c.in * 2, columns, c.stream), "clear dweight");
        }
        if (c.dbias) check(cudaMemsetAsync(c.dbias, 0, columns * type_size(c.bias_type), c.stream), "clear dbias");
        return;
    }
    const Span dy(c.dy, c.rows, c.out, c.dy_stride, 2), pre(c.pre, c.rows, columns, c.pre_stride, 2);
    const Span x(c.dweight ? c.x : nullptr, c.rows, c.in, c.x_stride, 2);
    const Span w(c.dx ? c.weight : nullptr, columns, c.in, c.weight_stride, 2);
    const Span out[3] = {Span(c.dx, c.rows, c.in, c.dx_stride, 2), Span(c.dweight, columns, c.in, c.dweight_stride, 2),
                         Span(c.dbias, 1, columns, columns, type_size(c.bias_type))};
    for (int i = 0; i < 3; ++i) {
        if (out[i].overlaps(dy) || out[i].overlaps(pre) || out[i].overlaps(x) || out[i].overlaps(w) || out[i].overlaps(out[(i + 1) % 3])) {
            raise(T8B_EINVAL, std::string(what) + ": an output overlaps another argument");
        }
    }
    c.what = T8B_WORKSPACE_BACKWARD;
    if (c.dweight && !tma_rows(c.x, c.rows, c.x_stride, 2)) c.what |= T8B_WORKSPACE_X;
    if (c.dx && !tma_rows(c.weight, columns, c.weight_stride, 2)) c.what |= T8B_WORKSPACE_WEIGHT;
    if ((c.dx || c.dweight) && (reads_pre || !tma_rows(c.dy, c.rows, c.dy_stride, 2))) c.what |= T8B_WORKSPACE_DZ;
    check_workspace(what, workspace, workspace_bytes, Workspace(c.rows, c.in, c.out, c.gated, c.what).bytes);
    c.workspace = static_cast<unsigned char*>(workspace);
    if (type == T8B_BF16) {
        linear_backward<bf16>(c);
    } else {
        linear_backward<f16>(c);
    }
}

size_t workspace_size(int64_t rows, int64_t in, int64_t out, bool gated, int what) {
    if (rows < 1 || rows > kMostRows || in < 1 || out < 1 || in > kMostColumns || out > kMostColumns) return 0;
    return Workspace(rows, in, out, gated, what).bytes;
}

}  // namespace
}  // namespace op
}  // namespace t8b

using namespace t8b;
using namespace t8b::op;

extern "C" size_t t8b_linear_workspace(int64_t rows, int64_t in, int64_t out, int what) {
    return workspace_size(rows, in, out, false, what);
}
extern "C" size_t t8b_gated_workspace(int64_t rows, int64_t in, int64_t out, int what) {
    return workspace_size(rows, in, out, true, what);
}

extern "C" int t8b_linear_forward(int type, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                  const void* bias, int bias_type, int activation, const void* residual,
                                  int64_t residual_stride, int64_t rows, int64_t in, int64_t out, void* y, int y_type,
                                  int64_t y_stride, void* pre, int64_t pre_stride, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    return guarded([&] {
        LinearCall c{x, weight, bias, residual, y, pre, x_stride, weight_stride, residual_stride, y_stride, pre_stride, rows, in,
                     out, bias_type, activation, y_type, false, 0, nullptr, static_cast<cudaStream_t>(stream)};
        forward("linear", type, c, workspace, workspace_bytes);
    });
}

extern "C" int t8b_gated_forward(int type, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                 const void* bias, int bias_type, int activation, int64_t rows, int64_t in, int64_t out,
                                 void* h, int64_t h_stride, void* pre, int64_t pre_stride, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    return guarded([&] {
        LinearCall c{x, weight, bias, nullptr, h, pre, x_stride, weight_stride, 0, h_stride, pre_stride, rows, in, out,
                     bias_type, activation, type, true, 0, nullptr, static_cast<cudaStream_t>(stream)};
        forward("gated", type, c, workspace, workspace_bytes);
    });
}

extern "C" int t8b_linear_backward(int type, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                   const void* weight, int64_t weight_stride, const void* pre, int64_t pre_stride,
                                   int bias_type, int activation, int64_t rows, int64_t in, int64_t out, void* dx,
                                   int64_t dx_stride, void* dweight, int64_t dweight_stride, void* dbias, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    return guarded([&] {
        LinearGradCall c{dy, x, weight, pre, dx, dweight, dbias, dy_stride, x_stride, weight_stride, pre_stride, dx_stride,
                         dweight_stride, rows, in, out, bias_type, activation, false, 0, nullptr, static_cast<cudaStream_t>(stream)};
        backward("linear", type, c, workspace, workspace_bytes);
    });
}

extern "C" int t8b_gated_backward(int type, const void* dh, int64_t dh_stride, const void* x, int64_t x_stride,
                                  const void* weight, int64_t weight_stride, const void* pre, int64_t pre_stride,
                                  int bias_type, int activation, int64_t rows, int64_t in, int64_t out, void* dx,
                                  int64_t dx_stride, void* dweight, int64_t dweight_stride, void* dbias, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    return guarded([&] {
        LinearGradCall c{dh, x, weight, pre, dx, dweight, dbias, dh_stride, x_stride, weight_stride, pre_stride, dx_stride,
                         dweight_stride, rows, in, out, bias_type, activation, true, 0, nullptr, static_cast<cudaStream_t>(stream)};
        backward("gated", type, c, workspace, workspace_bytes);
    });
}

extern "C" int t8b_operators_status(void* stream) {
    return guarded([&] {
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        static std::mutex mutex;
        static unsigned reported[64];
        int device = 0;
        check(cudaGetDevice(&device), "cudaGetDevice");
        unsigned count = 0;
        check(cudaMemcpyAsync(&count, stall_count(), sizeof(count), cudaMemcpyDeviceToHost, st), "read stall count");
        check(cudaStreamSynchronize(st), "read stall count");
        const std::lock_guard<std::mutex> lock(mutex);
        unsigned& last = reported[device & 63];
        if (static_cast<int>(count - last) <= 0) return;  // nothing new, or another caller has read further
        last = count;
        raise(T8B_ECUDA, "a wait inside an operator's kernel ran out");
    });
}

namespace t8b {
namespace op {
namespace {

// One thread waits as the products' kernels do, on a barrier that nothing arrives at, and counts the
// stall as they do once `limit` polls are over.
__global__ void k_stall(uint32_t limit, unsigned* stalls) {
    __shared__ uint64_t bar;
    __shared__ int abort;
    if (threadIdx.x != 0) return;
    abort = 0;
    tc::bar_init(&bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!tc::bar_wait(&bar, 0, &abort, limit)) atomicAdd(stalls, 1u);
}

}  // namespace
}  // namespace op
}  // namespace t8b

extern "C" int t8b_debug_operators_stall(uint32_t spin_limit, void* stream) {
    return guarded([&] {
        if (spin_limit == 0 || spin_limit > (1u << 20)) raise(T8B_EINVAL, "operators stall: 1 to 2^20 polls");
        launch("k_stall", k_stall, 1, 32, 0, static_cast<cudaStream_t>(stream), spin_limit, stall_count());
        check(cudaGetLastError(), "operators stall");
    });
}
