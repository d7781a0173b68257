// Python extension `_native`: the host path between the Python functions and libbi8.so.
//
// Every public operation is one call into this module: it validates its operands, allocates the results and the scratch from
// torch's caching allocator, and enqueues the kernels through the C ABI of include/bi8.h on torch's current stream.  Written
// against the CPython call protocol (METH_FASTCALL) without a binding layer, because a decode-sized layer is 9 us of device
// time: the same steps in Python (tensor views, torch.empty, attribute look-ups, one ctypes call with twenty converted
// arguments) took 40 us per call and were what bounded every call below about 50 us.
//
// Nothing here computes: the operations' meaning, shapes and layouts are described in triton_functions.py, and there is no
// path for tensors that are not on a CUDA device.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <optional>
#include <string>
#include <vector>

#include "../../include/bi8.h"

namespace {

using at::Tensor;

// ---- errors: the Python exception types that the functions have always raised ------------------------------------------
struct PyFail {
    PyObject* type;          // borrowed: a builtin exception class or g_error_class
    std::string text;
};
PyObject* g_error_class = nullptr;       // blockwise_int8_linear_b200._lib.Bi8Error, set when the module is loaded

[[noreturn]] void value_error(std::string text) { throw PyFail{PyExc_ValueError, std::move(text)}; }
[[noreturn]] void assertion(const char* text) { throw PyFail{PyExc_AssertionError, text}; }

void check(int status, const char* what) {
    if (status != BI8_OK)
        throw PyFail{g_error_class ? g_error_class : PyExc_RuntimeError,
                     std::string(what) + " failed with status " + std::to_string(status) + ": " + bi8_last_error_string()};
}

std::string shape_of(const Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}
std::string shape_of(int64_t a, int64_t b) { return "[" + std::to_string(a) + ", " + std::to_string(b) + "]"; }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return BI8_BF16;
        case at::kHalf: return BI8_F16;
        case at::kFloat: return BI8_F32;
        default: value_error(std::string("unsupported dtype ") + c10::toString(t) + ": expected bfloat16, float16 or float32");
    }
}

// ---- allocation and streams ---------------------------------------------------------------------------------------------
// the allocator behind torch.empty, without the dispatcher in front of it
Tensor empty_on(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// Sizes of the buffers that one call carves out of a single allocation.
struct Carve {
    int64_t bytes = 0;
    int64_t take(int64_t n) {
        const int64_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
};

// Scratch of one call: partial results of divided tiles, quantized activations that no caller sees.  A call is several launches, and
// the interpreter lock is not held while they are enqueued, so two threads that share a stream may enqueue theirs
// alternately, and calls on forked streams of one capture become branches of a graph that may run at the same time: scratch
// belongs to the call, not to its stream or capture.  The allocator gives the memory to others only behind what the
// call has enqueued on its stream (the returned tensor is held until then), and while a stream is captured it takes it
// from the capture's memory pool, which stays reserved for the graph's lifetime.
Tensor scratch(const Tensor& like, int64_t bytes) { return bytes > 0 ? empty_on(like, {bytes}, at::kByte) : Tensor(); }

// Makes the operand's device current for a call and names its current stream.
struct OnDevice {
    c10::cuda::CUDAGuard guard;
    c10::cuda::CUDAStream stream;
    explicit OnDevice(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index())) {}
    void* raw() const { return stream.stream(); }
};

// ---- matrices -----------------------------------------------------------------------------------------------------------
// A matrix with contiguous rows: where it lies, its row pitch in elements, and the tensor that owns it.
struct Mat {
    Tensor owner;
    const void* ptr = nullptr;
    int64_t rows = 0, cols = 0, ld = 0;
};

bool rows_contiguous(int64_t rows, int64_t cols, int64_t s0, int64_t s1) {
    return (cols == 1 || s1 == 1) && (rows <= 1 || s0 >= cols);
}

Mat mat(const Tensor& t, int64_t rows, int64_t cols, int64_t s0, int64_t s1, bool transposed) {
    Mat m;
    m.rows = rows;
    m.cols = cols;
    if (rows_contiguous(rows, cols, s0, s1)) {
        m.owner = t;
        m.ld = rows > 1 ? s0 : std::max<int64_t>(cols, 1);
    } else {
        m.owner = (transposed ? t.t() : t).contiguous();
        m.ld = std::max<int64_t>(cols, 1);
    }
    m.ptr = m.owner.data_ptr();
    return m;
}

Mat mat2d(const Tensor& t) {
    if (t.dim() != 2) value_error("expected a 2-D tensor, got " + shape_of(t));
    return mat(t, t.size(0), t.size(1), t.stride(0), t.stride(1), false);
}

Mat mat2d_t(const Tensor& t) {          // the transpose of a 2-D tensor
    return mat(t, t.size(1), t.size(0), t.stride(1), t.stride(0), true);
}

// [..., K] as [rows, K]
Mat mat_rows(const Tensor& t) {
    if (t.dim() == 2) return mat2d(t);
    if (t.dim() == 0) value_error("expected a tensor with a feature dimension, got a scalar");
    const int64_t k = t.size(-1), rows = k ? t.numel() / k : t.numel();
    if (t.is_contiguous()) return mat(t, rows, k, k, 1, false);
    return mat2d(t.reshape({-1, k}));
}

void need_cuda(const Tensor& t) {
    if (!t.is_cuda()) assertion("x.is_cuda");
}

// Row pitch of a quantized matrix: the next multiple of 16 bytes, which is what the wide kernels and the tensor-core GEMM take.
int64_t pitch16(int64_t n) { return (n + 15) / 16 * 16; }

// int8 [rows, cols], dense, or (`pitched`) with rows that begin on 16-byte boundaries: a view of a wider buffer where cols is not
// a multiple of 16
Tensor empty_q(const Tensor& like, int64_t rows, int64_t cols, bool pitched) {
    const int64_t ld = pitched ? pitch16(cols) : cols;
    Tensor t = empty_on(like, {rows, ld}, at::kChar);
    return ld == cols ? t : t.narrow(1, 0, cols);
}

// Copy with a 16-byte aligned row pitch of an int8 operand that has none; the bytes between K and the pitch are never read.  What
// is copied is the matrix that `m` describes, at its address and with its pitch: the owner itself may be that matrix or
// its transpose, which its shape does not tell where both have the same.
bool on_boundaries(const Mat& m) { return m.ld % 16 == 0 && reinterpret_cast<uintptr_t>(m.ptr) % 16 == 0; }
Mat repitch(const Mat& m, const OnDevice& on) {
    if (on_boundaries(m)) return m;
    Mat out = m;
    out.ld = pitch16(m.cols);
    out.owner = empty_on(m.owner, {m.rows, out.ld}, at::kChar);
    out.ptr = out.owner.data_ptr();
    check(bi8_copy_rows(static_cast<const int8_t*>(m.ptr), m.ld, static_cast<int8_t*>(out.owner.data_ptr()), out.ld, m.rows, m.cols, on.raw()),
          "bi8_copy_rows");
    return out;
}

// Whether that is worth its launches.  Without it the GEMM is the CUDA-core kernel's, whose time grows with K for any output: against copy
// and tensor cores 4.5 and 5 us at K = 65 (1 to 40 rows, 64 to 4000 columns), 7 and 5 at 129, 11 and 6 at 257, 20 and 7 at 513, 36
// and 8 at 1001; and with the output for any K: 1024 x 2000 takes 11 and 7 us at K = 17, 19 and 7 at 65, 29 and 8 at 129, 8192 x 4096
// takes 126 and 24, 260 and 28, 407 and 35.  A launch is 2.5 us of host time: the lines are where it is paid for.
bool worth_repitch(int64_t m, int64_t n, int64_t k) { return k % 16 != 0 && (k >= 256 || m * n >= (1ll << 27) / (k + 64)); }

// ---- quantizers ---------------------------------------------------------------------------------------------------------
struct Quantized {
    Tensor q, s;
    int64_t ld() const { return std::max(q.stride(0), q.size(1)); }      // of what empty_q gives, a single row's too
};

// Whether a quantized tensor that a caller gets has a row pitch of 16 bytes.  Callers may view, save or hand on what they get, so it
// is dense, except for large 16-bit matrices: there the re-pitching copy that the GEMM would make of it costs more than a
// launch, and such callers have always got a view.
bool pitched_result(const Tensor& x, int64_t block) {
    const int64_t r = x.size(0), c = x.size(1);
    return x.element_size() == 2 && block % 16 == 0 && r * c >= (1 << 22) && std::min(r, c) >= 256;
}

// `operand`: the result goes into a GEMM and to nobody else, so it gets the pitch that the GEMM wants
Quantized quantize_rowwise(const Tensor& x, int64_t block, bool operand) {
    need_cuda(x);
    OnDevice on(x);
    const Mat m = mat2d(x);
    const int code = dtype_code(x.scalar_type());
    Quantized r{empty_q(x, m.rows, m.cols, operand || pitched_result(x, block)), empty_on(x, {ceil_div(m.cols, block), m.rows}, at::kFloat)};
    check(bi8_quantize_rowwise_pitched(m.ptr, code, m.ld, r.q.mutable_data_ptr<int8_t>(), r.ld(), r.s.mutable_data_ptr<float>(), m.rows, m.cols,
                                       (int)block, on.raw()),
          "bi8_quantize_rowwise");
    return r;
}

Quantized quantize_colwise(const Tensor& x, int64_t block, bool operand) {
    need_cuda(x);
    OnDevice on(x);
    const Mat m = mat2d(x);
    const int code = dtype_code(x.scalar_type());
    Quantized r{empty_q(x, m.cols, m.rows, operand || pitched_result(x, block)), empty_on(x, {ceil_div(m.rows, block), m.cols}, at::kFloat)};
    check(bi8_quantize_colwise_pitched(m.ptr, code, m.ld, r.q.mutable_data_ptr<int8_t>(), r.ld(), r.s.mutable_data_ptr<float>(), m.rows, m.cols,
                                       (int)block, on.raw()),
          "bi8_quantize_colwise");
    return r;
}

struct Dual {
    Quantized row, col;
};

Dual quantize_dual(const Tensor& x, int64_t block) {
    need_cuda(x);
    OnDevice on(x);
    const Mat m = mat2d(x);
    const int code = dtype_code(x.scalar_type());
    const bool pitched = pitched_result(x, block);
    Dual d{{empty_q(x, m.rows, m.cols, pitched), empty_on(x, {ceil_div(m.cols, block), m.rows}, at::kFloat)},
           {empty_q(x, m.cols, m.rows, pitched), empty_on(x, {ceil_div(m.rows, block), m.cols}, at::kFloat)}};
    check(bi8_quantize_dual_pitched(m.ptr, code, m.ld, d.row.q.mutable_data_ptr<int8_t>(), d.row.ld(), d.row.s.mutable_data_ptr<float>(),
                                    d.col.q.mutable_data_ptr<int8_t>(), d.col.ld(), d.col.s.mutable_data_ptr<float>(), m.rows, m.cols,
                                    (int)block, on.raw()),
          "bi8_quantize_dual");
    return d;
}

void check_scales(const Tensor& s, int64_t nb, int64_t rows, int64_t block, const char* name) {
    if (s.dim() != 2 || s.size(0) != nb || s.size(1) != rows || s.scalar_type() != at::kFloat)
        value_error(std::string(name) + " must be float32 " + shape_of(nb, rows) + " for block " + std::to_string(block) + ", got " +
                    c10::toString(s.scalar_type()) + " " + shape_of(s));
}

Tensor dequantize(const Tensor& q, const Tensor& state, int64_t block, at::ScalarType out_type) {
    need_cuda(q);
    if (q.dim() != 2) value_error("expected a 2-D tensor, got " + shape_of(q));
    if (q.scalar_type() != at::kChar) value_error(std::string("expected an int8 tensor, got ") + c10::toString(q.scalar_type()));
    const int64_t m = q.size(0), k = q.size(1);
    check_scales(state, ceil_div(k, block), m, block, "state");
    OnDevice on(q);
    const Mat x = mat2d(q);
    const Tensor s = state.contiguous();
    Tensor out = empty_on(q, {m, k}, out_type);
    check(bi8_dequantize_rowwise_pitched(static_cast<const int8_t*>(x.ptr), x.ld, s.const_data_ptr<float>(), out.data_ptr(), dtype_code(out_type), m, k, (int)block, on.raw()),
          "bi8_dequantize_rowwise");
    return out;
}

// ---- GEMM ---------------------------------------------------------------------------------------------------------------
// Bias operand: a contiguous vector of a type the kernels read, or nothing.
struct Bias {
    Tensor owner;
    const void* ptr = nullptr;
    int code = 0;
    Bias(const Tensor& b, int64_t n) {
        if (!b.defined()) return;
        if (b.numel() != n) value_error("bias must have " + std::to_string(n) + " elements, got " + std::to_string(b.numel()));
        owner = (b.dim() == 1 ? b : b.reshape({n})).contiguous();
        const at::ScalarType t = owner.scalar_type();
        if (t != at::kBFloat16 && t != at::kHalf && t != at::kFloat) owner = owner.to(at::kFloat);
        ptr = owner.data_ptr();
        code = dtype_code(owner.scalar_type());
    }
};

// Workspace of a GEMM call: without seeds no parts of a tile meet in a cluster, and those that would have take one.
size_t gemm_workspace(int64_t m, int64_t n, int64_t k, int64_t block, int flags) {
    return flags & BI8_GEMM_NO_SEED ? bi8_gemm_workspace_bytes(m, n, k, (int)block) : bi8_gemm_workspace_used(m, n, k, (int)block);
}

struct Operands {
    Mat a, bt;
};

// Brings both int8 operands to the form the library takes: a [M, K] and b^T [N, K] with contiguous rows.
Operands gemm_operands(const Tensor& a, const Tensor& b, const OnDevice& on) {
    need_cuda(a);
    if (a.dim() != 2 || b.dim() != 2) value_error("expected 2-D operands, got " + shape_of(a) + " and " + shape_of(b));
    if (a.size(1) != b.size(0)) assertion("incompatible dimensions");
    if (a.scalar_type() != at::kChar || b.scalar_type() != at::kChar)
        value_error(std::string("operands must be int8, got ") + c10::toString(a.scalar_type()) + " and " + c10::toString(b.scalar_type()));
    Operands o{mat2d(a), mat2d_t(b)};
    // The tensor-core kernels need 16-byte aligned operand rows: where it is worth it both operands are re-pitched once.  Not for
    // a narrow output of more rows than the decode kernel takes: callers get the reference's order of operations there,
    // from the CUDA cores.
    const int64_t m = o.a.rows, n = o.bt.rows;
    if (worth_repitch(m, n, a.size(1)) && (m <= 64 || m * n >= 128 * 128)) {
        o.a = repitch(o.a, on);
        o.bt = repitch(o.bt, on);
    }
    return o;
}

Tensor gemm(const Tensor& a_in, const Tensor& b_in, const Tensor& state_x, const Tensor& state_w, const Tensor& bias_in, int64_t block,
            at::ScalarType out_type, int flags) {
    need_cuda(a_in);
    OnDevice on(a_in);
    const Operands o = gemm_operands(a_in, b_in, on);
    const int64_t m = o.a.rows, n = o.bt.rows, k = o.a.cols, nb = ceil_div(k, block);
    check_scales(state_x, nb, m, block, "state_x");
    check_scales(state_w, nb, n, block, "state_w");
    const Tensor sx = state_x.contiguous(), sw = state_w.contiguous();
    Tensor c = empty_on(a_in, {m, n}, out_type);
    const Bias bias(bias_in, n);
    const size_t ws_bytes = gemm_workspace(m, n, k, block, flags);
    const Tensor ws = scratch(a_in, (int64_t)ws_bytes);
    check(bi8_gemm_dequant(static_cast<const int8_t*>(o.a.ptr), o.a.ld, static_cast<const int8_t*>(o.bt.ptr), o.bt.ld, sx.const_data_ptr<float>(),
                           sw.const_data_ptr<float>(), bias.ptr, bias.code, c.data_ptr(), n, dtype_code(out_type), m, n, k, (int)block,
                           ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, flags, on.raw()),
          "bi8_gemm_dequant");
    return c;
}

Tensor block_partials(const Tensor& a, const Tensor& b, int64_t block, int flags) {
    need_cuda(a);
    OnDevice on(a);
    const Operands o = gemm_operands(a, b, on);
    const int64_t m = o.a.rows, n = o.bt.rows, k = o.a.cols;
    Tensor out = at::zeros({ceil_div(k, block), m, n}, at::TensorOptions().dtype(at::kInt).device(a.device()));
    check(bi8_gemm_block_partials(static_cast<const int8_t*>(o.a.ptr), o.a.ld, static_cast<const int8_t*>(o.bt.ptr), o.bt.ld,
                                  out.mutable_data_ptr<int32_t>(), m, n, k, (int)block, flags, on.raw()),
          "bi8_gemm_block_partials");
    return out;
}

// ---- producer step + quantizer + GEMM + residual ------------------------------------------------------------------------
// Operands of a fused producer step with a shared row pitch.
struct Pre {
    int op;
    Mat x, x2;
    Tensor weight;
    Pre(int op_, const Tensor& x_in, const Tensor& x2_in, const Tensor& w_in) : op(op_), x(mat_rows(x_in)) {
        if (op == BI8_PRE_SILU_MUL) {
            if (!x2_in.defined() || x2_in.sizes() != x_in.sizes() || x2_in.scalar_type() != x_in.scalar_type() || x2_in.device() != x_in.device())
                value_error("silu_mul needs a second operand with x's shape, dtype and device");
            x2 = mat_rows(x2_in);
            if (x2.ld != x.ld) {           // e.g. one of the two was copied: give both the same row pitch
                x = mat_rows(x_in.contiguous());
                x2 = mat_rows(x2_in.contiguous());
            }
        }
        if (op == BI8_PRE_RMSNORM && w_in.defined()) {
            if (w_in.numel() != x.cols) value_error("norm weight must have " + std::to_string(x.cols) + " elements, got " + std::to_string(w_in.numel()));
            weight = (w_in.dim() == 1 ? w_in : w_in.reshape({-1})).to(x_in.scalar_type()).contiguous();
        }
    }
    const void* weight_ptr() const { return weight.defined() ? weight.data_ptr() : nullptr; }
};

Quantized quantize_pre(int op, const Tensor& x_in, const Tensor& x2, const Tensor& weight, double eps, int64_t block) {
    need_cuda(x_in);
    if (x_in.dim() != 2) value_error("expected a 2-D tensor, got " + shape_of(x_in));
    OnDevice on(x_in);
    const Pre pre(op, x_in, x2, weight);
    const int64_t m = pre.x.rows, k = pre.x.cols;
    Quantized r{empty_q(x_in, m, k, false), empty_on(x_in, {ceil_div(k, block), m}, at::kFloat)};
    check(bi8_quantize_rowwise_pre_pitched(op, pre.x.ptr, pre.x2.ptr, dtype_code(x_in.scalar_type()), pre.x.ld, pre.weight_ptr(), (float)eps,
                                   r.q.mutable_data_ptr<int8_t>(), r.ld(), r.s.mutable_data_ptr<float>(), m, k, (int)block, on.raw()),
          "bi8_quantize_rowwise_pre");
    return r;
}

// y = pre(x) W^T (+ bias) (+ residual) for x [..., K] and the int8 weights as `w` = [N, K] (or, with `w_transposed`, its [K, N] view)
Tensor linear(int op, const Tensor& x_in, const Tensor& w, bool w_transposed, const Tensor& state_w, const Tensor& bias_in, const Tensor& x2,
              const Tensor& norm_weight, double eps, const Tensor& residual, const Tensor& out_in, int64_t block, at::ScalarType out_type, int flags) {
    need_cuda(x_in);
    if (w.dim() != 2) value_error("expected 2-D weights, got " + shape_of(w));
    if (x_in.dim() == 0 || x_in.size(-1) != w.size(w_transposed ? 0 : 1)) assertion("incompatible dimensions");
    if (w.scalar_type() != at::kChar) value_error(std::string("weights must be int8, got ") + c10::toString(w.scalar_type()));
    OnDevice on(x_in);
    const Pre pre(op, x_in, x2, norm_weight);
    Mat bt = w_transposed ? mat2d_t(w) : mat2d(w);
    const int64_t m = pre.x.rows, k = pre.x.cols, n = bt.rows, nb = ceil_div(k, block);
    check_scales(state_w, nb, n, block, "state_w");
    const Tensor sw = state_w.contiguous();
    c10::SmallVector<int64_t, 6> shape(x_in.sizes().begin(), x_in.sizes().end());
    shape.back() = n;
    Tensor out = out_in, res = residual;
    int64_t ldc = n, ldr = 0;
    auto check_2d = [&](const Tensor& t, const char* name) {
        if (t.dim() != 2 || t.size(0) != m || t.size(1) != n || t.scalar_type() != out_type || t.stride(1) != 1 || t.device() != x_in.device())
            value_error(std::string(name) + " must be " + c10::toString(out_type) + " " + shape_of(m, n) + " with contiguous rows on " + x_in.device().str());
        return m > 1 ? t.stride(0) : std::max<int64_t>(n, 1);
    };
    if (out.defined()) ldc = check_2d(out, "out");
    else out = empty_on(x_in, shape, out_type);
    if (res.defined()) {
        if (res.dim() != 2 && n > 0) res = res.reshape({-1, n});
        ldr = check_2d(res, "residual");
    }
    const Bias bias(bias_in, n);
    Tensor target = out;
    if (res.defined() && out.data_ptr() == res.data_ptr() && !(m <= 64 && bias.ptr == nullptr && n % 4 == 0 && k % 16 == 0 && ldc == ldr)) {
        target = empty_on(x_in, {m, n}, out_type);          // not the path that may update in place
        ldc = n;
    }
    const int x_code = dtype_code(x_in.scalar_type());
    const void* res_ptr = res.defined() ? res.data_ptr() : nullptr;
    auto fused = [&](int8_t* xq, float* sx, void* ws, size_t ws_bytes) {
        return bi8_gemm_dequant_fused_pre(op, pre.x.ptr, pre.x2.ptr, x_code, pre.x.ld, pre.weight_ptr(), (float)eps, xq, sx,
                                          static_cast<const int8_t*>(bt.ptr), bt.ld, sw.const_data_ptr<float>(), bias.ptr, bias.code, res_ptr, ldr,
                                          target.data_ptr(), ldc, dtype_code(out_type), m, n, k, (int)block, ws, ws_bytes, flags, on.raw());
    };
    auto finish = [&] {
        if (!target.is_same(out)) out.copy_(target);
        return out;
    };
    // The form that quantizes inside the GEMM needs no scratch, whose allocation is 0.6 us of such a call (one token through
    // 4096 x 4096: 8.8 us with it, 8.2 without).  Where that form does not apply nothing has been launched.
    if (m <= 16 && m * k <= BI8_ONE_LAUNCH_VALUES && k % 16 == 0) {
        const int rc = fused(nullptr, nullptr, nullptr, 0);
        if (rc != BI8_ERR_WORKSPACE) {
            check(rc, "bi8_gemm_dequant_fused_pre");
            return finish();
        }
    }
    const size_t ws_bytes = gemm_workspace(m, n, k, block, flags);
    // the quantized activations live in the call's scratch behind the GEMM's workspace
    Carve carve;
    carve.take((int64_t)ws_bytes);
    const int64_t xq_at = carve.take(m * pitch16(k)), sx_at = carve.take(nb * m * 4);
    // Weights whose rows are not 16-byte aligned (of a layer, a checkpoint's dense copy) are copied to rows that are where the GEMM is
    // long enough to gain from it.
    const bool copy_w = k % 16 != 0 && worth_repitch(m, n, k) && !on_boundaries(bt);
    const int64_t w_at = copy_w ? carve.take(n * pitch16(k)) : 0;
    const Tensor ws = scratch(x_in, carve.bytes);
    char* ws_ptr = ws.defined() ? static_cast<char*>(ws.data_ptr()) : nullptr;
    int8_t* xq = reinterpret_cast<int8_t*>(ws_ptr + xq_at);
    float* sx = reinterpret_cast<float*>(ws_ptr + sx_at);
    void* gemm_ws = ws_bytes ? ws_ptr : nullptr;
    if (k % 16 != 0) {
        // rows that are not 16-byte aligned: the activations are quantized into rows that are, with the copy in one launch if they are few
        // (one after another it is the copy first: the GEMM starts early behind the short quantizer)
        bi8_quantize_task tasks[2] = {};
        bi8_quantize_task &tw = tasks[0], &tx = tasks[1];
        if (copy_w) {
            tw.x = bt.ptr;
            tw.x_dtype = BI8_I8;
            tw.ldx = bt.ld;
            tw.rows = n;
            tw.cols = k;
            tw.q_row = reinterpret_cast<int8_t*>(ws_ptr + w_at);
            tw.ldq_row = pitch16(k);
            bt.ptr = tw.q_row;
            bt.ld = tw.ldq_row;
        }
        if (op == BI8_PRE_NONE) {
            tx.x = pre.x.ptr;
            tx.x_dtype = x_code;
            tx.ldx = pre.x.ld;
            tx.rows = m;
            tx.cols = k;
            tx.q_row = xq;
            tx.ldq_row = pitch16(k);
            tx.s_row = sx;
            check(bi8_quantize_many(copy_w ? tasks : &tx, copy_w ? 2 : 1, (int)block, on.raw()), "bi8_quantize_many");
        } else {
            if (copy_w) check(bi8_quantize_many(&tw, 1, (int)block, on.raw()), "bi8_quantize_many");
            check(bi8_quantize_rowwise_pre_pitched(op, pre.x.ptr, pre.x2.ptr, x_code, pre.x.ld, pre.weight_ptr(), (float)eps, xq, pitch16(k), sx, m, k,
                                                   (int)block, on.raw()),
                  "bi8_quantize_rowwise_pre");
        }
        check(bi8_gemm_dequant_residual(xq, pitch16(k), static_cast<const int8_t*>(bt.ptr), bt.ld, sx, sw.const_data_ptr<float>(), bias.ptr, bias.code,
                                        res_ptr, ldr, target.data_ptr(), ldc, dtype_code(out_type), m, n, k, (int)block, gemm_ws, ws_bytes,
                                        flags & ~BI8_GEMM_QUANT_IN_KERNEL, on.raw()),
              "bi8_gemm_dequant_residual");
        return finish();
    }
    check(fused(xq, sx, gemm_ws, ws_bytes), "bi8_gemm_dequant_fused_pre");
    return finish();
}

// ---- training: forward and backward as one autograd node ----------------------------------------------------------------
// What the Python side knows at call time; the backward pass looks it up again (block size and result type are module-level
// knobs, and the cache of quantized weights is a dict on the weight).
PyObject* g_config = nullptr;            // the module blockwise_int8_linear_b200.block_linear_config

int64_t config_block() {                 // with the interpreter lock
    PyObject* v = PyObject_GetAttrString(g_config, "GROUP_SIZE");
    if (!v) throw python_error();
    const long long b = PyLong_AsLongLong(v);
    Py_DECREF(v);
    if (b == -1 && PyErr_Occurred()) throw python_error();
    if (b < 1 || b > 0x7fffffff) value_error("block size must be positive, got " + std::to_string(b));
    return b;
}
at::ScalarType config_dtype() {          // with the interpreter lock
    PyObject* v = PyObject_GetAttrString(g_config, "INPUT_OUTPUT_TORCH_TYPE");
    if (!v) throw python_error();
    const bool is_dtype = THPDtype_Check(v);
    const at::ScalarType t = is_dtype ? reinterpret_cast<THPDtype*>(v)->scalar_type : at::kFloat;
    Py_DECREF(v);
    if (!is_dtype) throw PyFail{PyExc_TypeError, "INPUT_OUTPUT_TORCH_TYPE must be a torch.dtype"};
    (void)dtype_code(t);
    return t;
}

// A quantized matrix as the kernels see it: int8 rows with pitch ld, block scales [blocks, rows].
struct QRef {
    int8_t* q = nullptr;
    float* s = nullptr;
    int64_t rows = 0, cols = 0, ld = 0;
};

// Where a quantized [rows, cols] lies in one allocation of the call, and the reference to it once that exists.  The training
// passes keep no tensor of an intermediate result: one allocation per pass instead of two per quantization.
struct QPlan {
    int64_t rows = 0, cols = 0, q_at = 0, s_at = 0;
    QPlan() = default;
    QPlan(Carve& c, int64_t rows_, int64_t cols_, int64_t block) : rows(rows_), cols(cols_) {
        q_at = c.take(rows * pitch16(cols));
        s_at = c.take(ceil_div(cols, block) * rows * 4);
    }
    QRef in(void* mem) const {
        char* m = static_cast<char*>(mem);
        return {reinterpret_cast<int8_t*>(m + q_at), reinterpret_cast<float*>(m + s_at), rows, cols, pitch16(cols)};
    }
};

QRef ref_of(const Quantized& r) {
    return {static_cast<int8_t*>(r.q.data_ptr()), static_cast<float*>(r.s.data_ptr()), r.q.size(0), r.q.size(1),
            r.ld()};
}

// The quantizations of a pass, which share a launch where they are small.
struct Tasks {
    bi8_quantize_task list[4];
    int n = 0;
    // x row-wise and / or column-wise
    void add(const Mat& m, int code, const QRef* row, const QRef* col) {
        bi8_quantize_task t{};
        t.x = m.ptr;
        t.x_dtype = code;
        t.ldx = m.ld;
        t.rows = m.rows;
        t.cols = m.cols;
        if (row) {
            t.q_row = row->q;
            t.ldq_row = row->ld;
            t.s_row = row->s;
        }
        if (col) {
            t.q_col = col->q;
            t.ldq_col = col->ld;
            t.s_col = col->s;
        }
        list[n++] = t;
    }
    bool fits(int64_t block) const { return n > 0 && bi8_quantize_many_fits(list, n, (int)block) != 0; }
    void run(int64_t block, void* stream) const {
        if (n > 0) check(bi8_quantize_many(list, n, (int)block, stream), "bi8_quantize_many");
    }
};
// out = a b^T (+ bias); `ws` of at least bi8_gemm_workspace_used
void gemm_into(const QRef& a, const QRef& b, const Bias* bias, int64_t block, const Tensor& out, void* ws, size_t ws_bytes, void* stream) {
    check(bi8_gemm_dequant(a.q, a.ld, b.q, b.ld, a.s, b.s, bias ? bias->ptr : nullptr, bias ? bias->code : 0, out.data_ptr(), b.rows,
                           dtype_code(out.scalar_type()), a.rows, b.rows, a.cols, (int)block, ws_bytes ? ws : nullptr, ws_bytes, 0, stream),
          "bi8_gemm_dequant");
}

// One blocking of a weight from the cache dict under `key`, or undefined tensors.
Quantized cache_get(PyObject* cache, const char* key) {
    if (!cache) return {};
    pybind11::gil_scoped_acquire gil;
    PyObject* hit = PyDict_GetItemString(cache, key);
    if (hit && PyTuple_Check(hit) && PyTuple_GET_SIZE(hit) == 2)
        return {THPVariable_Unpack(PyTuple_GET_ITEM(hit, 0)), THPVariable_Unpack(PyTuple_GET_ITEM(hit, 1))};
    return {};
}
void cache_put(PyObject* cache, const char* key, const Quantized& r) {
    pybind11::gil_scoped_acquire gil;
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw python_error();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(r.q));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(r.s));
    const int rc = PyDict_SetItemString(cache, key, pair);
    Py_DECREF(pair);
    if (rc != 0) throw python_error();
}

Tensor as_bytes(const Tensor& like, int64_t bytes) { return empty_on(like, {std::max<int64_t>(bytes, 1)}, at::kByte); }

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Backward of y = x W^T + bias with both GEMMs in blockwise int8 (block_linear.py:85-112 in the reference).
struct LinearBackward : public Node {
    SavedVariable x;                     // x itself, or (x_quantized) the bytes of its column-wise int8 copy and scales
    SavedVariable weight;
    bool x_quantized = false, has_bias = false, fuse_dual = true;
    int64_t block = 0;
    std::vector<int64_t> x_sizes;
    PyObject* cache = nullptr;           // owned reference to the weight's cache dict, or null

    ~LinearBackward() override {
        if (cache && Py_IsInitialized()) {
            pybind11::gil_scoped_acquire gil;
            Py_DECREF(cache);
        }
    }
    std::string name() const override { return "blockwise_int8_linearBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        weight.reset_data();
    }
    variable_list apply(variable_list&& grads) override;
};

variable_list LinearBackward::apply(variable_list&& grads) {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    // A backward pass that is itself recorded: the bias gradient is a sum of G that can be differentiated again.  The two products
    // of quantized operands cannot.
    const bool want_b = has_bias && task_should_compute_output(2), recorded = at::GradMode::is_enabled() && grads[0].requires_grad();
    int64_t b = 0;
    at::ScalarType type;
    try {
        {
            pybind11::gil_scoped_acquire gil;
            b = config_block();
            type = config_dtype();
        }
        if (x_quantized && b != block)
            throw std::runtime_error("GROUP_SIZE changed between the forward and the backward pass of a BlockInt8Linear");
        std::lock_guard<std::mutex> lock(mutex_);
        auto self = getptr();
        const Tensor saved_x = x.unpack(self), w = weight.unpack(self);
        at::AutoDispatchBelowADInplaceOrView below_autograd;
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = want_b && !recorded;
        need_cuda(grads[0]);
        OnDevice on(grads[0]);
        const Mat g = mat_rows(grads[0]), wm = mat2d(w);
        const int g_code = dtype_code(grads[0].scalar_type()), w_code = dtype_code(w.scalar_type());
        const int64_t m = g.rows, n = g.cols, k = wm.cols;
        Mat xm;
        if (need_w && !x_quantized) xm = mat_rows(saved_x);

        // every intermediate result of this pass lies in one allocation
        const Quantized cached = need_x ? cache_get(cache, "col") : Quantized{};
        Quantized fresh;                                     // the weight's other blocking, where the cache is to keep it
        const size_t ws_x = need_x ? bi8_gemm_workspace_used(m, k, n, (int)b) : 0, ws_w = need_w ? bi8_gemm_workspace_used(n, k, m, (int)b) : 0,
                     ws_b = need_b ? bi8_column_sum_workspace_bytes(m, n) : 0,
                     ws_d = need_b && need_x && need_w && fuse_dual ? bi8_quantize_dual_sum_workspace_bytes(g_code, m, n, (int)b) : 0;
        Carve carve;
        const int64_t ws_at = carve.take((int64_t)std::max({ws_x, ws_w, ws_b, ws_d}));
        QPlan g_row, g_col, w_col, x_col;
        if (need_x) g_row = QPlan(carve, m, n, b);
        if (need_w) g_col = QPlan(carve, n, m, b);
        if (need_x && !cached.q.defined() && !cache) w_col = QPlan(carve, k, n, b);
        if (need_w && x_quantized) {
            Carve kept;
            x_col = QPlan(kept, k, m, b);                    // the layout in which train_linear saved it
        } else if (need_w) {
            x_col = QPlan(carve, k, m, b);
        }
        const Tensor mem = as_bytes(grads[0], carve.bytes);
        void* const base = mem.data_ptr();
        void* const ws = static_cast<char*>(base) + ws_at;
        void* const st = on.raw();

        // All operands first: G (in both blockings with one read, where the layer fuses them), the weight along N and the tokens of x.
        const QRef gr = need_x ? g_row.in(base) : QRef{}, gc = need_w ? g_col.in(base) : QRef{};
        Tasks tasks;
        if (need_x && need_w && fuse_dual) {
            tasks.add(g, g_code, &gr, &gc);
        } else {
            if (need_x) tasks.add(g, g_code, &gr, nullptr);
            if (need_w) tasks.add(g, g_code, nullptr, &gc);
        }
        QRef wt, xt;
        if (need_x) {
            // A cached blocking is still valid: unpacking the weight raised if it was modified since the forward pass.
            if (cached.q.defined()) wt = ref_of(cached);
            else {
                if (cache) {
                    fresh = Quantized{empty_q(w, k, n, true), empty_on(w, {ceil_div(n, b), k}, at::kFloat)};
                    wt = ref_of(fresh);
                } else {
                    wt = w_col.in(base);
                }
                tasks.add(wm, w_code, nullptr, &wt);
            }
        }
        if (need_w) {
            xt = x_col.in(x_quantized ? saved_x.data_ptr() : base);
            if (!x_quantized) tasks.add(xm, dtype_code(saved_x.scalar_type()), nullptr, &xt);
        }
        // small passes: the bias gradient rides in the same launch
        bool summed = false;
        if (need_b) {
            out[2] = empty_on(grads[0], {n}, grads[0].scalar_type());
            if (tasks.n > 0 && tasks.list[0].x == g.ptr) {
                tasks.list[0].sum = out[2].data_ptr();
                summed = tasks.fits(b);
                if (!summed) tasks.list[0].sum = nullptr;
            }
            if (!summed && ws_d && m > 0 && n > 0) {
                // larger ones: from the read that makes both blockings
                check(bi8_quantize_dual_sum(g.ptr, g_code, g.ld, gr.q, gr.ld, gr.s, gc.q, gc.ld, gc.s, out[2].data_ptr(), m, n, (int)b, ws, ws_d, st),
                      "bi8_quantize_dual_sum");
                for (int i = 1; i < tasks.n; ++i) tasks.list[i - 1] = tasks.list[i];
                --tasks.n;
                summed = true;
            }
        }
        tasks.run(b, st);
        if (fresh.q.defined()) cache_put(cache, "col", fresh);
        if (need_x) {
            // contraction over N, both operands blocked along N (block_linear.py:92-95)
            out[0] = empty_on(grads[0], x_sizes, type);
            gemm_into(gr, wt, nullptr, b, out[0], ws, ws_x, st);
        }
        if (need_w) {
            // contraction over the tokens, both operands blocked along M (block_linear.py:100-104)
            out[1] = empty_on(grads[0], {n, k}, type);
            gemm_into(gc, xt, nullptr, b, out[1], ws, ws_w, st);
        }
        if (need_b && !summed) {
            check(bi8_column_sum(g.ptr, g_code, g.ld, out[2].data_ptr(), m, n, ws_b ? ws : nullptr, ws_b, st), "bi8_column_sum");
        }
    } catch (const PyFail& e) {
        pybind11::gil_scoped_acquire gil;
        PyErr_SetString(e.type, e.text.c_str());
        python_error err;
        err.persist();
        throw err;
    }
    if (want_b && recorded) out[2] = grads[0].reshape({-1, grads[0].size(-1)}).sum(0);
    return out;
}

// y = x W^T (+ bias), every operand quantized on the fly, recorded for backward when a gradient is wanted.  With `fuse_dual`
// a layer whose weight is trained reads x once for both of its blockings and keeps the int8 transposed copy instead of x.
Tensor train_linear(const Tensor& x_in, const Tensor& w, const Tensor& bias_in, int64_t block, at::ScalarType type, bool fuse_dual, PyObject* cache) {
    need_cuda(x_in);
    if (x_in.dim() == 0 || w.dim() != 2 || x_in.size(-1) != w.size(1)) assertion("incompatible dimensions");
    const bool grad = at::GradMode::is_enabled() && (x_in.requires_grad() || w.requires_grad() || (bias_in.defined() && bias_in.requires_grad()));
    std::shared_ptr<LinearBackward> node;
    if (grad) {
        node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, w, bias_in));
    }
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below_autograd;
        OnDevice on(x_in);
        const Mat x = mat_rows(x_in), wm = mat2d(w);
        const int x_code = dtype_code(x_in.scalar_type()), w_code = dtype_code(w.scalar_type());
        const int64_t m = x.rows, n = wm.rows, k = wm.cols;
        const bool keep = node && w.requires_grad() && fuse_dual;
        const Quantized cached = cache_get(cache, "row");
        Quantized fresh;
        const size_t ws_bytes = bi8_gemm_workspace_used(m, n, k, (int)block);
        Carve carve, kept;
        const int64_t ws_at = carve.take((int64_t)ws_bytes);
        const QPlan x_row(carve, m, k, block), x_col = keep ? QPlan(kept, k, m, block) : QPlan();
        const QPlan w_row = !cached.q.defined() && !cache ? QPlan(carve, n, k, block) : QPlan();
        const Tensor mem = as_bytes(x_in, carve.bytes);
        void* const base = mem.data_ptr();
        void* const st = on.raw();
        const QRef xq = x_row.in(base);
        Tasks tasks;
        if (keep) {
            const Tensor saved = as_bytes(x_in, kept.bytes);
            const QRef xt = x_col.in(saved.data_ptr());
            tasks.add(x, x_code, &xq, &xt);
            node->x = SavedVariable(saved, false);
            node->x_quantized = true;
        } else {
            tasks.add(x, x_code, &xq, nullptr);
        }
        QRef wq;
        if (cached.q.defined()) {
            wq = ref_of(cached);
        } else if (cache) {
            fresh = Quantized{empty_q(w, n, k, true), empty_on(w, {ceil_div(k, block), n}, at::kFloat)};
            wq = ref_of(fresh);
            tasks.add(wm, w_code, &wq, nullptr);
        } else {
            wq = w_row.in(base);
            tasks.add(wm, w_code, &wq, nullptr);
        }
        tasks.run(block, st);
        if (fresh.q.defined()) cache_put(cache, "row", fresh);
        const Bias bias(bias_in, n);
        c10::SmallVector<int64_t, 6> shape(x_in.sizes().begin(), x_in.sizes().end());
        shape.back() = n;
        out = empty_on(x_in, shape, type);
        gemm_into(xq, wq, bias.ptr ? &bias : nullptr, block, out, static_cast<char*>(base) + ws_at, ws_bytes, st);
    }
    if (node) {
        if (!node->x_quantized) node->x = SavedVariable(x_in, false);
        node->weight = SavedVariable(w, false);
        node->has_bias = bias_in.defined();
        node->fuse_dual = fuse_dual;
        node->block = block;
        node->x_sizes = x_in.sizes().vec();
        if (cache) {
            pybind11::gil_scoped_acquire gil;
            Py_INCREF(cache);
            node->cache = cache;
        }
        torch::autograd::set_history(out, node);
    }
    return out;
}

// ---- decode step: rotary embedding and cache append ---------------------------------------------------------------------
Tensor rope_cache_append(const Tensor& qkv_in, const Tensor& cis_in, const Tensor& pos, const Tensor& kcache, const Tensor& vcache) {
    need_cuda(qkv_in);
    if (qkv_in.dim() != 4 || qkv_in.size(1) != 3 || qkv_in.size(3) % 2 != 0) value_error("expected [B, 3, H, D] with even D, got " + shape_of(qkv_in));
    const int64_t b = qkv_in.size(0), h = qkv_in.size(2), d = qkv_in.size(3);
    OnDevice on(qkv_in);
    const Tensor qkv = qkv_in.contiguous();
    // complex64 [D/2] or float32 (cos, sin) pairs: the same bytes
    const bool cplx = cis_in.scalar_type() == at::kComplexFloat;
    if ((!cplx && cis_in.scalar_type() != at::kFloat) || cis_in.numel() * (cplx ? 2 : 1) != d || !cis_in.is_contiguous())
        value_error("cis must hold " + std::to_string(d / 2) + " contiguous (cos, sin) float32 pairs");
    if (pos.scalar_type() != at::kLong || pos.numel() != 1 || pos.device() != qkv.device())
        value_error("pos must be an int64 tensor with one element on the activations' device");
    if (kcache.dim() != 4) value_error("caches must be 4-D, got " + shape_of(kcache));
    const int64_t max_len = kcache.size(2);
    for (const Tensor* c : {&kcache, &vcache})
        if (c->dim() != 4 || c->size(0) != b || c->size(1) != h || c->size(2) != max_len || c->size(3) != d || c->scalar_type() != qkv.scalar_type() ||
            !c->is_contiguous() || c->device() != qkv.device())
            value_error(std::string("caches must be contiguous ") + c10::toString(qkv.scalar_type()) + " [" + std::to_string(b) + ", " + std::to_string(h) +
                        ", max_len, " + std::to_string(d) + "] on " + qkv.device().str());
    Tensor q = empty_on(qkv, {b, h, 1, d}, qkv.scalar_type());
    check(bi8_rope_cache_append(qkv.data_ptr(), dtype_code(qkv.scalar_type()), static_cast<const float*>(cis_in.data_ptr()),
                                static_cast<const long long*>(pos.data_ptr()), q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(), b, h, d, max_len, on.raw()),
          "bi8_rope_cache_append");
    return q;
}

// ---- weights and key/value caches in 4-bit blocks ---------------------------------------------------------------------------
// These have no derivatives: a tensor that wants a gradient, or brings a tangent, would lose it silently.
void no_gradient(const Tensor& t, const char* what) {
    if (!t.defined()) return;
    if (at::GradMode::is_enabled() && t.requires_grad())
        throw PyFail{PyExc_RuntimeError, std::string(what) + " has no backward pass: call it under torch.no_grad() or on detached tensors"};
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        throw PyFail{PyExc_RuntimeError, std::string(what) + " has no forward-mode derivative: call it on tensors without tangents"};
}
int dtype_code16(at::ScalarType t, const char* what) {
    if (t != at::kBFloat16 && t != at::kHalf) value_error(std::string(what) + " must be bfloat16 or float16, got " + c10::toString(t));
    return dtype_code(t);
}
void same_device(const Tensor& t, const Tensor& like, const char* what) {
    if (t.defined() && t.device() != like.device()) value_error(std::string(what) + " must be on " + like.device().str() + ", got " + t.device().str());
}
void check_block4(int64_t block) {
    if (block != 32 && block != 64 && block != 128) value_error("4-bit blocks have 32, 64 or 128 values, got " + std::to_string(block));
}
using Sizes = c10::SmallVector<int64_t, 6>;
Sizes with_last(const Tensor& t, int64_t last) {
    Sizes s(t.sizes().begin(), t.sizes().end());
    s.back() = last;
    return s;
}

Quantized quantize_int4(const Tensor& x, int64_t block) {
    need_cuda(x);
    no_gradient(x, "quantize_block_int4");
    if (x.dim() == 0) value_error("expected a tensor with a feature dimension, got a scalar");
    const int code = dtype_code16(x.scalar_type(), "values");
    check_block4(block);
    OnDevice on(x);
    const int64_t k = x.size(-1);
    Quantized r{empty_on(x, with_last(x, ceil_div(k, 2)), at::kByte), empty_on(x, with_last(x, ceil_div(k, block)), x.scalar_type())};
    if (x.numel() == 0) return r;
    const Mat m = mat_rows(x);
    check(bi8_quantize_int4(m.ptr, code, m.ld, r.q.mutable_data_ptr<uint8_t>(), ceil_div(k, 2), r.s.data_ptr(), m.rows, k, (int)block, on.raw()),
          "bi8_quantize_int4");
    return r;
}

// scales [..., blocks] of codes [..., bytes]
void check_scales4(const Tensor& state, const Tensor& codes, int64_t blocks, int64_t block) {
    const Sizes want = with_last(codes, blocks);
    if (state.sizes() != at::IntArrayRef(want))
        value_error("state must have " + std::to_string(blocks) + " scales per row for block " + std::to_string(block) + ", got " + shape_of(state) +
                    " for codes " + shape_of(codes));
    same_device(state, codes, "state");
}

Tensor dequantize_int4(const Tensor& codes, const Tensor& state, int64_t block, int64_t features, at::ScalarType out_type) {
    need_cuda(codes);
    no_gradient(state, "dequantize_block_int4");
    if (codes.dim() == 0 || codes.scalar_type() != at::kByte) value_error(std::string("codes must be uint8 with a feature dimension, got ") + c10::toString(codes.scalar_type()));
    const int code = dtype_code16(state.scalar_type(), "state");
    check_block4(block);
    const int64_t k = features < 0 ? 2 * codes.size(-1) : features;
    if (ceil_div(k, 2) != codes.size(-1)) value_error(std::to_string(k) + " features do not have " + std::to_string(codes.size(-1)) + " bytes of codes");
    check_scales4(state, codes, ceil_div(k, block), block);
    OnDevice on(codes);
    Tensor out = empty_on(codes, with_last(codes, k), out_type);
    if (out.numel() == 0) return out;
    const Mat m = mat_rows(codes);
    const Tensor s = state.contiguous();
    check(bi8_dequantize_int4(static_cast<const uint8_t*>(m.ptr), m.ld, s.data_ptr(), code, out.data_ptr(), dtype_code(out_type), m.rows, k, (int)block, on.raw()),
          "bi8_dequantize_int4");
    return out;
}

Tensor matmul_int4(const Tensor& x_in, const Tensor& codes, const Tensor& state, const Tensor& bias_in, const Tensor& residual, int64_t block,
                   at::ScalarType out_type) {
    need_cuda(x_in);
    for (const Tensor* t : {&x_in, &state, &bias_in, &residual}) no_gradient(*t, "int4_matmul");
    if (x_in.dim() == 0) value_error("expected a tensor with a feature dimension, got a scalar");
    const int code = dtype_code16(x_in.scalar_type(), "activations");
    check_block4(block);
    const int64_t k = x_in.size(-1);
    if (codes.dim() != 2 || codes.scalar_type() != at::kByte || codes.size(1) != ceil_div(k, 2))
        value_error("codes must be uint8 [N, " + std::to_string(ceil_div(k, 2)) + "] for " + std::to_string(k) + " features, got " +
                    c10::toString(codes.scalar_type()) + " " + shape_of(codes));
    same_device(codes, x_in, "codes");
    check_scales4(state, codes, ceil_div(k, block), block);
    if (state.scalar_type() != x_in.scalar_type())
        value_error(std::string("activations and scales must have one type, got ") + c10::toString(x_in.scalar_type()) + " and " + c10::toString(state.scalar_type()));
    same_device(bias_in, x_in, "bias");
    OnDevice on(x_in);
    const int64_t n = codes.size(0), m = k ? x_in.numel() / k : c10::multiply_integers(x_in.sizes().begin(), x_in.sizes().end() - 1);
    const Bias bias(bias_in, n);
    Tensor out = empty_on(x_in, with_last(x_in, n), out_type);
    Mat res;
    if (residual.defined()) {
        if (residual.sizes() != out.sizes() || residual.scalar_type() != out_type)
            value_error(std::string("residual must be ") + c10::toString(out_type) + " " + shape_of(out) + ", got " + c10::toString(residual.scalar_type()) + " " +
                        shape_of(residual));
        same_device(residual, x_in, "residual");
        if (out.numel() > 0) res = mat_rows(residual);
    }
    if (out.numel() == 0) return out;
    const Mat x = k ? mat_rows(x_in) : Mat{}, w = mat2d(codes);
    const Tensor s = state.contiguous();
    check(bi8_matmul_int4(x.ptr, code, std::max(x.ld, k), static_cast<const uint8_t*>(w.ptr), w.ld, s.data_ptr(), bias.ptr, bias.code, res.ptr, res.ld,
                          out.data_ptr(), n, dtype_code(out_type), m, n, k, (int)block, on.raw()),
          "bi8_matmul_int4");
    return out;
}

// Whether heads, sequences, or keys and values of a cache [B, H, rows, width] with dense rows share memory.  Nested steps and tensors that lie
// apart, as nearly every cache has them, are told by a few comparisons; anything else (keys and values interleaved in one tensor, steps
// that interlock) by all of its parts in order.
bool parts_overlap(const Tensor& k, const Tensor& v) {
    struct Part {
        uintptr_t begin, end;
    };
    Part whole[2];
    bool nested = true;
    for (const Tensor* t : {&k, &v}) {
        if (t->numel() == 0) return false;
        const int64_t part = t->size(2) * t->size(3);
        int64_t n[2] = {t->size(0), t->size(1)}, step[2] = {t->stride(0), t->stride(1)};
        for (int i = 0; i < 2; ++i)
            if (n[i] == 1) step[i] = 0;
        if (step[0] > step[1]) std::swap(n[0], n[1]), std::swap(step[0], step[1]);
        const int64_t inner = (n[0] - 1) * step[0] + part;
        nested = nested && (n[0] == 1 || step[0] >= part) && (n[1] == 1 || step[1] >= inner);
        const uintptr_t at = reinterpret_cast<uintptr_t>(t->data_ptr());
        whole[t == &v] = {at, at + (uintptr_t)(((n[1] - 1) * step[1] + inner) * t->element_size())};
    }
    if (nested && (whole[0].end <= whole[1].begin || whole[1].end <= whole[0].begin)) return false;
    std::vector<Part> parts;
    for (const Tensor* t : {&k, &v})
        for (int64_t i = 0; i < t->size(0); ++i)
            for (int64_t j = 0; j < t->size(1); ++j) {
                const uintptr_t at = reinterpret_cast<uintptr_t>(t->data_ptr()) + (uintptr_t)((i * t->stride(0) + j * t->stride(1)) * t->element_size());
                parts.push_back({at, at + (uintptr_t)(t->size(2) * t->size(3) * t->element_size())});
            }
    std::sort(parts.begin(), parts.end(), [](const Part& a, const Part& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < parts.size(); ++i)
        if (parts[i].begin < parts[i - 1].end) return true;
    return false;
}

// The cache's tensors as the library takes them.  `written`: its parts must not share memory.
bi8_int4_cache cache4(const Tensor& k, const Tensor& k_state, const Tensor& v, const Tensor& v_state, const Tensor& like, int64_t b, int64_t d, bool written) {
    if (k.dim() != 4) value_error("cache codes must be 4-D, got " + shape_of(k));
    const int64_t h = k.size(1), rows = k.size(2);
    int64_t steps[8];
    int at = 0;
    for (const Tensor* t : {&k, &v, &k_state, &v_state}) {
        const bool codes = t == &k || t == &v;
        const int64_t width = codes ? d / 2 : d / 64;
        const at::ScalarType type = codes ? at::kByte : like.scalar_type();
        const bool dense = t->dim() == 4 && (width <= 1 || t->stride(3) == 1) && (rows <= 1 || t->stride(2) == width);
        if (t->dim() != 4 || t->size(0) != b || t->size(1) != h || t->size(2) != rows || t->size(3) != width || t->scalar_type() != type || !dense ||
            t->device() != like.device())
            value_error(std::string("cache ") + (codes ? "codes" : "scales") + " must be " + c10::toString(type) + " [" + std::to_string(b) + ", " +
                        std::to_string(h) + ", " + std::to_string(rows) + ", " + std::to_string(width) + "] with dense rows on " + like.device().str() + ", got " +
                        c10::toString(t->scalar_type()) + " " + shape_of(*t));
        for (int dim = 0; dim < 2; ++dim) steps[at++] = t->size(dim) > 1 ? t->stride(dim) : 0;
    }
    if (written && (parts_overlap(k, v) || parts_overlap(k_state, v_state)))
        value_error("a cache that is written must not share memory between sequences, heads, or keys and values");
    return {static_cast<uint8_t*>(k.data_ptr()), static_cast<uint8_t*>(v.data_ptr()), k_state.data_ptr(), v_state.data_ptr(),
            steps[0], steps[1], steps[2], steps[3], steps[4], steps[5], steps[6], steps[7], rows};
}

// One int64 for all sequences or one for each: its address and step.
struct PerSequence {
    const long long* ptr = nullptr;
    int64_t step = 0;
    PerSequence(const Tensor& t, const Tensor& like, int64_t b, const char* what) {
        if (!t.defined()) return;
        if (t.scalar_type() != at::kLong || t.device() != like.device() || !(t.numel() == 1 || (t.dim() == 1 && t.size(0) == b)))
            value_error(std::string(what) + " must be an int64 tensor with one element or " + std::to_string(b) + " on the activations' device");
        ptr = static_cast<const long long*>(t.data_ptr());
        step = t.numel() == 1 ? 0 : t.stride(0);
    }
};

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

Tensor rope_cache_append_int4(const Tensor& qkv_in, const Tensor& cis_in, const Tensor& pos, const Tensor& k, const Tensor& k_state, const Tensor& v,
                              const Tensor& v_state) {
    need_cuda(qkv_in);
    for (const Tensor* t : {&qkv_in, &cis_in, &k_state, &v_state}) no_gradient(*t, "rope_cache_append_int4");
    if (qkv_in.dim() != 4) value_error("expected [B, T, Hq + 2 Hkv, D], got " + shape_of(qkv_in));
    const int code = dtype_code16(qkv_in.scalar_type(), "activations");
    const int64_t b = qkv_in.size(0), t = qkv_in.size(1), d = qkv_in.size(3);
    if (d != 64 && d != 128 && d != 256) value_error("head size must be 64, 128 or 256, got " + std::to_string(d));
    const bi8_int4_cache cache = cache4(k, k_state, v, v_state, qkv_in, b, d, true);
    const int64_t hkv = k.size(1), hq = qkv_in.size(2) - 2 * hkv;
    if (hkv < 1 || hq < hkv || hq % hkv != 0) value_error(std::to_string(qkv_in.size(2)) + " heads are not Hq + 2 * " + std::to_string(hkv) + " with Hq a multiple of " + std::to_string(hkv));
    OnDevice on(qkv_in);
    Tensor qkv = qkv_in.contiguous();
    if (qkv.numel() > 0 && !aligned16(qkv)) qkv = qkv.clone();
    // complex64 [rows, D/2] or float32 (cos, sin) pairs: the same bytes
    const bool cplx = cis_in.scalar_type() == at::kComplexFloat;
    if ((!cplx && cis_in.scalar_type() != at::kFloat) || cis_in.dim() != (cplx ? 2 : 3) || cis_in.size(1) != d / 2 || (!cplx && cis_in.size(2) != 2) ||
        cis_in.device() != qkv.device())
        value_error("cis must hold [rows, " + std::to_string(d / 2) + "] (cos, sin) float32 pairs on the activations' device");
    Tensor cis = cis_in.is_conj() ? cis_in.resolve_conj().contiguous() : cis_in.contiguous();
    if (cis.numel() > 0 && !aligned16(cis)) cis = cis.clone();
    const PerSequence p(pos, qkv, b, "pos");
    Tensor q = empty_on(qkv, {b, hq, t, d}, qkv.scalar_type());
    check(bi8_rope_cache_append_int4(qkv.data_ptr(), code, static_cast<const float*>(cis.data_ptr()), cis.size(0), p.ptr, p.step, q.data_ptr(), &cache, b, t, hq,
                                     hkv, d, on.raw()),
          "bi8_rope_cache_append_int4");
    return q;
}

Tensor attention_int4(const Tensor& q_in, const Tensor& k, const Tensor& k_state, const Tensor& v, const Tensor& v_state, const Tensor& lengths,
                      const Tensor& starts, double scale) {
    need_cuda(q_in);
    for (const Tensor* t : {&q_in, &k_state, &v_state}) no_gradient(*t, "attention_int4_cache");
    if (q_in.dim() != 4) value_error("expected queries [B, Hq, T, D], got " + shape_of(q_in));
    const int code = dtype_code16(q_in.scalar_type(), "queries");
    const int64_t b = q_in.size(0), hq = q_in.size(1), t = q_in.size(2), d = q_in.size(3);
    if (d != 64 && d != 128 && d != 256) value_error("head size must be 64, 128 or 256, got " + std::to_string(d));
    const bi8_int4_cache cache = cache4(k, k_state, v, v_state, q_in, b, d, false);
    const int64_t hkv = k.size(1);
    if (hkv < 1 || hq < 1 || hq % hkv != 0) value_error(std::to_string(hq) + " query heads do not divide over " + std::to_string(hkv) + " cache heads");
    OnDevice on(q_in);
    const PerSequence len(lengths, q_in, b, "lengths"), start(starts, q_in, b, "starts");
    if (!(std::abs(scale) <= 2e38)) value_error("scale must be a number of at most 2e38, got " + std::to_string(scale));
    Tensor out = empty_on(q_in, {b, hq, t, d}, q_in.scalar_type());
    if (out.numel() == 0) return out;
    Tensor q = q_in;
    int64_t steps[3];
    bool ok = q.stride(3) == 1 && aligned16(q);
    for (int i = 0; i < 3; ++i) {
        steps[i] = q.size(i) > 1 ? q.stride(i) : 0;
        ok = ok && steps[i] % 8 == 0;
    }
    if (!ok) {
        q = q.clone(at::MemoryFormat::Contiguous);
        steps[0] = hq * t * d, steps[1] = t * d, steps[2] = d;
    }
    const size_t bytes = bi8_attention_int4_workspace_bytes(b, t, hq, hkv, d, cache.max_len);
    const Tensor ws = scratch(q, (int64_t)bytes);
    check(bi8_attention_int4(q.data_ptr(), code, steps[0], steps[1], steps[2], &cache, len.ptr, len.step, start.ptr, start.step, (float)scale, out.data_ptr(), b, t,
                             hq, hkv, d, ws.defined() ? ws.data_ptr() : nullptr, bytes, on.raw()),
          "bi8_attention_int4");
    return out;
}

// ---- rotary positions and a paged key/value cache -----------------------------------------------------------------------------
// A table of angles: complex64 [rows, R/2] or float32 [rows, R/2, 2] (cos, sin), the same bytes.  Dense and on a 16-byte boundary.
struct Angles {
    Tensor owner;
    const float* ptr = nullptr;
    int64_t rows = 0, features = 0;
    Angles(const Tensor& cis, const Tensor& like) {
        const bool cplx = cis.scalar_type() == at::kComplexFloat;
        if ((!cplx && cis.scalar_type() != at::kFloat) || cis.dim() != (cplx ? 2 : 3) || (!cplx && cis.size(2) != 2))
            value_error(std::string("cis must hold [rows, pairs] (cos, sin) float32 pairs, got ") + c10::toString(cis.scalar_type()) + " " + shape_of(cis));
        same_device(cis, like, "cis");
        owner = cis.resolve_conj().resolve_neg().contiguous();
        if (owner.numel() > 0 && !aligned16(owner)) owner = owner.clone();
        ptr = static_cast<const float*>(owner.data_ptr());
        rows = cis.size(0);
        features = 2 * cis.size(1);
    }
};

Tensor rope(const Tensor& x, const Tensor& cis, const Tensor& positions, int64_t layout, bool conjugate);

// The rotation is linear and its transpose is the rotation the other way, so its gradient can be differentiated again.
struct RopeBackward : public Node {
    SavedVariable cis, positions;
    int64_t layout = 0;
    bool conjugate = false;
    std::string name() const override { return "ropeBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        cis.reset_data();
        positions.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        variable_list out(1);
        if (!grads[0].defined() || !task_should_compute_output(0)) return out;
        Tensor table, at;
        {
            std::lock_guard<std::mutex> lock(mutex_);
            table = cis.unpack(getptr());
            at = positions.unpack(getptr());
        }
        try {
            out[0] = rope(grads[0], table, at, layout, conjugate);
        } catch (const PyFail& e) {
            throw std::runtime_error(e.text);
        }
        return out;
    }
};

Tensor rope_values(const Tensor& x_in, const Tensor& cis, const Tensor& positions, int64_t layout, bool conjugate) {
    at::AutoDispatchBelowADInplaceOrView below_autograd;
    OnDevice on(x_in);
    const Angles angles(cis, x_in);
    const Tensor plain = x_in.resolve_neg(), x = plain.size(-1) > 1 && plain.stride(-1) != 1 ? plain.contiguous() : plain;
    const int lead = (int)x.dim() - 3;
    const int64_t b = lead ? x.size(0) : 1, t = x.size(lead), h = x.size(lead + 1), d = x.size(lead + 2);
    const int64_t pos_tok = positions.defined() && t > 1 ? positions.stride(-1) : 0;
    const int64_t pos_batch = positions.defined() && positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    Tensor out = empty_on(x, x.sizes(), x.scalar_type());
    check(bi8_rope(x.data_ptr(), dtype_code(x.scalar_type()), lead && b > 1 ? x.stride(0) : 0, t > 1 ? x.stride(lead) : 0, h > 1 ? x.stride(lead + 1) : 0, angles.ptr,
                   angles.rows, angles.features, positions.defined() ? static_cast<const long long*>(positions.data_ptr()) : nullptr, pos_batch, pos_tok,
                   out.data_ptr(), b, t, h, d, (int)layout, conjugate, on.raw()),
          "bi8_rope");
    return out;
}

Tensor rope(const Tensor& x, const Tensor& cis, const Tensor& positions, int64_t layout, bool conjugate) {
    need_cuda(x);
    if (x.dim() != 3 && x.dim() != 4) value_error("expected [B, T, H, D] or [T, H, D], got " + shape_of(x));
    (void)dtype_code(x.scalar_type());
    const int64_t pairs = cis.dim() > 1 ? cis.size(1) : 0;
    if (pairs < 1 || 2 * pairs > x.size(-1))
        value_error("a table of " + std::to_string(pairs) + " pairs does not fit heads of " + std::to_string(x.size(-1)) + " features");
    if (at::GradMode::is_enabled() && cis.requires_grad())
        throw PyFail{PyExc_RuntimeError, "rope has no backward pass for its table: call it with a detached one"};
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && (x._fw_grad(0).defined() || cis._fw_grad(0).defined()))
        throw PyFail{PyExc_RuntimeError, "rope has no forward-mode derivative: call it on tensors without tangents"};
    if (positions.defined()) {
        const int64_t t = x.size(-3);
        const bool fits = positions.dim() == 1 ? positions.size(0) == t
                                               : positions.dim() == 2 && x.dim() == 4 && positions.size(1) == t && (positions.size(0) == x.size(0) || positions.size(0) == 1);
        if (positions.scalar_type() != at::kLong || !fits)
            value_error("positions must be int64 [T] or [B, T] for activations " + shape_of(x) + ", got " + c10::toString(positions.scalar_type()) + " " +
                        shape_of(positions));
        same_device(positions, x, "positions");
    }
    Tensor out = rope_values(x, cis, positions, layout, conjugate);
    if (at::GradMode::is_enabled() && x.requires_grad()) {
        auto node = std::shared_ptr<RopeBackward>(new RopeBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->cis = SavedVariable(cis, false);
        node->positions = SavedVariable(positions, false);
        node->layout = layout;
        node->conjugate = !conjugate;
        torch::autograd::set_history(out, node);
    }
    return out;
}

// Whether no two values of k and v [pages, heads, rows, D], features dense, share memory, as far as nested steps show it: every step reaches past
// what is inside it, and keys and values lie apart, or have the same steps and their distance is one more such step.
bool values_apart(const Tensor& k, const Tensor& v) {
    if (k.numel() == 0 || v.numel() == 0) return true;
    auto nested = [](const Tensor& t, int64_t other, int64_t* extent) {
        std::pair<int64_t, int64_t> dims[4];                 // step, count
        int count = 0;
        for (int i = 0; i < 3; ++i)
            if (t.size(i) > 1) dims[count++] = {t.stride(i), t.size(i)};
        if (other > 0) dims[count++] = {other, 2};
        std::sort(dims, dims + count);
        int64_t reach = t.size(3);
        for (int i = 0; i < count; ++i) {
            if (dims[i].first < reach) return false;
            reach += dims[i].first * (dims[i].second - 1);
        }
        *extent = reach;
        return true;
    };
    int64_t k_reach = 0, v_reach = 0;
    if (!nested(k, 0, &k_reach) || !nested(v, 0, &v_reach)) return false;
    const int64_t size = k.element_size(), at = (int64_t)reinterpret_cast<uintptr_t>(k.data_ptr()), bt = (int64_t)reinterpret_cast<uintptr_t>(v.data_ptr());
    if (at + k_reach * size <= bt || bt + v_reach * size <= at) return true;
    for (int i = 0; i < 3; ++i)
        if (k.size(i) > 1 && k.stride(i) != v.stride(i)) return false;
    const int64_t apart = at < bt ? bt - at : at - bt;
    return apart > 0 && apart % size == 0 && nested(k, apart / size, &k_reach);
}

bi8_paged_cache paged_cache(const Tensor& k, const Tensor& v, const Tensor& like, int64_t d) {
    if (k.dim() != 4) value_error("cache pages must be 4-D, got " + shape_of(k));
    for (const Tensor* t : {&k, &v})
        if (t->dim() != 4 || t->sizes() != k.sizes() || t->size(3) != d || t->scalar_type() != like.scalar_type() || t->device() != like.device() ||
            (d > 1 && t->stride(3) != 1))
            value_error(std::string("cache pages must be ") + c10::toString(like.scalar_type()) + " [pages, heads, rows, " + std::to_string(d) +
                        "] with dense features on " + like.device().str() + ", keys and values alike, got " + c10::toString(t->scalar_type()) + " " + shape_of(*t));
    if (k.is_neg() || v.is_neg()) value_error("a cache must hold its values as they are, not negated ones of another tensor");
    if (k.size(1) < 1) value_error("a cache needs a head, got " + shape_of(k));
    if (k.size(2) < 1 || k.size(2) % 16 != 0) value_error("pages must have a multiple of 16 rows, got " + std::to_string(k.size(2)));
    int64_t steps[6];
    for (int i = 0; i < 6; ++i) {
        const Tensor& t = i < 3 ? k : v;
        steps[i] = t.size(i % 3) > 1 ? t.stride(i % 3) : 0;
        if (steps[i] % 8 != 0) value_error("steps of a cache must be multiples of 8 values");
    }
    if (k.numel() > 0 && (!aligned16(k) || !aligned16(v))) value_error("a cache must begin on a 16-byte boundary");
    if (!values_apart(k, v)) value_error("pages, heads, rows, keys and values of a cache must not share memory");
    return {k.data_ptr(), v.data_ptr(), steps[0], steps[1], steps[2], steps[3], steps[4], steps[5], k.size(0), k.size(1), k.size(2), d};
}

// The sequences of a batch of n tokens.  The struct's tensors live as long as this does.
struct Batch {
    Tensor pages_owner, cu_owner;
    bi8_sequences s{};
    Batch(const Tensor& pages, const Tensor& lengths, const Tensor& cu_tokens, const Tensor& starts, const Tensor& like, int64_t n) {
        if (pages.dim() != 2 || pages.scalar_type() != at::kInt)
            value_error(std::string("pages must be int32 [B, width], got ") + c10::toString(pages.scalar_type()) + " " + shape_of(pages));
        same_device(pages, like, "pages");
        pages_owner = pages.size(1) > 1 && pages.stride(1) != 1 ? pages.contiguous() : pages;
        const int64_t b = pages.size(0);
        const PerSequence len(lengths, like, b, "lengths"), start(starts, like, b, "starts");
        if (cu_tokens.defined()) {
            if (cu_tokens.scalar_type() != at::kLong || cu_tokens.dim() != 1 || cu_tokens.size(0) != b + 1)
                value_error("cu_tokens must be int64 [" + std::to_string(b + 1) + "], got " + c10::toString(cu_tokens.scalar_type()) + " " + shape_of(cu_tokens));
            same_device(cu_tokens, like, "cu_tokens");
            cu_owner = cu_tokens.contiguous();
        } else if (b == 0 ? n != 0 : n % b != 0) {
            value_error(std::to_string(n) + " tokens do not divide over " + std::to_string(b) + " sequences: give cu_tokens");
        }
        if (b == 0 && n != 0) value_error("tokens without a sequence");
        s.lengths = len.ptr;
        s.lengths_step = len.step;
        s.starts = start.ptr;
        s.starts_step = start.step;
        s.cu_tokens = cu_owner.defined() ? static_cast<const long long*>(cu_owner.data_ptr()) : nullptr;
        s.page_table = static_cast<const int*>(pages_owner.data_ptr());
        s.table_step = b > 1 ? pages_owner.stride(0) : 0;
        s.width = pages.size(1);
        s.B = b;
        s.N = n;
    }
};

// [N, heads, D] with dense features, steps that are multiples of 8 and a 16-byte boundary: the tensor itself or a copy
Tensor packed_tokens(const Tensor& given, int64_t (&steps)[2]) {
    const Tensor t = given.resolve_neg();
    bool ok = t.stride(2) == 1 && aligned16(t);
    for (int i = 0; i < 2; ++i) {
        steps[i] = t.size(i) > 1 ? t.stride(i) : 0;
        ok = ok && steps[i] % 8 == 0;
    }
    if (ok) return t;
    steps[0] = t.size(1) * t.size(2), steps[1] = t.size(2);
    return t.clone(at::MemoryFormat::Contiguous);
}

int64_t head_size(const Tensor& t) {
    const int64_t d = t.size(2);
    if (d != 64 && d != 128 && d != 256) value_error("head size must be 64, 128 or 256, got " + std::to_string(d));
    return d;
}

Tensor rope_cache_append_paged(const Tensor& qkv_in, const Tensor& cis_in, const Tensor& k, const Tensor& v, const Tensor& pages, const Tensor& lengths,
                               const Tensor& cu_tokens, int64_t layout) {
    need_cuda(qkv_in);
    for (const Tensor* t : {&qkv_in, &cis_in, &k, &v}) no_gradient(*t, "rope_cache_append_paged");
    if (qkv_in.dim() != 3) value_error("expected [N, Hq + 2 Hkv, D], got " + shape_of(qkv_in));
    const int code = dtype_code16(qkv_in.scalar_type(), "activations");
    const int64_t n = qkv_in.size(0), d = head_size(qkv_in);
    const bi8_paged_cache cache = paged_cache(k, v, qkv_in, d);
    const int64_t hkv = k.size(1), hq = qkv_in.size(1) - 2 * hkv;
    if (hq < hkv || hq % hkv != 0)
        value_error(std::to_string(qkv_in.size(1)) + " heads are not Hq + 2 * " + std::to_string(hkv) + " with Hq a multiple of " + std::to_string(hkv));
    OnDevice on(qkv_in);
    const Angles angles(cis_in, qkv_in);
    if (angles.features < 16 || angles.features > d || angles.features % 16 != 0)
        value_error("rotated features must be a multiple of 16 of the " + std::to_string(d) + ", got " + std::to_string(angles.features));
    const Batch batch(pages, lengths, cu_tokens, Tensor(), qkv_in, n);
    Tensor q = empty_on(qkv_in, {n, hq, d}, qkv_in.scalar_type());
    if (q.numel() == 0) return q;
    int64_t steps[2];
    const Tensor qkv = packed_tokens(qkv_in, steps);
    check(bi8_rope_cache_append_paged(qkv.data_ptr(), code, steps[0], steps[1], angles.ptr, angles.rows, angles.features, (int)layout, q.data_ptr(), &cache, &batch.s,
                                      hq, on.raw()),
          "bi8_rope_cache_append_paged");
    return q;
}

Tensor attention_paged(const Tensor& q_in, const Tensor& k, const Tensor& v, const Tensor& pages, const Tensor& lengths, const Tensor& cu_tokens,
                       const Tensor& starts, double scale) {
    need_cuda(q_in);
    for (const Tensor* t : {&q_in, &k, &v}) no_gradient(*t, "attention_paged_cache");
    if (q_in.dim() != 3) value_error("expected queries [N, Hq, D], got " + shape_of(q_in));
    const int code = dtype_code16(q_in.scalar_type(), "queries");
    const int64_t n = q_in.size(0), hq = q_in.size(1), d = head_size(q_in);
    const bi8_paged_cache cache = paged_cache(k, v, q_in, d);
    const int64_t hkv = k.size(1);
    if (hq < 1 || hq % hkv != 0) value_error(std::to_string(hq) + " query heads do not divide over " + std::to_string(hkv) + " cache heads");
    if (!(std::abs(scale) <= 2e38)) value_error("scale must be a number of at most 2e38, got " + std::to_string(scale));
    OnDevice on(q_in);
    const Batch batch(pages, lengths, cu_tokens, starts, q_in, n);
    Tensor out = empty_on(q_in, {n, hq, d}, q_in.scalar_type());
    if (out.numel() == 0) return out;
    int64_t steps[2];
    const Tensor q = packed_tokens(q_in, steps);
    const size_t bytes = bi8_attention_paged_workspace_bytes(batch.s.B, n, hq, hkv, d, batch.s.width * cache.page_rows, cu_tokens.defined());
    const Tensor ws = scratch(q, (int64_t)bytes);
    check(bi8_attention_paged(q.data_ptr(), code, steps[0], steps[1], &cache, &batch.s, (float)scale, out.data_ptr(), hq, ws.defined() ? ws.data_ptr() : nullptr, bytes,
                              on.raw()),
          "bi8_attention_paged");
    return out;
}

// ---- bindings -----------------------------------------------------------------------------------------------------------
struct Args {
    PyObject* const* a;
    Py_ssize_t n;
    const Tensor& tensor(int i) const {
        if (!THPVariable_Check(a[i])) throw PyFail{PyExc_TypeError, std::string("expected a tensor, got ") + Py_TYPE(a[i])->tp_name};
        return THPVariable_Unpack(a[i]);
    }
    Tensor optional(int i) const { return a[i] == Py_None ? Tensor() : tensor(i); }
    int64_t integer(int i) const {
        const long long v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        return v;
    }
    double number(int i) const {
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) throw python_error();
        return v;
    }
    at::ScalarType dtype(int i) const {
        if (!THPDtype_Check(a[i])) throw PyFail{PyExc_TypeError, "expected a torch.dtype"};
        const at::ScalarType t = reinterpret_cast<THPDtype*>(a[i])->scalar_type;
        (void)dtype_code(t);
        return t;
    }
    int64_t block(int i) const {
        const int64_t b = integer(i);
        if (b < 1 || b > 0x7fffffff) value_error("block size must be positive, got " + std::to_string(b));
        return b;
    }
};

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const Quantized& r) {
    PyObject* t = PyTuple_New(2);
    PyTuple_SET_ITEM(t, 0, wrap(r.q));
    PyTuple_SET_ITEM(t, 1, wrap(r.s));
    return t;
}
PyObject* wrap(const Dual& d) {
    PyObject* t = PyTuple_New(4);
    PyTuple_SET_ITEM(t, 0, wrap(d.row.q));
    PyTuple_SET_ITEM(t, 1, wrap(d.row.s));
    PyTuple_SET_ITEM(t, 2, wrap(d.col.q));
    PyTuple_SET_ITEM(t, 3, wrap(d.col.s));
    return t;
}

// Runs `body` without the interpreter lock (kernel launches can block when the launch queue is full) and turns its exceptions into Python's.
template <typename Body>
PyObject* call(const char* name, const Args& args, Py_ssize_t want, Body body, bool records_history = false) {
    try {
        if (args.n != want) throw PyFail{PyExc_TypeError, std::string(name) + " takes " + std::to_string(want) + " arguments, got " + std::to_string(args.n)};
        auto result = [&] {
            auto work = body(args);            // reads the arguments with the lock held
            pybind11::gil_scoped_release no_gil;
            std::optional<at::AutoDispatchBelowADInplaceOrView> below_autograd;
            if (!records_history) below_autograd.emplace();
            return work();
        }();
        return wrap(result);
    } catch (const PyFail& e) {
        PyErr_SetString(e.type, e.text.c_str());
        return nullptr;
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

#define BI8_METHOD(name) PyObject* name##_py(PyObject*, PyObject* const* a, Py_ssize_t n)

BI8_METHOD(quantize_rowwise) {   // x, block, whether the result is only a GEMM operand
    return call("quantize_rowwise", {a, n}, 3, [](const Args& g) {
        return [x = g.tensor(0), b = g.block(1), operand = g.integer(2) != 0] { return quantize_rowwise(x, b, operand); };
    });
}
BI8_METHOD(quantize_colwise) {   // x, block, whether the result is only a GEMM operand
    return call("quantize_colwise", {a, n}, 3, [](const Args& g) {
        return [x = g.tensor(0), b = g.block(1), operand = g.integer(2) != 0] { return quantize_colwise(x, b, operand); };
    });
}
BI8_METHOD(quantize_dual) {
    return call("quantize_dual", {a, n}, 2, [](const Args& g) { return [x = g.tensor(0), b = g.block(1)] { return quantize_dual(x, b); }; });
}
BI8_METHOD(quantize_pre) {       // op, x, x2, weight, eps, block
    return call("quantize_pre", {a, n}, 6, [](const Args& g) {
        return [op = (int)g.integer(0), x = g.tensor(1), x2 = g.optional(2), w = g.optional(3), eps = g.number(4), b = g.block(5)] {
            return quantize_pre(op, x, x2, w, eps, b);
        };
    });
}
BI8_METHOD(dequantize) {         // q, state, block, dtype
    return call("dequantize", {a, n}, 4, [](const Args& g) {
        return [q = g.tensor(0), s = g.tensor(1), b = g.block(2), t = g.dtype(3)] { return dequantize(q, s, b, t); };
    });
}
BI8_METHOD(gemm) {               // a, b, state_x, state_w, bias, block, dtype, flags
    return call("gemm", {a, n}, 8, [](const Args& g) {
        return [x = g.tensor(0), y = g.tensor(1), sx = g.tensor(2), sw = g.tensor(3), bias = g.optional(4), b = g.block(5), t = g.dtype(6),
                f = (int)g.integer(7)] { return gemm(x, y, sx, sw, bias, b, t, f); };
    });
}
BI8_METHOD(block_partials) {     // a, b, block, flags
    return call("block_partials", {a, n}, 4, [](const Args& g) {
        return [x = g.tensor(0), y = g.tensor(1), b = g.block(2), f = (int)g.integer(3)] { return block_partials(x, y, b, f); };
    });
}
BI8_METHOD(matmul) {             // op, x [M, K], b [K, N], state_w, bias, x2, norm_weight, eps, residual, out, block, dtype, flags
    return call("matmul", {a, n}, 13, [](const Args& g) {
        if (g.tensor(1).dim() != 2) {
            need_cuda(g.tensor(1));
            value_error("expected a 2-D tensor, got " + shape_of(g.tensor(1)));
        }
        return [op = (int)g.integer(0), x = g.tensor(1), w = g.tensor(2), sw = g.tensor(3), bias = g.optional(4), x2 = g.optional(5), nw = g.optional(6),
                eps = g.number(7), res = g.optional(8), out = g.optional(9), b = g.block(10), t = g.dtype(11), f = (int)g.integer(12)] {
            return linear(op, x, w, true, sw, bias, x2, nw, eps, res, out, b, t, f);
        };
    });
}
BI8_METHOD(linear) {             // op, x [..., K], W int8 [N, K], state_w, bias, x2, norm_weight, eps, residual, block, dtype
    return call("linear", {a, n}, 11, [](const Args& g) {
        return [op = (int)g.integer(0), x = g.tensor(1), w = g.tensor(2), sw = g.tensor(3), bias = g.optional(4), x2 = g.optional(5), nw = g.optional(6),
                eps = g.number(7), res = g.optional(8), b = g.block(9), t = g.dtype(10)] {
            return linear(op, x, w, false, sw, bias, x2, nw, eps, res, Tensor(), b, t, 0);
        };
    });
}
BI8_METHOD(train_linear) {       // x [..., K], W [N, K], bias, fuse_dual, cache dict or None: block size and type from the config module
    return call("train_linear", {a, n}, 5, [](const Args& g) {
        PyObject* cache = g.a[4] == Py_None ? nullptr : g.a[4];
        if (cache && !PyDict_Check(cache)) throw PyFail{PyExc_TypeError, "the weight cache must be a dict"};
        return [x = g.tensor(0), w = g.tensor(1), bias = g.optional(2), fuse = PyObject_IsTrue(g.a[3]) == 1, b = config_block(), t = config_dtype(), cache] {
            return train_linear(x, w, bias, b, t, fuse, cache);
        };
    }, true);
}
BI8_METHOD(rope_cache_append) {  // qkv, cis, pos, kcache, vcache
    return call("rope_cache_append", {a, n}, 5, [](const Args& g) {
        return [q = g.tensor(0), c = g.tensor(1), p = g.tensor(2), k = g.tensor(3), v = g.tensor(4)] { return rope_cache_append(q, c, p, k, v); };
    });
}
BI8_METHOD(quantize_int4) {      // x, block
    return call("quantize_int4", {a, n}, 2, [](const Args& g) { return [x = g.tensor(0), b = g.block(1)] { return quantize_int4(x, b); }; });
}
BI8_METHOD(dequantize_int4) {    // codes, state, block, features or -1, dtype
    return call("dequantize_int4", {a, n}, 5, [](const Args& g) {
        return [q = g.tensor(0), s = g.tensor(1), b = g.block(2), k = g.integer(3), t = g.dtype(4)] { return dequantize_int4(q, s, b, k, t); };
    });
}
BI8_METHOD(matmul_int4) {        // x, codes, state, bias, residual, block, dtype
    return call("matmul_int4", {a, n}, 7, [](const Args& g) {
        return [x = g.tensor(0), q = g.tensor(1), s = g.tensor(2), bias = g.optional(3), res = g.optional(4), b = g.block(5), t = g.dtype(6)] {
            return matmul_int4(x, q, s, bias, res, b, t);
        };
    });
}
BI8_METHOD(rope_cache_append_int4) {  // qkv, cis, pos, k, k_state, v, v_state
    return call("rope_cache_append_int4", {a, n}, 7, [](const Args& g) {
        return [x = g.tensor(0), c = g.tensor(1), p = g.tensor(2), k = g.tensor(3), ks = g.tensor(4), v = g.tensor(5), vs = g.tensor(6)] {
            return rope_cache_append_int4(x, c, p, k, ks, v, vs);
        };
    });
}
BI8_METHOD(attention_int4) {     // q, k, k_state, v, v_state, lengths, starts, scale
    return call("attention_int4", {a, n}, 8, [](const Args& g) {
        return [q = g.tensor(0), k = g.tensor(1), ks = g.tensor(2), v = g.tensor(3), vs = g.tensor(4), len = g.tensor(5), start = g.optional(6),
                scale = g.number(7)] { return attention_int4(q, k, ks, v, vs, len, start, scale); };
    });
}
BI8_METHOD(rope) {               // x, cis, positions, layout
    return call("rope", {a, n}, 4, [](const Args& g) {
        return [x = g.tensor(0), c = g.tensor(1), p = g.optional(2), l = g.integer(3)] { return rope(x, c, p, l, false); };
    }, true);
}
BI8_METHOD(rope_cache_append_paged) {  // qkv, cis, k, v, pages, lengths, cu_tokens, layout
    return call("rope_cache_append_paged", {a, n}, 8, [](const Args& g) {
        return [x = g.tensor(0), c = g.tensor(1), k = g.tensor(2), v = g.tensor(3), p = g.tensor(4), len = g.tensor(5), cu = g.optional(6), l = g.integer(7)] {
            return rope_cache_append_paged(x, c, k, v, p, len, cu, l);
        };
    });
}
BI8_METHOD(attention_paged) {    // q, k, v, pages, lengths, cu_tokens, starts, scale
    return call("attention_paged", {a, n}, 8, [](const Args& g) {
        return [q = g.tensor(0), k = g.tensor(1), v = g.tensor(2), p = g.tensor(3), len = g.tensor(4), cu = g.optional(5), start = g.optional(6),
                scale = g.number(7)] { return attention_paged(q, k, v, p, len, cu, start, scale); };
    });
}
BI8_METHOD(bind) {               // the exception class of failed library calls, the configuration module
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "bind takes 2 arguments");
        return nullptr;
    }
    g_error_class = Py_NewRef(a[0]);
    g_config = Py_NewRef(a[1]);
    Py_RETURN_NONE;
}

#define BI8_ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name##_py)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {BI8_ENTRY(quantize_rowwise), BI8_ENTRY(quantize_colwise), BI8_ENTRY(quantize_dual), BI8_ENTRY(quantize_pre),
                         BI8_ENTRY(dequantize), BI8_ENTRY(gemm), BI8_ENTRY(block_partials), BI8_ENTRY(matmul), BI8_ENTRY(linear),
                         BI8_ENTRY(train_linear), BI8_ENTRY(rope_cache_append), BI8_ENTRY(quantize_int4), BI8_ENTRY(dequantize_int4),
                         BI8_ENTRY(matmul_int4), BI8_ENTRY(rope_cache_append_int4), BI8_ENTRY(attention_int4), BI8_ENTRY(rope),
                         BI8_ENTRY(rope_cache_append_paged), BI8_ENTRY(attention_paged), BI8_ENTRY(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "Host path of the blockwise-int8 operations.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
