// spectral._C: the torch.ops.spectral operators, a thin shim over the C ABI
// (include/spectral_b200.h).
//
// The schemas, defaults, argument checks and messages are the reference's
// (csrc/torch/ops.cpp:47-475), so code and tests written against it keep working: the checks
// made here raise RuntimeError (TORCH_CHECK), the C ABI's SPECTRAL_INVALID_ARGUMENT is rethrown
// as std::invalid_argument (ValueError), as the reference's drivers do. Every operator is
// registered for the CUDA dispatch key only, so CPU tensors get the dispatcher's
// NotImplementedError (four also have gradients, through the AutogradCUDA key). A binding checks, makes its input contiguous, allocates the output and
// any workspace with at::empty (torch's caching allocator, stream-ordered), and launches on the
// current stream under a device guard. Nothing here runs on the CPU.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/spectral_b200.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

namespace {

using variable_list_t = std::vector<at::Tensor>;

void check_status(int status)
{
    if (status == SPECTRAL_OK) {
        return;
    }
    const std::string message = spectral_last_error();
    if (status == SPECTRAL_INVALID_ARGUMENT) {
        throw std::invalid_argument(message);
    }
    TORCH_CHECK(false, message);
}

void* stream() { return static_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

const void* cptr(const at::Tensor& t) { return t.const_data_ptr(); }
void* mptr(at::Tensor& t) { return t.numel() == 0 ? nullptr : t.mutable_data_ptr(); }

void check_complex64_cuda(const at::Tensor& t, const char* name)
{
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == at::kComplexFloat, name, " must be complex64, got ",
                t.scalar_type());
}

void check_float32_cuda(const at::Tensor& t)
{
    TORCH_CHECK(t.is_cuda(), "x must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == at::kFloat, "x must be float32, got ", t.scalar_type());
}

struct ImplInfo {
    std::string name;
    int max_n;
    int max_c2c_n;
    int max_real_n;
    bool has_columns;
};

std::string impl_names()
{
    std::string names;
    for (int i = 0; i < spectral_impl_count(); ++i) {
        names += names.empty() ? "" : ", ";
        names += spectral_impl_name(i);
    }
    return names;
}

ImplInfo find_impl(c10::string_view impl_name)
{
    const std::string name(impl_name.data(), impl_name.size());
    TORCH_CHECK(spectral_impl_find(name.c_str()) >= 0, "unknown FFT implementation '", name,
                "' (available: ", impl_names(), ")");
    ImplInfo info{name, 0, 0, 0, false};
    int has_columns = 0;
    check_status(spectral_impl_limits(name.c_str(), &info.max_n, &info.max_c2c_n,
                                      &info.max_real_n, &has_columns, nullptr, nullptr));
    info.has_columns = has_columns != 0;
    return info;
}

int batch_of(const at::Tensor& x, int64_t row, const char* op)
{
    const int64_t batch = x.numel() / row;
    TORCH_CHECK(batch <= INT_MAX, op, ": too many transforms");
    return static_cast<int>(batch);
}

// The library reads and writes every array as 8-byte values; a contiguous float32 view can start
// at an odd element, so such an input is copied to a fresh (aligned) allocation first.
at::Tensor contiguous_aligned(const at::Tensor& x)
{
    at::Tensor c = x.contiguous();
    if ((reinterpret_cast<uintptr_t>(c.const_data_ptr()) & 7u) != 0) {
        c = c.clone(at::MemoryFormat::Contiguous);
    }
    return c;
}

at::Tensor workspace(size_t count, const at::Tensor& like)
{
    return at::empty({static_cast<int64_t>(count)}, like.options().dtype(at::kComplexFloat));
}

void check_real_size(int64_t n, const ImplInfo& impl, const char* op)
{
    TORCH_CHECK(n >= 2 && (n & (n - 1)) == 0, op,
                ": the real transform size must be a power of two of at least 2, got ", n);
    TORCH_CHECK(n <= impl.max_real_n, op, ": ", impl.name, " supports real sizes up to ",
                impl.max_real_n, ", got ", n);
}

at::Tensor scale_cuda(const at::Tensor& x, double alpha)
{
    check_complex64_cuda(x, "x");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    at::Tensor y = at::empty_like(xc);
    check_status(spectral_scale(cptr(xc), mptr(y), static_cast<size_t>(xc.numel()),
                                static_cast<float>(alpha), stream()));
    return y;
}

at::Tensor fft_c2c_cuda(const at::Tensor& x, bool inverse, c10::string_view impl_name)
{
    check_complex64_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "fft_c2c: x needs at least one dimension");
    const ImplInfo impl = find_impl(impl_name);
    if (x.numel() == 0) {
        return at::empty_like(x, at::MemoryFormat::Contiguous);
    }
    const int64_t n = x.size(-1);
    TORCH_CHECK((n & (n - 1)) == 0, "fft_c2c: the last dimension must be a power of two, got ", n);
    TORCH_CHECK(n <= impl.max_c2c_n, "fft_c2c: ", impl.name, " supports sizes up to ",
                impl.max_c2c_n, ", got ", n);
    const int batch = batch_of(x, n, "fft_c2c");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    at::Tensor y = at::empty_like(xc);
    check_status(spectral_c2c(impl.name.c_str(), cptr(xc), mptr(y), static_cast<int>(n), batch,
                              inverse ? 1 : 0, stream()));
    return y;
}

at::Tensor fft_r2c_cuda(const at::Tensor& x, c10::string_view impl_name)
{
    check_float32_cuda(x);
    TORCH_CHECK(x.dim() >= 1, "fft_r2c: x needs at least one dimension");
    const ImplInfo impl = find_impl(impl_name);
    const int64_t n = x.size(-1);
    check_real_size(n, impl, "fft_r2c");
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n / 2 + 1;
    at::Tensor y = at::empty(shape, x.options().dtype(at::kComplexFloat));
    if (x.numel() == 0) {
        return y;
    }
    const int batch = batch_of(x, n, "fft_r2c");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    size_t count = 0;
    check_status(spectral_real_workspace(impl.name.c_str(), static_cast<int>(n), batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_r2c(impl.name.c_str(), xc.const_data_ptr<float>(), mptr(y),
                              static_cast<int>(n), batch, mptr(work), stream()));
    return y;
}

at::Tensor fft_c2r_cuda(const at::Tensor& x, int64_t n, c10::string_view impl_name)
{
    check_complex64_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "fft_c2r: x needs at least one dimension");
    const ImplInfo impl = find_impl(impl_name);
    check_real_size(n, impl, "fft_c2r");
    TORCH_CHECK(x.size(-1) == n / 2 + 1, "fft_c2r: an output of ", n, " points needs n/2 + 1 = ",
                n / 2 + 1, " inputs per transform, got ", x.size(-1));
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n;
    at::Tensor y = at::empty(shape, x.options().dtype(at::kFloat));
    if (x.numel() == 0) {
        return y;
    }
    const int batch = batch_of(x, n / 2 + 1, "fft_c2r");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    size_t count = 0;
    check_status(spectral_real_workspace(impl.name.c_str(), static_cast<int>(n), batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_c2r(impl.name.c_str(), cptr(xc), y.mutable_data_ptr<float>(),
                              static_cast<int>(n), batch, mptr(work), stream()));
    return y;
}

// "auto" picks the strided column kernel when the implementation has one (ops.cpp:187-202).
int parse_columns(c10::string_view text, const ImplInfo& impl)
{
    const std::string s(text.data(), text.size());
    if (s == "auto") {
        return impl.has_columns ? SPECTRAL_COLUMNS_STRIDED : SPECTRAL_COLUMNS_TRANSPOSE;
    }
    if (s == "strided") {
        TORCH_CHECK(impl.has_columns, impl.name,
                    " has no strided column kernel; use columns=\"transpose\"");
        return SPECTRAL_COLUMNS_STRIDED;
    }
    TORCH_CHECK(s == "transpose", "columns must be \"auto\", \"strided\", or \"transpose\", got '",
                s, "'");
    return SPECTRAL_COLUMNS_TRANSPOSE;
}

struct Shape2d {
    int64_t n1;
    int64_t n2;
    int batch;
};

Shape2d shape2d(const at::Tensor& x, int64_t n2, int64_t n2_stored, const char* op)
{
    TORCH_CHECK(x.dim() >= 2, op, ": x needs at least two dimensions");
    const int64_t n1 = x.size(-2);
    TORCH_CHECK(n1 >= 1 && n2 >= 1, op, ": empty transform dimensions");
    return {n1, n2, batch_of(x, n1 * n2_stored, op)};
}

at::Tensor fft2_c2c_cuda(const at::Tensor& x, bool inverse, c10::string_view impl_name,
                         c10::string_view columns)
{
    check_complex64_cuda(x, "x");
    const ImplInfo impl = find_impl(impl_name);
    const int method = parse_columns(columns, impl);
    TORCH_CHECK(x.dim() >= 2, "fft2_c2c: x needs at least two dimensions");
    if (x.numel() == 0) {
        return at::empty_like(x, at::MemoryFormat::Contiguous);
    }
    const Shape2d s = shape2d(x, x.size(-1), x.size(-1), "fft2_c2c");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    at::Tensor y = at::empty_like(xc);
    const auto n1 = static_cast<int>(s.n1);
    const auto n2 = static_cast<int>(s.n2);
    size_t count = 0;
    check_status(spectral_fft2_c2c_workspace(impl.name.c_str(), method, n1, n2, s.batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_fft2_c2c(impl.name.c_str(), method, cptr(xc), mptr(y), n1, n2, s.batch,
                                   inverse ? 1 : 0, mptr(work), stream()));
    return y;
}

at::Tensor fft2_r2c_cuda(const at::Tensor& x, c10::string_view impl_name, c10::string_view columns)
{
    check_float32_cuda(x);
    const ImplInfo impl = find_impl(impl_name);
    const int method = parse_columns(columns, impl);
    TORCH_CHECK(x.dim() >= 2, "fft2_r2c: x needs at least two dimensions");
    const int64_t n2 = x.size(-1);
    check_real_size(n2, impl, "fft2_r2c");
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n2 / 2 + 1;
    at::Tensor y = at::empty(shape, x.options().dtype(at::kComplexFloat));
    if (x.numel() == 0) {
        return y;
    }
    const Shape2d s = shape2d(x, n2, n2, "fft2_r2c");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    const auto n1 = static_cast<int>(s.n1);
    size_t count = 0;
    check_status(spectral_fft2_r2c_workspace(impl.name.c_str(), method, n1, static_cast<int>(n2),
                                             s.batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_fft2_r2c(impl.name.c_str(), method, xc.const_data_ptr<float>(), mptr(y),
                                   n1, static_cast<int>(n2), s.batch, mptr(work), stream()));
    return y;
}

at::Tensor fft2_c2r_cuda(const at::Tensor& x, int64_t n2, c10::string_view impl_name,
                         c10::string_view columns)
{
    check_complex64_cuda(x, "x");
    const ImplInfo impl = find_impl(impl_name);
    const int method = parse_columns(columns, impl);
    TORCH_CHECK(x.dim() >= 2, "fft2_c2r: x needs at least two dimensions");
    check_real_size(n2, impl, "fft2_c2r");
    TORCH_CHECK(x.size(-1) == n2 / 2 + 1, "fft2_c2r: an output of ", n2,
                " columns needs n2/2 + 1 = ", n2 / 2 + 1, " input columns, got ", x.size(-1));
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n2;
    at::Tensor y = at::empty(shape, x.options().dtype(at::kFloat));
    if (x.numel() == 0) {
        return y;
    }
    const Shape2d s = shape2d(x, n2, n2 / 2 + 1, "fft2_c2r");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    const auto n1 = static_cast<int>(s.n1);
    size_t count = 0;
    check_status(spectral_fft2_c2r_workspace(impl.name.c_str(), method, n1, static_cast<int>(n2),
                                             s.batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_fft2_c2r(impl.name.c_str(), method, cptr(xc), y.mutable_data_ptr<float>(),
                                   n1, static_cast<int>(n2), s.batch, mptr(work), stream()));
    return y;
}

at::Tensor fft_c2c_pruned_cuda(const at::Tensor& x, int64_t n, int64_t keep, bool inverse,
                               c10::string_view impl_name)
{
    check_complex64_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "fft_c2c_pruned: x needs at least one dimension");
    const ImplInfo impl = find_impl(impl_name);
    TORCH_CHECK(n >= 1 && n <= INT_MAX && keep >= 1 && keep <= n,
                "fft_c2c_pruned: need 1 <= keep <= n, got keep = ", keep, ", n = ", n);
    const int64_t row_in = inverse ? keep : n;
    TORCH_CHECK(x.size(-1) == row_in, "fft_c2c_pruned: expected ", row_in,
                " values in the last dimension, got ", x.size(-1));
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = inverse ? n : keep;
    at::Tensor y = at::empty(shape, x.options());
    if (x.numel() == 0) {
        return y;
    }
    const int batch = batch_of(x, row_in, "fft_c2c_pruned");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    size_t count = 0;
    check_status(spectral_c2c_pruned_workspace(impl.name.c_str(), static_cast<int>(n),
                                               static_cast<int>(keep), batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_c2c_pruned(impl.name.c_str(), cptr(xc), mptr(y), static_cast<int>(n),
                                     static_cast<int>(keep), batch, inverse ? 1 : 0, mptr(work),
                                     stream()));
    return y;
}

at::Tensor rfft2_modes_cuda(const at::Tensor& x, int64_t m1, int64_t m2, c10::string_view impl_name)
{
    check_float32_cuda(x);
    TORCH_CHECK(x.dim() >= 2, "rfft2_modes: x needs at least two dimensions");
    const ImplInfo impl = find_impl(impl_name);
    const int64_t n1 = x.size(-2);
    const int64_t n2 = x.size(-1);
    TORCH_CHECK(m1 >= 1 && 2 * m1 <= n1 && m2 >= 1 && m2 <= n2 / 2 + 1,
                "rfft2_modes: need 1 <= m1 <= n1/2 and 1 <= m2 <= n2/2 + 1, got m1 = ", m1,
                ", m2 = ", m2, " for ", n1, " x ", n2);
    std::vector<int64_t> shape = x.sizes().vec();
    shape[shape.size() - 2] = 2 * m1;
    shape.back() = m2;
    at::Tensor y = at::empty(shape, x.options().dtype(at::kComplexFloat));
    if (x.numel() == 0) {
        return y;
    }
    const int batch = batch_of(x, n1 * n2, "rfft2_modes");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    const int a = static_cast<int>(n1);
    const int b = static_cast<int>(n2);
    const int p = static_cast<int>(m1);
    const int q = static_cast<int>(m2);
    size_t count = 0;
    check_status(spectral_rfft2_modes_workspace(impl.name.c_str(), a, b, p, q, batch, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_rfft2_modes(impl.name.c_str(), xc.const_data_ptr<float>(), mptr(y), a, b,
                                      p, q, batch, mptr(work), stream()));
    return y;
}

at::Tensor irfft2_modes_cuda(const at::Tensor& modes, int64_t n1, int64_t n2,
                             c10::string_view impl_name)
{
    check_complex64_cuda(modes, "modes");
    TORCH_CHECK(modes.dim() >= 2, "irfft2_modes: modes needs at least two dimensions");
    const ImplInfo impl = find_impl(impl_name);
    const int64_t two_m1 = modes.size(-2);
    const int64_t m2 = modes.size(-1);
    TORCH_CHECK(two_m1 % 2 == 0 && two_m1 >= 2 && two_m1 <= n1 && m2 >= 1 && m2 <= n2 / 2 + 1,
                "irfft2_modes: modes of shape (", two_m1, ", ", m2, ") do not fit an output of ", n1,
                " x ", n2);
    std::vector<int64_t> shape = modes.sizes().vec();
    shape[shape.size() - 2] = n1;
    shape.back() = n2;
    at::Tensor y = at::empty(shape, modes.options().dtype(at::kFloat));
    if (modes.numel() == 0) {
        return y;
    }
    const int batch = batch_of(modes, two_m1 * m2, "irfft2_modes");
    const c10::cuda::CUDAGuard guard(modes.device());
    const at::Tensor mc = contiguous_aligned(modes);
    const int a = static_cast<int>(n1);
    const int b = static_cast<int>(n2);
    const int p = static_cast<int>(two_m1 / 2);
    const int q = static_cast<int>(m2);
    size_t count = 0;
    check_status(spectral_irfft2_modes_workspace(impl.name.c_str(), a, b, p, q, batch, &count));
    at::Tensor work = workspace(count, modes);
    check_status(spectral_irfft2_modes(impl.name.c_str(), cptr(mc), y.mutable_data_ptr<float>(), a,
                                       b, p, q, batch, mptr(work), stream()));
    return y;
}

// x (..., cin, modes...) complex64, w (cin, cout, modes...) complex64 -> (..., cout, modes...):
// the per-mode contraction of an FNO spectral convolution. Not one of the reference's operators
// (it has no implementation of it); an addition of this library.
at::Tensor mode_contract_cuda(const at::Tensor& x, const at::Tensor& w)
{
    check_complex64_cuda(x, "x");
    check_complex64_cuda(w, "w");
    TORCH_CHECK(x.dim() >= 2 && w.dim() == x.dim(),
                "mode_contract: x (batch..., cin, modes...) and w (cin, cout, modes...) need the "
                "same number of mode dimensions");
    const int64_t mode_dims = w.dim() - 2;
    const int64_t lead = x.dim() - mode_dims - 1;  // batch dimensions of x
    TORCH_CHECK(lead == 1, "mode_contract: x must be (batch, cin, modes...)");
    TORCH_CHECK(x.size(1) == w.size(0), "mode_contract: x has ", x.size(1), " channels, w expects ",
                w.size(0));
    for (int64_t d = 0; d < mode_dims; ++d) {
        TORCH_CHECK(x.size(2 + d) == w.size(2 + d), "mode_contract: mode shapes differ");
    }
    std::vector<int64_t> shape = x.sizes().vec();
    shape[1] = w.size(1);
    at::Tensor y = at::empty(shape, x.options());
    if (y.numel() == 0) {
        return y;
    }
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    const at::Tensor wc = contiguous_aligned(w);
    const int64_t modes = x.numel() / (x.size(0) * x.size(1));
    check_status(spectral_mode_contract(cptr(xc), cptr(wc), mptr(y), x.size(0),
                                        static_cast<int>(x.size(1)), static_cast<int>(w.size(1)),
                                        modes, stream()));
    return y;
}

// The fused radio-signal kernels behind spectral.rf: x is (..., n) complex64, each leading index
// one signal. The Python layer picks these for the stockham implementations and nfft <= 4096.
at::Tensor spectrum_frames_cuda(const at::Tensor& x, int64_t nfft, const c10::optional<at::Tensor>& window,
                                c10::string_view impl_name)
{
    check_complex64_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "spectrum: x needs at least one dimension");
    const std::string impl(impl_name.data(), impl_name.size());
    const int64_t n = x.size(-1);
    int64_t rows = 1;  // the product of the leading dimensions (x may be empty)
    for (int64_t d = 0; d + 1 < x.dim(); ++d) {
        rows *= x.size(d);
    }
    TORCH_CHECK(nfft >= 2 && nfft <= 4096 && (nfft & (nfft - 1)) == 0,
                "spectrum: nfft must be a power of two from 2 to 4096, got ", nfft);
    const int64_t frames = n == 0 ? 1 : (n + nfft - 1) / nfft;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
    shape.push_back(frames);
    shape.push_back(nfft);
    at::Tensor y = at::empty(shape, x.options());
    at::Tensor wc;
    if (window.has_value()) {
        TORCH_CHECK(window->is_cuda() && window->scalar_type() == at::kFloat && window->dim() == 1
                        && window->size(0) == nfft,
                    "spectrum: the window must be a float32 CUDA tensor of nfft = ", nfft, " values");
        wc = window->contiguous();
    }
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    check_status(spectral_spectrum(impl.c_str(), n == 0 ? nullptr : cptr(xc),
                                   window.has_value() ? wc.const_data_ptr<float>() : nullptr, mptr(y), n,
                                   static_cast<int>(nfft), rows, stream()));
    return y;
}

at::Tensor fir_overlap_save_cuda(const at::Tensor& x, const at::Tensor& taps_spectrum, int64_t taps,
                                 int64_t nfft, c10::string_view impl_name)
{
    check_complex64_cuda(x, "x");
    check_complex64_cuda(taps_spectrum, "taps_spectrum");
    TORCH_CHECK(x.dim() >= 1, "fir: x needs at least one dimension");
    TORCH_CHECK(taps_spectrum.dim() == 1 && taps_spectrum.size(0) == nfft,
                "fir: taps_spectrum must hold nfft = ", nfft, " values");
    TORCH_CHECK(taps >= 1 && taps <= nfft, "fir: need 1 <= taps <= nfft");
    const std::string impl(impl_name.data(), impl_name.size());
    at::Tensor y = at::empty(x.sizes(), x.options());
    const int64_t n = x.size(-1);
    const int64_t rows = n == 0 ? 0 : x.numel() / n;
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = contiguous_aligned(x);
    const at::Tensor hc = contiguous_aligned(taps_spectrum);
    check_status(spectral_fir(impl.c_str(), n == 0 ? nullptr : cptr(xc), cptr(hc),
                              n == 0 ? nullptr : mptr(y), n, static_cast<int>(nfft),
                              static_cast<int>(taps), rows, stream()));
    return y;
}

// One stage of the Navier-Stokes step (spectral.flow.gpu): writes f0 (predictor) and out.
void flow_stage_cuda(const at::Tensor& x, const at::Tensor& w, at::Tensor& f0, at::Tensor& out,
                     const at::Tensor& derive, const at::Tensor& forcing, const at::Tensor& mask,
                     const at::Tensor& explicit_factor, const at::Tensor& implicit_factor, at::Tensor& work,
                     int64_t n, int64_t m, double dt, int64_t stage, c10::string_view impl_name)
{
    for (const at::Tensor* t : {&x, &w, const_cast<const at::Tensor*>(&f0), const_cast<const at::Tensor*>(&out),
                                &derive, &forcing, const_cast<const at::Tensor*>(&work)}) {
        check_complex64_cuda(*t, "flow_stage arrays");
        TORCH_CHECK(t->is_contiguous(), "flow_stage: arrays must be contiguous");
    }
    for (const at::Tensor* t : {&mask, &explicit_factor, &implicit_factor}) {
        TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kFloat && t->is_contiguous(),
                    "flow_stage: mask and factors must be contiguous float32 CUDA tensors");
    }
    const int64_t plane = 2 * m * m;
    TORCH_CHECK(x.numel() % plane == 0 && w.numel() == x.numel() && f0.numel() == x.numel() && out.numel() == x.numel(),
                "flow_stage: states must be (batch, 2m, m)");
    TORCH_CHECK(derive.numel() == 4 * plane && forcing.numel() == plane && mask.numel() == plane,
                "flow_stage: derive (4, 2m, m), forcing and mask (2m, m)");
    const int64_t batch = x.numel() / plane;
    const int64_t vs = explicit_factor.numel() == plane ? 0 : plane;
    TORCH_CHECK(explicit_factor.numel() == implicit_factor.numel()
                    && (vs == 0 || explicit_factor.numel() == batch * plane),
                "flow_stage: the factors must be (2m, m) or (batch, 2m, m)");
    size_t count = 0;
    check_status(spectral_flow_workspace(static_cast<int>(n), static_cast<int>(m), batch, &count));
    TORCH_CHECK(static_cast<size_t>(work.numel()) >= count, "flow_stage: work needs ", count, " values");
    const std::string impl(impl_name.data(), impl_name.size());
    const c10::cuda::CUDAGuard guard(x.device());
    check_status(spectral_flow_stage(impl.c_str(), cptr(x), cptr(w), mptr(f0), mptr(out), cptr(derive), cptr(forcing),
                                     mask.const_data_ptr<float>(), explicit_factor.const_data_ptr<float>(),
                                     implicit_factor.const_data_ptr<float>(), vs, mptr(work), static_cast<int>(n),
                                     static_cast<int>(m), batch, static_cast<float>(dt), static_cast<int>(stage),
                                     stream()));
}

// --- the pointwise half of an FNO block: additions of this library ------------------------------

int dtype_code(const at::Tensor& t, const char* op, const char* name)
{
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor");
    switch (t.scalar_type()) {
        case at::kFloat: return SPECTRAL_FLOAT32;
        case at::kBFloat16: return SPECTRAL_BFLOAT16;
        case at::kHalf: return SPECTRAL_FLOAT16;
        default: break;
    }
    TORCH_CHECK(false, op, ": ", name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

int activation_code(c10::string_view activation, const char* op)
{
    if (activation == "none") {
        return SPECTRAL_ACT_NONE;
    }
    if (activation == "silu") {
        return SPECTRAL_ACT_SILU;
    }
    TORCH_CHECK(activation == "gelu", op, ": activation must be 'none', 'silu' or 'gelu', got '",
                std::string(activation.data(), activation.size()), "'");
    return SPECTRAL_ACT_GELU;
}

int small_int(int64_t v, const char* op, const char* name)
{
    TORCH_CHECK(v <= INT_MAX, op, ": ", name, " is too large: ", v);
    return static_cast<int>(v);
}

// `t` must be of x's type and device.
void check_like(const at::Tensor& t, const at::Tensor& x, const char* op, const char* name)
{
    TORCH_CHECK(t.is_cuda() && t.device() == x.device(), op, ": ", name, " must be on the device of x");
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), op, ": ", name, " must be ", x.scalar_type(), " as x, got ",
                t.scalar_type());
}

// An optional per-channel parameter: `channels` float32 values, contiguous (undefined if not given).
at::Tensor channel_parameter(const c10::optional<at::Tensor>& t, const at::Tensor& x, int64_t channels, const char* op,
                             const char* name)
{
    if (!t.has_value() || !t->defined()) {
        return at::Tensor();
    }
    TORCH_CHECK(t->is_cuda() && t->device() == x.device() && t->scalar_type() == at::kFloat && t->dim() == 1
                    && t->size(0) == channels,
                op, ": ", name, " must be a float32 tensor of ", channels, " values on the device of x");
    return t->contiguous();
}

const float* fptr(const at::Tensor& t) { return t.defined() && t.numel() > 0 ? t.const_data_ptr<float>() : nullptr; }

std::vector<int64_t> scale_shape(const at::Tensor& x)
{
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = (shape.back() + SPECTRAL_PACK8_BLOCK - 1) / SPECTRAL_PACK8_BLOCK;
    return shape;
}

int64_t rows_of(const at::Tensor& x)
{
    int64_t rows = 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) {
        rows *= x.size(d);
    }
    return rows;
}

// codes int8 of `like`'s shape with one float32 scale per row and block, contiguous.
void check_packed(const at::Tensor& codes, const at::Tensor& scales, const char* op)
{
    TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kChar && codes.dim() >= 1, op,
                ": codes must be an int8 CUDA tensor with at least one dimension");
    TORCH_CHECK(scales.is_cuda() && scales.device() == codes.device() && scales.scalar_type() == at::kFloat
                    && scales.sizes() == at::IntArrayRef(scale_shape(codes)),
                op, ": scales must be float32 of shape ", at::IntArrayRef(scale_shape(codes)), " on the device of codes");
}

std::tuple<at::Tensor, at::Tensor> pack8_cuda(const at::Tensor& x)
{
    const int dtype = dtype_code(x, "pack8", "x");
    TORCH_CHECK(x.dim() >= 1, "pack8: x needs at least one dimension");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = x.contiguous();
    at::Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
    at::Tensor scales = at::empty(scale_shape(x), x.options().dtype(at::kFloat));
    check_status(spectral_pack8(cptr(xc), dtype, mptr(codes), static_cast<float*>(mptr(scales)), rows_of(x),
                                small_int(x.size(-1), "pack8", "the last dimension"), stream()));
    return {codes, scales};
}

at::Tensor unpack8_cuda(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype)
{
    check_packed(codes, scales, "unpack8");
    const c10::cuda::CUDAGuard guard(codes.device());
    at::Tensor x = at::empty(codes.sizes(), codes.options().dtype(dtype));
    const int code = dtype_code(x, "unpack8", "the result");
    const at::Tensor cc = codes.contiguous();
    const at::Tensor sc = scales.contiguous();
    check_status(spectral_unpack8(cptr(cc), fptr(sc), mptr(x), code, rows_of(codes),
                                  small_int(codes.size(-1), "unpack8", "the last dimension"), stream()));
    return x;
}

struct NormSizes {
    int64_t batch;
    int64_t points;
    int channels;
    int groups;
};

NormSizes norm_sizes(const at::Tensor& x, int64_t groups, const char* op)
{
    TORCH_CHECK(x.dim() >= 2, op, ": x must be (batch, ..., channels)");
    NormSizes s{x.size(0), 1, small_int(x.size(-1), op, "the number of channels"), small_int(groups, op, "groups")};
    for (int64_t d = 1; d + 1 < x.dim(); ++d) {
        s.points *= x.size(d);
    }
    TORCH_CHECK(groups >= 1 && s.channels >= 1 && s.channels % groups == 0, op, ": groups must divide the number of channels, got ",
                groups, " groups of ", s.channels, " channels");
    return s;
}

// x (batch, ..., channels) lies in memory as (batch, channels, ...), in a shape and alignment that the
// library's channels-first kernels take.
bool channels_first(const at::Tensor& x, const NormSizes& n)
{
    const int64_t values = 16 / x.element_size();
    return !x.is_contiguous() && n.channels % 8 == 0 && n.points % values == 0 && x.movedim(-1, 1).is_contiguous()
           && (reinterpret_cast<uintptr_t>(x.const_data_ptr()) & 15u) == 0;
}

// x with its channels last in memory.
at::Tensor last_contiguous(const at::Tensor& x, int dtype, const NormSizes& n)
{
    if (x.numel() == 0 || !channels_first(x, n)) {
        return x.contiguous();
    }
    at::Tensor y = at::empty(x.sizes(), x.options());
    check_status(spectral_channels_last(cptr(x), mptr(y), dtype, n.batch, n.points, n.channels, stream()));
    return y;
}

// stats: (2, batch, groups), the means and the reciprocal standard deviations (undefined if not wanted).
struct NormResult {
    at::Tensor y;
    at::Tensor stats;
    at::Tensor codes;
    at::Tensor scales;
};

NormResult norm_forward(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight,
                        const c10::optional<at::Tensor>& bias, double eps, c10::string_view activation, bool keep8,
                        bool keep_stats)
{
    constexpr const char* op = "group_norm_act";
    const int dtype = dtype_code(x, op, "x");
    const NormSizes n = norm_sizes(x, groups, op);
    const int act = activation_code(activation, op);
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor w = channel_parameter(weight, x, n.channels, op, "weight");
    const at::Tensor b = channel_parameter(bias, x, n.channels, op, "bias");
    const bool first = x.numel() > 0 && !keep8 && channels_first(x, n);
    const at::Tensor xc = first ? x : last_contiguous(x, dtype, n);
    at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor stats;
    at::Tensor codes;
    at::Tensor scales;
    if (keep_stats) {
        stats = at::empty({2, n.batch, groups}, x.options().dtype(at::kFloat));
    }
    if (keep8) {
        codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
        scales = at::empty(scale_shape(x), x.options().dtype(at::kFloat));
    }
    if (x.numel() == 0) {
        if (keep_stats) {
            stats.zero_();
        }
        return {y, stats, codes, scales};
    }
    size_t count = 0;
    check_status(spectral_group_norm_act_workspace(dtype, n.batch, n.points, n.channels, n.groups, &count));
    at::Tensor work = workspace(count, x);
    float* mean = keep_stats ? static_cast<float*>(mptr(stats)) : nullptr;
    check_status(spectral_group_norm_act(cptr(xc), fptr(w), fptr(b), mptr(y), mean,
                                         keep_stats ? mean + n.batch * groups : nullptr, keep8 ? mptr(codes) : nullptr,
                                         keep8 ? static_cast<float*>(mptr(scales)) : nullptr, dtype, first ? 1 : 0, n.batch,
                                         n.points, n.channels, n.groups, static_cast<float>(eps), act, mptr(work), stream()));
    return {y, stats, codes, scales};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
group_norm_act_cuda(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight,
                    const c10::optional<at::Tensor>& bias, double eps, c10::string_view activation, bool keep8)
{
    const NormResult r = norm_forward(x, groups, weight, bias, eps, activation, keep8, true);
    return {r.y, r.stats.select(0, 0), r.stats.select(0, 1), r.codes, r.scales};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor>
norm_backward(const at::Tensor& dy, const c10::optional<at::Tensor>& x, const c10::optional<at::Tensor>& codes,
              const c10::optional<at::Tensor>& scales, const c10::optional<at::Tensor>& weight,
              const c10::optional<at::Tensor>& bias, const float* mean, const float* rstd, int64_t groups,
              c10::string_view activation)
{
    constexpr const char* op = "group_norm_act_backward";
    const int dtype = dtype_code(dy, op, "dy");
    const NormSizes n = norm_sizes(dy, groups, op);
    const int act = activation_code(activation, op);
    TORCH_CHECK(x.has_value() != codes.has_value() && codes.has_value() == scales.has_value(), op,
                ": needs either x or codes with scales");
    const c10::cuda::CUDAGuard guard(dy.device());
    at::Tensor xc;
    at::Tensor cc;
    at::Tensor sc;
    if (x.has_value()) {
        check_like(*x, dy, op, "x");
        TORCH_CHECK(x->sizes() == dy.sizes(), op, ": x and dy must have one shape");
        xc = last_contiguous(*x, dtype, n);
    } else {
        check_packed(*codes, *scales, op);
        TORCH_CHECK(codes->device() == dy.device() && codes->sizes() == dy.sizes(), op,
                    ": codes must have the shape and device of dy");
        cc = codes->contiguous();
        sc = scales->contiguous();
    }
    const at::Tensor w = channel_parameter(weight, dy, n.channels, op, "weight");
    const at::Tensor b = channel_parameter(bias, dy, n.channels, op, "bias");
    const at::Tensor dyc = last_contiguous(dy, dtype, n);
    at::Tensor dx = at::empty(dy.sizes(), dy.options());
    at::Tensor dweight = at::empty({n.channels}, dy.options().dtype(at::kFloat));
    at::Tensor dbias = at::empty_like(dweight);
    size_t count = 0;
    check_status(spectral_group_norm_act_backward_workspace(dtype, n.batch, n.points, n.channels, n.groups, &count));
    at::Tensor work = workspace(count, dy);
    check_status(spectral_group_norm_act_backward(
        cptr(dyc), xc.defined() ? cptr(xc) : nullptr, cc.defined() ? cptr(cc) : nullptr, fptr(sc), fptr(w), fptr(b),
        mean, rstd, mptr(dx), static_cast<float*>(mptr(dweight)), static_cast<float*>(mptr(dbias)), dtype, n.batch, n.points,
        n.channels, n.groups, act, mptr(work), stream()));
    return {dx, dweight, dbias};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor>
group_norm_act_backward_cuda(const at::Tensor& dy, const c10::optional<at::Tensor>& x,
                             const c10::optional<at::Tensor>& codes, const c10::optional<at::Tensor>& scales,
                             const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& bias,
                             const at::Tensor& mean, const at::Tensor& rstd, int64_t groups, c10::string_view activation)
{
    constexpr const char* op = "group_norm_act_backward";
    const NormSizes n = norm_sizes(dy, groups, op);
    for (const at::Tensor* t : {&mean, &rstd}) {
        TORCH_CHECK(t->is_cuda() && t->device() == dy.device() && t->scalar_type() == at::kFloat && t->dim() == 2
                        && t->size(0) == n.batch && t->size(1) == groups && t->is_contiguous(),
                    op, ": mean and rstd must be contiguous float32 (batch, groups) on the device of dy");
    }
    return norm_backward(dy, x, codes, scales, weight, bias, fptr(mean), fptr(rstd), groups, activation);
}

struct MlpSizes {
    int64_t tokens;
    int channels;
    int hidden;
    int outputs;
};

// x is (..., channels); its rows are the tokens.
MlpSizes mlp_sizes(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up, const at::Tensor& w_down,
                   const char* op)
{
    TORCH_CHECK(x.dim() >= 1, op, ": x needs at least one dimension");
    TORCH_CHECK(w_gate.dim() == 2 && w_up.dim() == 2 && w_down.dim() == 2, op, ": the weights must be matrices");
    TORCH_CHECK(w_gate.size(1) == x.size(-1) && w_up.sizes() == w_gate.sizes() && w_down.size(1) == w_gate.size(0), op,
                ": x (..., channels), w_gate and w_up (hidden, channels) and w_down (outputs, hidden) do not match: ",
                x.sizes(), ", ", w_gate.sizes(), ", ", w_up.sizes(), ", ", w_down.sizes());
    return {rows_of(x), small_int(x.size(-1), op, "the number of channels"), small_int(w_gate.size(0), op, "hidden"),
            small_int(w_down.size(0), op, "outputs")};
}

at::Tensor gated_mlp_cuda(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up, const at::Tensor& w_down,
                          c10::string_view activation)
{
    constexpr const char* op = "gated_mlp";
    const int dtype = dtype_code(x, op, "x");
    check_like(w_gate, x, op, "w_gate");
    check_like(w_up, x, op, "w_up");
    check_like(w_down, x, op, "w_down");
    const MlpSizes n = mlp_sizes(x, w_gate, w_up, w_down, op);
    const int act = activation_code(activation, op);
    const c10::cuda::CUDAGuard guard(x.device());
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n.outputs;
    at::Tensor y = at::empty(shape, x.options());
    const at::Tensor xc = x.contiguous();
    const at::Tensor wg = w_gate.contiguous();
    const at::Tensor wu = w_up.contiguous();
    const at::Tensor wd = w_down.contiguous();
    size_t count = 0;
    check_status(spectral_gated_mlp_workspace_for(cptr(xc), cptr(wg), cptr(wu), cptr(wd), dtype, n.tokens, n.channels, n.hidden, n.outputs, &count));
    at::Tensor work = workspace(count, x);
    check_status(spectral_gated_mlp(cptr(xc), cptr(wg), cptr(wu), cptr(wd), mptr(y), dtype, n.tokens, n.channels, n.hidden,
                                    n.outputs, act, mptr(work), stream()));
    return y;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>
gated_mlp_backward_cuda(const at::Tensor& dy, const c10::optional<at::Tensor>& x, const c10::optional<at::Tensor>& codes,
                        const c10::optional<at::Tensor>& scales, const at::Tensor& w_gate, const at::Tensor& w_up,
                        const at::Tensor& w_down, c10::string_view activation)
{
    constexpr const char* op = "gated_mlp_backward";
    const int dtype = dtype_code(dy, op, "dy");
    TORCH_CHECK(x.has_value() != codes.has_value() && codes.has_value() == scales.has_value(), op,
                ": needs either x or codes with scales");
    check_like(w_gate, dy, op, "w_gate");
    check_like(w_up, dy, op, "w_up");
    check_like(w_down, dy, op, "w_down");
    const c10::cuda::CUDAGuard guard(dy.device());
    at::Tensor xc;
    at::Tensor cc;
    at::Tensor sc;
    if (x.has_value()) {
        check_like(*x, dy, op, "x");
        xc = x->contiguous();
    } else {
        check_packed(*codes, *scales, op);
        TORCH_CHECK(codes->device() == dy.device(), op, ": codes must be on the device of dy");
        cc = codes->contiguous();
        sc = scales->contiguous();
    }
    const at::Tensor& input = x.has_value() ? *x : *codes;
    const MlpSizes n = mlp_sizes(input, w_gate, w_up, w_down, op);
    std::vector<int64_t> shape = input.sizes().vec();
    shape.back() = n.outputs;
    TORCH_CHECK(dy.sizes() == at::IntArrayRef(shape), op, ": dy must be ", at::IntArrayRef(shape), ", got ", dy.sizes());
    const int act = activation_code(activation, op);
    const at::Tensor dyc = dy.contiguous();
    const at::Tensor wg = w_gate.contiguous();
    const at::Tensor wu = w_up.contiguous();
    const at::Tensor wd = w_down.contiguous();
    at::Tensor dx = at::empty(input.sizes(), dy.options());
    at::Tensor dwg = at::empty(wg.sizes(), dy.options());
    at::Tensor dwu = at::empty(wg.sizes(), dy.options());
    at::Tensor dwd = at::empty(wd.sizes(), dy.options());
    size_t count = 0;
    check_status(spectral_gated_mlp_backward_workspace_for(cptr(dyc), xc.defined() ? cptr(xc) : nullptr, cc.defined() ? 1 : 0,
                                                           cptr(wg), cptr(wu), cptr(wd), dtype, n.tokens, n.channels, n.hidden, n.outputs, &count));
    at::Tensor work = workspace(count, dy);
    check_status(spectral_gated_mlp_backward(cptr(dyc), xc.defined() ? cptr(xc) : nullptr, cc.defined() ? cptr(cc) : nullptr,
                                             fptr(sc), cptr(wg), cptr(wu), cptr(wd), mptr(dx), mptr(dwg), mptr(dwu),
                                             mptr(dwd), dtype, n.tokens, n.channels, n.hidden, n.outputs, act, mptr(work),
                                             stream()));
    return {dx, dwg, dwu, dwd};
}

// --- reading from states of another length: additions of this library ---------------------------

// The values of a head side by side; other strides are the kernels' business.
at::Tensor head_rows(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

struct RotarySettings {
    int64_t rotated;
    double eps;
    double theta;
    std::string pairs;
};

int pairs_code(const std::string& pairs, const char* op)
{
    if (pairs == "halves") {
        return SPECTRAL_PAIRS_HALVES;
    }
    TORCH_CHECK(pairs == "neighbours", op, ": pairs must be 'halves' or 'neighbours', got '", pairs, "'");
    return SPECTRAL_PAIRS_NEIGHBOURS;
}

// One side of the call: x (batch, tokens, heads, dim), an optional weight and optional positions. Keeps what the
// descriptor points to.
struct RotarySide {
    at::Tensor x, weight, positions, dy, out, dweight;
    spectral_heads heads{};
    int axes = 0;
};

// `like`: the first side, whose type, device, batch and dim the others have.
RotarySide rotary_side(const at::Tensor& x, const c10::optional<at::Tensor>& weight, const c10::optional<at::Tensor>& positions,
                       const at::Tensor& like, const char* op, const char* name)
{
    TORCH_CHECK(x.dim() == 4, op, ": ", name, " must be (batch, tokens, heads, dim), got ", x.sizes());
    dtype_code(x, op, name);
    check_like(x, like, op, name);
    TORCH_CHECK(x.size(0) == like.size(0) && x.size(3) == like.size(3), op, ": q and k must agree in batch and dim, got ",
                like.sizes(), " and ", x.sizes());
    RotarySide s;
    s.x = head_rows(x);
    s.weight = channel_parameter(weight, x, x.size(3), op, name == std::string("q") ? "q_weight" : "k_weight");
    s.heads.x = cptr(s.x);
    for (int i = 0; i < 3; ++i) {
        s.heads.stride[i] = s.x.stride(i);
    }
    s.heads.weight = fptr(s.weight);
    s.heads.heads = small_int(x.size(2), op, "the number of heads");
    s.heads.tokens = x.size(1);
    if (positions.has_value() && positions->defined()) {
        s.positions = *positions;
        const at::Tensor& p = s.positions;
        TORCH_CHECK(p.is_cuda() && p.device() == x.device(), op, ": ", name, "_positions must be on the device of ", name);
        const bool shared = p.dim() == 2;
        TORCH_CHECK((shared || (p.dim() == 3 && p.size(0) == x.size(0))) && p.size(-2) == x.size(1) && p.size(-1) >= 1, op, ": ", name,
                    "_positions must be (tokens, axes) or (batch, tokens, axes) for ", name, " ", x.sizes(), ", got ", p.sizes());
        switch (p.scalar_type()) {
            case at::kFloat: s.heads.position_type = SPECTRAL_POSITIONS_FLOAT32; break;
            case at::kInt: s.heads.position_type = SPECTRAL_POSITIONS_INT32; break;
            case at::kLong: s.heads.position_type = SPECTRAL_POSITIONS_INT64; break;
            default: TORCH_CHECK(false, op, ": ", name, "_positions must be float32, int32 or int64, got ", p.scalar_type());
        }
        s.heads.positions = cptr(p);
        s.heads.position_stride[0] = shared ? 0 : p.stride(0);
        s.heads.position_stride[1] = p.stride(-2);
        s.heads.position_stride[2] = p.stride(-1);
        s.axes = small_int(p.size(-1), op, "the number of axes");
    }
    return s;
}

// The axes of the call: those of its positions (1 if there are none).
int rotary_axes(const std::vector<RotarySide>& sides, const char* op)
{
    int axes = 0;
    for (const RotarySide& s : sides) {
        TORCH_CHECK(axes == 0 || s.axes == 0 || s.axes == axes, op, ": q_positions and k_positions must have the same axes");
        axes = std::max(axes, s.axes);
    }
    return std::max(axes, 1);
}

// As many values of a head as `axes` spans of pairs hold, unless the caller says how many.
int rotary_values(int64_t rotated, int64_t dim, int axes, const char* op)
{
    if (rotated < 0) {
        return static_cast<int>(dim / (2LL * axes) * (2LL * axes));
    }
    return small_int(rotated, op, "rotated");
}

const char* side_name(size_t i) { return i == 1 ? "k" : "q"; }

variable_list_t rotary_forward(const variable_list_t& x, const std::vector<c10::optional<at::Tensor>>& weight,
                               const std::vector<c10::optional<at::Tensor>>& positions, const RotarySettings& set)
{
    constexpr const char* op = "qk_norm_rotary";
    const int dtype = dtype_code(x[0], op, "q");
    const int pairs = pairs_code(set.pairs, op);
    std::vector<RotarySide> sides;
    for (size_t i = 0; i < x.size(); ++i) {
        sides.push_back(rotary_side(x[i], weight[i], positions[i], x[0], op, side_name(i)));
    }
    const int axes = rotary_axes(sides, op);
    const int dim = small_int(x[0].size(3), op, "dim");
    const c10::cuda::CUDAGuard guard(x[0].device());
    variable_list_t out;
    for (RotarySide& s : sides) {
        out.push_back(at::empty(s.x.sizes(), s.x.options()));
        s.heads.out = mptr(out.back());
    }
    check_status(spectral_qk_norm_rotary(&sides[0].heads, sides.size() > 1 ? &sides[1].heads : nullptr, dtype, x[0].size(0), dim,
                                         rotary_values(set.rotated, dim, axes, op), axes, pairs, static_cast<float>(set.eps),
                                         static_cast<float>(set.theta), stream()));
    return out;
}

// dx of each side, then dweight of each (undefined without a weight). A side whose dy is undefined has neither.
variable_list_t rotary_backward(const variable_list_t& dy, const variable_list_t& x, const std::vector<c10::optional<at::Tensor>>& weight,
                                const std::vector<c10::optional<at::Tensor>>& positions, const RotarySettings& set)
{
    constexpr const char* op = "qk_norm_rotary_backward";
    const int dtype = dtype_code(x[0], op, "q");
    const int pairs = pairs_code(set.pairs, op);
    std::vector<RotarySide> sides;
    for (size_t i = 0; i < x.size(); ++i) {
        sides.push_back(rotary_side(x[i], weight[i], positions[i], x[0], op, side_name(i)));
    }
    const int axes = rotary_axes(sides, op);
    const int dim = small_int(x[0].size(3), op, "dim");
    const c10::cuda::CUDAGuard guard(x[0].device());
    const spectral_heads* given[2] = {nullptr, nullptr};
    size_t count = 0;
    check_status(spectral_qk_norm_rotary_backward_workspace(dim, &count));
    for (size_t i = 0; i < sides.size(); ++i) {
        RotarySide& s = sides[i];
        if (!dy[i].defined()) {
            continue;
        }
        check_like(dy[i], x[i], op, "dy");
        TORCH_CHECK(dy[i].sizes() == x[i].sizes(), op, ": dy must be ", x[i].sizes(), ", got ", dy[i].sizes());
        s.dy = dy[i].contiguous();
        s.out = at::empty(s.x.sizes(), s.x.options());
        s.heads.dy = cptr(s.dy);
        s.heads.out = mptr(s.out);
        if (s.weight.defined()) {
            s.dweight = at::empty(s.weight.sizes(), s.weight.options());
            s.heads.dweight = static_cast<float*>(mptr(s.dweight));
        }
        given[i] = &s.heads;
    }
    variable_list_t results;
    if (given[0] != nullptr || given[1] != nullptr) {
        at::Tensor work = workspace(count, x[0]);
        check_status(spectral_qk_norm_rotary_backward(given[0], given[1], dtype, x[0].size(0), dim, rotary_values(set.rotated, dim, axes, op), axes,
                                                      pairs, static_cast<float>(set.eps), static_cast<float>(set.theta), mptr(work), stream()));
    }
    for (const RotarySide& s : sides) {
        results.push_back(s.out);
    }
    for (const RotarySide& s : sides) {
        results.push_back(s.dweight);
    }
    return results;
}

std::vector<c10::optional<at::Tensor>> two(const c10::optional<at::Tensor>& a, const c10::optional<at::Tensor>& b) { return {a, b}; }

variable_list_t qk_norm_rotary_cuda(const at::Tensor& q, const c10::optional<at::Tensor>& k, const c10::optional<at::Tensor>& q_weight,
                                    const c10::optional<at::Tensor>& k_weight, const c10::optional<at::Tensor>& q_positions,
                                    const c10::optional<at::Tensor>& k_positions, double eps, double theta, int64_t rotated,
                                    c10::string_view pairs)
{
    variable_list_t x{q};
    if (k.has_value() && k->defined()) {
        x.push_back(*k);
    }
    return rotary_forward(x, two(q_weight, k_weight), two(q_positions, k_positions),
                          {rotated, eps, theta, std::string(pairs.data(), pairs.size())});
}

struct AttentionSizes {
    int64_t batch, queries, keys;
    int heads, kv_heads, dim;
};

AttentionSizes attention_sizes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const char* op)
{
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3), op,
                ": q (batch, queries, heads, dim) and k and v (batch, keys, kv_heads, dim) do not match: ", q.sizes(), ", ", k.sizes(), ", ",
                v.sizes());
    return {q.size(0), q.size(1), k.size(1), small_int(q.size(2), op, "heads"), small_int(k.size(2), op, "kv_heads"), small_int(q.size(3), op, "dim")};
}

// The call's arrays as the C ABI takes them.
struct AttentionArrays {
    at::Tensor q, k, v, lengths, mask;
    long long strides[9];
    AttentionSizes n;
    int dtype;
    float scale;
    int lengths64() const { return lengths.defined() && lengths.scalar_type() == at::kLong ? 1 : 0; }
    const void* lengths_ptr() const { return lengths.defined() && lengths.numel() > 0 ? cptr(lengths) : nullptr; }
    const void* mask_ptr() const { return mask.defined() && mask.numel() > 0 ? cptr(mask) : nullptr; }

    AttentionArrays(const at::Tensor& q0, const at::Tensor& k0, const at::Tensor& v0, const c10::optional<at::Tensor>& lengths0,
                    const c10::optional<at::Tensor>& mask0, c10::optional<double> scale0, const char* op)
    {
        dtype = dtype_code(q0, op, "q");
        check_like(k0, q0, op, "k");
        check_like(v0, q0, op, "v");
        n = attention_sizes(q0, k0, v0, op);
        q = head_rows(q0);
        k = head_rows(k0);
        v = head_rows(v0);
        const at::Tensor* arrays[3] = {&q, &k, &v};
        for (int i = 0; i < 9; ++i) {
            strides[i] = arrays[i / 3]->stride(i % 3);
        }
        scale = scale0.has_value() ? static_cast<float>(*scale0) : 1.0f / std::sqrt(static_cast<float>(n.dim));
        if (lengths0.has_value() && lengths0->defined()) {
            const at::Tensor& l = *lengths0;
            TORCH_CHECK(l.is_cuda() && l.device() == q.device() && (l.scalar_type() == at::kInt || l.scalar_type() == at::kLong)
                            && l.dim() == 1 && l.size(0) == n.batch,
                        op, ": lengths must be an int32 or int64 tensor of ", n.batch, " values on the device of q");
            lengths = l.contiguous();
        }
        if (mask0.has_value() && mask0->defined()) {
            const at::Tensor& m = *mask0;
            TORCH_CHECK(m.is_cuda() && m.device() == q.device() && m.scalar_type() == at::kBool && m.dim() == 2
                            && (m.size(0) == n.batch || m.size(0) == 1) && m.size(1) == n.keys,
                        op, ": mask must be a bool tensor (batch, keys) or (1, keys) on the device of q, got ", m.scalar_type(), " ", m.sizes());
            mask = m.expand({n.batch, n.keys}).contiguous();
        }
    }
};

// out; stats and, for 16-bit types, rest if they are kept.
struct AttentionResult {
    at::Tensor out, stats, rest;
};

AttentionResult attention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                     const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& mask,
                                                     c10::optional<double> scale, bool keep)
{
    constexpr const char* op = "cross_attention";
    TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(q.device());
    const AttentionArrays a(q, k, v, lengths, mask, scale, op);
    const AttentionSizes& n = a.n;
    at::Tensor out = at::empty(q.sizes(), q.options());
    at::Tensor stats;
    at::Tensor rest;
    if (keep) {
        stats = at::empty({n.batch, n.kv_heads, n.kv_heads > 0 ? n.queries * (n.heads / n.kv_heads) : 0, 2}, q.options().dtype(at::kFloat));
        rest = at::empty(q.scalar_type() == at::kFloat ? at::IntArrayRef({0}) : q.sizes(), q.options().dtype(at::kChar));
    }
    size_t count = 0;
    check_status(spectral_cross_attention_workspace(cptr(a.q), cptr(a.k), cptr(a.v), a.strides, a.dtype, n.batch, n.queries, n.keys, n.heads,
                                                    n.kv_heads, n.dim, &count));
    at::Tensor work = workspace(count, q);
    check_status(spectral_cross_attention(cptr(a.q), cptr(a.k), cptr(a.v), a.strides, a.lengths_ptr(), a.lengths64(), a.mask_ptr(), mptr(out),
                                          keep ? mptr(rest) : nullptr, keep ? static_cast<float*>(mptr(stats)) : nullptr, a.dtype, n.batch, n.queries, n.keys, n.heads,
                                          n.kv_heads, n.dim, a.scale, mptr(work), stream()));
    return {out, stats, rest};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cross_attention_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                        const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& mask,
                                                        c10::optional<double> scale)
{
    AttentionResult r = attention_forward(q, k, v, lengths, mask, scale, true);
    return {r.out, r.stats, r.rest};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor>
cross_attention_backward_cuda(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& out,
                              const at::Tensor& stats, const at::Tensor& rest, const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& mask,
                              c10::optional<double> scale)
{
    constexpr const char* op = "cross_attention_backward";
    TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(q.device());
    const AttentionArrays a(q, k, v, lengths, mask, scale, op);
    const AttentionSizes& n = a.n;
    check_like(dout, q, op, "dout");
    check_like(out, q, op, "out");
    TORCH_CHECK(dout.sizes() == q.sizes() && out.sizes() == q.sizes(), op, ": dout and out must be ", q.sizes(), ", got ", dout.sizes(), " and ",
                out.sizes());
    TORCH_CHECK(stats.is_cuda() && stats.device() == q.device() && stats.scalar_type() == at::kFloat && n.kv_heads > 0
                    && stats.numel() == 2 * n.batch * n.queries * n.heads,
                op, ": stats must be what cross_attention returned");
    TORCH_CHECK(rest.is_cuda() && rest.device() == q.device() && rest.scalar_type() == at::kChar && (rest.numel() == 0 || rest.sizes() == q.sizes()),
                op, ": rest must be what cross_attention returned");
    const at::Tensor dc = dout.contiguous();
    const at::Tensor oc = out.contiguous();
    const at::Tensor sc = stats.contiguous();
    const at::Tensor rc = rest.contiguous();
    at::Tensor dq = at::empty(q.sizes(), q.options());
    at::Tensor dk = at::empty(k.sizes(), q.options());
    at::Tensor dv = at::empty(v.sizes(), q.options());
    size_t count = 0;
    check_status(spectral_cross_attention_backward_workspace(cptr(dc), cptr(a.q), cptr(a.k), cptr(a.v), a.strides, a.dtype, n.batch, n.queries, n.keys,
                                                             n.heads, n.kv_heads, n.dim, &count));
    at::Tensor work = workspace(count, q);
    check_status(spectral_cross_attention_backward(cptr(dc), cptr(a.q), cptr(a.k), cptr(a.v), a.strides, cptr(oc), rc.numel() > 0 ? cptr(rc) : nullptr, fptr(sc), a.lengths_ptr(),
                                                   a.lengths64(), a.mask_ptr(), mptr(dq), mptr(dk), mptr(dv), a.dtype, n.batch, n.queries, n.keys,
                                                   n.heads, n.kv_heads, n.dim, a.scale, mptr(work), stream()));
    return {dq, dk, dv};
}

// --- the same with gradients: what spectral.nn calls ----------------------------------------------
// Functions of torch's autograd engine in C++ (the Python class's bookkeeping took longer than the
// kernels of a small layer). Each keeps only its input for the backward pass, in 8 bits if asked.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients of gradients are not computed: asking for them is an error, not a silent zero. In a backward pass
// with create_graph, the results depend on the forward pass's inputs and on the upstream gradient; they get
// this node as their history, whose edges lead to all of those, so that differentiating them raises
// wherever the answer would need it, and using their values alone does not.
struct NotDifferentiable : torch::autograd::Node {
    explicit NotDifferentiable(std::string name) : op(std::move(name)) {}
    variable_list apply(variable_list&&) override { TORCH_CHECK(false, op, ": the backward pass is not differentiable itself"); }
    std::string op;
};

// An upstream gradient that is a leaf can only ask for gradients of gradients: refused at once.
void check_once(const variable_list& grads, const char* op)
{
    for (const at::Tensor& g : grads) {
        TORCH_CHECK(!(at::GradMode::is_enabled() && g.defined() && g.requires_grad() && !g.grad_fn()), op,
                    ": the backward pass is not differentiable itself");
    }
}

// The end of a backward pass: `results` with the history above if there is to be one. `create_graph` is grad mode
// as the pass was entered.
variable_list finish_once(bool create_graph, const char* op, const variable_list& grads, variable_list results)
{
    if (!create_graph) {
        return results;
    }
    torch::autograd::edge_list edges;
    for (const torch::autograd::Edge& e : torch::autograd::get_current_node()->next_edges()) {
        if (e.is_valid()) {
            edges.push_back(e);
        }
    }
    for (const at::Tensor& g : grads) {
        if (g.defined() && g.requires_grad()) {
            edges.push_back(torch::autograd::impl::gradient_edge(g));
        }
    }
    const auto node = std::make_shared<NotDifferentiable>(op);
    node->set_next_edges(std::move(edges));
    for (at::Tensor& t : results) {
        if (t.defined()) {
            torch::autograd::impl::set_gradient_edge(t, {node, node->add_input_metadata(t)});
        }
    }
    return results;
}

bool wants_grad(std::initializer_list<const at::Tensor*> tensors)
{
    if (!at::GradMode::is_enabled()) {
        return false;
    }
    for (const at::Tensor* t : tensors) {
        if (t->defined() && t->requires_grad()) {
            return true;
        }
    }
    return false;
}

// Nor are forward-mode derivatives: a result without its tangent would be a silent zero too. (These do not depend
// on requires_grad or on grad mode.)
void check_no_tangent(const char* op, std::initializer_list<const at::Tensor*> tensors)
{
    for (const at::Tensor* t : tensors) {
        TORCH_CHECK(!(t->defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined()), op,
                    ": forward-mode derivatives are not computed");
    }
}

c10::optional<at::Tensor> optional_of(const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; }

struct GroupNormActFunction : torch::autograd::Function<GroupNormActFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                              const c10::optional<at::Tensor>& bias, int64_t groups, double eps, std::string activation,
                              bool checkpoint8)
    {
        at::AutoDispatchBelowAutograd guard;
        const NormResult r = norm_forward(x, groups, weight, bias, eps, activation, checkpoint8, true);
        const at::Tensor w = weight.value_or(at::Tensor());
        const at::Tensor b = bias.value_or(at::Tensor());
        ctx->save_for_backward(checkpoint8 ? variable_list{w, b, r.stats, r.codes, r.scales}
                                           : variable_list{w, b, r.stats, x});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["activation"] = activation;
        return r.y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_once(grads, "group_norm_act");
        const bool create_graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        const variable_list kept = ctx->get_saved_variables();
        const bool packed = kept.size() == 5;
        const std::string activation = ctx->saved_data["activation"].toStringRef();
        const at::Tensor& stats = kept[2];
        const float* mean = fptr(stats);
        auto [dx, dweight, dbias] = norm_backward(
            grads[0], packed ? c10::nullopt : optional_of(kept[3]), packed ? optional_of(kept[3]) : c10::nullopt,
            packed ? optional_of(kept[4]) : c10::nullopt, optional_of(kept[0]), optional_of(kept[1]), mean,
            mean == nullptr ? nullptr : mean + stats.numel() / 2, ctx->saved_data["groups"].toInt(), activation);
        const at::Tensor none;
        return finish_once(create_graph, "group_norm_act", grads,
                           {dx, kept[0].defined() ? dweight : none, kept[1].defined() ? dbias : none, none, none, none, none});
    }
};

at::Tensor group_norm_act_layer_cuda(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight,
                                     const c10::optional<at::Tensor>& bias, double eps, c10::string_view activation, bool)
{
    return norm_forward(x, groups, weight, bias, eps, activation, false, false).y;
}

at::Tensor group_norm_act_layer_autograd(const at::Tensor& x, int64_t groups, const c10::optional<at::Tensor>& weight,
                                         const c10::optional<at::Tensor>& bias, double eps, c10::string_view activation,
                                         bool checkpoint8)
{
    const at::Tensor w = weight.value_or(at::Tensor());
    const at::Tensor b = bias.value_or(at::Tensor());
    check_no_tangent("group_norm_act", {&x, &w, &b});
    if (wants_grad({&x, &w, &b})) {
        return GroupNormActFunction::apply(x, weight, bias, groups, eps, std::string(activation.data(), activation.size()), checkpoint8);
    }
    at::AutoDispatchBelowAutograd guard;
    return group_norm_act_layer_cuda(x, groups, weight, bias, eps, activation, checkpoint8);
}

struct GatedMlpFunction : torch::autograd::Function<GatedMlpFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up,
                              const at::Tensor& w_down, std::string activation, bool checkpoint8)
    {
        at::AutoDispatchBelowAutograd guard;
        const at::Tensor y = gated_mlp_cuda(x, w_gate, w_up, w_down, activation);
        variable_list kept{w_gate, w_up, w_down};
        if (checkpoint8) {
            auto [codes, scales] = pack8_cuda(x);
            kept.push_back(codes);
            kept.push_back(scales);
        } else {
            kept.push_back(x);
        }
        ctx->save_for_backward(std::move(kept));
        ctx->saved_data["activation"] = activation;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_once(grads, "gated_mlp");
        const bool create_graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        const variable_list kept = ctx->get_saved_variables();
        const bool packed = kept.size() == 5;
        const std::string activation = ctx->saved_data["activation"].toStringRef();
        auto [dx, dwg, dwu, dwd] = gated_mlp_backward_cuda(
            grads[0], packed ? c10::nullopt : optional_of(kept[3]), packed ? optional_of(kept[3]) : c10::nullopt,
            packed ? optional_of(kept[4]) : c10::nullopt, kept[0], kept[1], kept[2], activation);
        return finish_once(create_graph, "gated_mlp", grads, {dx, dwg, dwu, dwd, at::Tensor(), at::Tensor()});
    }
};

at::Tensor gated_mlp_layer_cuda(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up,
                                const at::Tensor& w_down, c10::string_view activation, bool)
{
    return gated_mlp_cuda(x, w_gate, w_up, w_down, activation);
}

at::Tensor gated_mlp_layer_autograd(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up,
                                    const at::Tensor& w_down, c10::string_view activation, bool checkpoint8)
{
    check_no_tangent("gated_mlp", {&x, &w_gate, &w_up, &w_down});
    if (wants_grad({&x, &w_gate, &w_up, &w_down})) {
        return GatedMlpFunction::apply(x, w_gate, w_up, w_down, std::string(activation.data(), activation.size()), checkpoint8);
    }
    at::AutoDispatchBelowAutograd guard;
    return gated_mlp_layer_cuda(x, w_gate, w_up, w_down, activation, checkpoint8);
}

struct QkNormRotaryFunction : torch::autograd::Function<QkNormRotaryFunction> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const c10::optional<at::Tensor>& k,
                                 const c10::optional<at::Tensor>& q_weight, const c10::optional<at::Tensor>& k_weight,
                                 const c10::optional<at::Tensor>& q_positions, const c10::optional<at::Tensor>& k_positions, double eps,
                                 double theta, int64_t rotated, std::string pairs)
    {
        at::AutoDispatchBelowAutograd guard;
        variable_list out = qk_norm_rotary_cuda(q, k, q_weight, k_weight, q_positions, k_positions, eps, theta, rotated, pairs);
        const at::Tensor none;
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({q, k.value_or(none), q_weight.value_or(none), k_weight.value_or(none), q_positions.value_or(none),
                                k_positions.value_or(none)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["theta"] = theta;
        ctx->saved_data["rotated"] = rotated;
        ctx->saved_data["pairs"] = pairs;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_once(grads, "qk_norm_rotary");
        const bool create_graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        const variable_list kept = ctx->get_saved_variables();
        variable_list x{kept[0]};
        if (kept[1].defined()) {
            x.push_back(kept[1]);
        }
        variable_list d = rotary_backward(grads, x, two(optional_of(kept[2]), optional_of(kept[3])), two(optional_of(kept[4]), optional_of(kept[5])),
                                          {ctx->saved_data["rotated"].toInt(), ctx->saved_data["eps"].toDouble(),
                                           ctx->saved_data["theta"].toDouble(), ctx->saved_data["pairs"].toStringRef()});
        const at::Tensor none;
        const bool both = x.size() == 2;
        return finish_once(create_graph, "qk_norm_rotary", grads,
                           {d[0], both ? d[1] : none, both ? d[2] : d[1], both ? d[3] : none, none, none, none, none, none, none});
    }
};

variable_list qk_norm_rotary_layer_autograd(const at::Tensor& q, const c10::optional<at::Tensor>& k, const c10::optional<at::Tensor>& q_weight,
                                            const c10::optional<at::Tensor>& k_weight, const c10::optional<at::Tensor>& q_positions,
                                            const c10::optional<at::Tensor>& k_positions, double eps, double theta, int64_t rotated,
                                            c10::string_view pairs)
{
    const at::Tensor kt = k.value_or(at::Tensor());
    const at::Tensor qw = q_weight.value_or(at::Tensor());
    const at::Tensor kw = k_weight.value_or(at::Tensor());
    const at::Tensor qp = q_positions.value_or(at::Tensor());
    const at::Tensor kp = k_positions.value_or(at::Tensor());
    check_no_tangent("qk_norm_rotary", {&q, &kt, &qw, &kw, &qp, &kp});
    TORCH_CHECK(!wants_grad({&qp, &kp}), "qk_norm_rotary: positions have no gradient; detach them");
    // Without keys their weight has no part in the call, so no gradient either.
    if (wants_grad({&q, &kt, &qw}) || (kt.defined() && wants_grad({&kw}))) {
        return QkNormRotaryFunction::apply(q, k, q_weight, k_weight, q_positions, k_positions, eps, theta, rotated,
                                           std::string(pairs.data(), pairs.size()));
    }
    at::AutoDispatchBelowAutograd guard;
    return qk_norm_rotary_cuda(q, k, q_weight, k_weight, q_positions, k_positions, eps, theta, rotated, pairs);
}

struct CrossAttentionFunction : torch::autograd::Function<CrossAttentionFunction> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& mask, c10::optional<double> scale)
    {
        at::AutoDispatchBelowAutograd guard;
        const AttentionResult r = attention_forward(q, k, v, lengths, mask, scale, true);
        const at::Tensor none;
        ctx->save_for_backward({q, k, v, r.out, r.stats, r.rest, lengths.value_or(none), mask.value_or(none)});
        ctx->saved_data["scale"] = scale;
        return r.out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_once(grads, "cross_attention");
        const bool create_graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        const variable_list kept = ctx->get_saved_variables();
        auto [dq, dk, dv] = cross_attention_backward_cuda(grads[0], kept[0], kept[1], kept[2], kept[3], kept[4], kept[5], optional_of(kept[6]),
                                                          optional_of(kept[7]), ctx->saved_data["scale"].toOptional<double>());
        const at::Tensor none;
        return finish_once(create_graph, "cross_attention", grads, {dq, dk, dv, none, none, none});
    }
};

at::Tensor cross_attention_layer_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& lengths,
                                      const c10::optional<at::Tensor>& mask, c10::optional<double> scale)
{
    return attention_forward(q, k, v, lengths, mask, scale, false).out;
}

at::Tensor cross_attention_layer_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& lengths,
                                          const c10::optional<at::Tensor>& mask, c10::optional<double> scale)
{
    check_no_tangent("cross_attention", {&q, &k, &v});
    if (wants_grad({&q, &k, &v})) {
        return CrossAttentionFunction::apply(q, k, v, lengths, mask, scale);
    }
    at::AutoDispatchBelowAutograd guard;
    return cross_attention_layer_cuda(q, k, v, lengths, mask, scale);
}

// spectral._C.fft_impls(): the registry's names, in order, as a tuple of str.
PyObject* py_fft_impls(PyObject*, PyObject*)
{
    const int count = spectral_impl_count();
    PyObject* names = PyTuple_New(count);
    if (names == nullptr) {
        return nullptr;
    }
    for (int i = 0; i < count; ++i) {
        PyObject* name = PyUnicode_FromString(spectral_impl_name(i));
        if (name == nullptr) {
            Py_DECREF(names);
            return nullptr;
        }
        PyTuple_SET_ITEM(names, i, name);
    }
    return names;
}

PyMethodDef module_methods[] = {
    {"fft_impls", py_fft_impls, METH_NOARGS, "Names of the FFT implementations, in order."},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

TORCH_LIBRARY(spectral, m)
{
    m.def("scale(Tensor x, float alpha) -> Tensor");
    m.def("fft_c2c(Tensor x, bool inverse=False, str impl=\"naive\") -> Tensor");
    m.def("fft_r2c(Tensor x, str impl=\"naive\") -> Tensor");
    m.def("fft_c2r(Tensor x, int n, str impl=\"naive\") -> Tensor");
    m.def("fft2_c2c(Tensor x, bool inverse=False, str impl=\"naive\", str columns=\"auto\")"
          " -> Tensor");
    m.def("fft2_r2c(Tensor x, str impl=\"naive\", str columns=\"auto\") -> Tensor");
    m.def("fft2_c2r(Tensor x, int n2, str impl=\"naive\", str columns=\"auto\") -> Tensor");
    m.def("fft_c2c_pruned(Tensor x, int n, int keep, bool inverse=False, str impl=\"naive\")"
          " -> Tensor");
    m.def("rfft2_modes(Tensor x, int m1, int m2, str impl=\"naive\") -> Tensor");
    m.def("irfft2_modes(Tensor modes, int n1, int n2, str impl=\"naive\") -> Tensor");
    m.def("mode_contract(Tensor x, Tensor w) -> Tensor");
    m.def("spectrum_frames(Tensor x, int nfft, Tensor? window=None, str impl=\"stockham_r8\") -> Tensor");
    m.def("fir_overlap_save(Tensor x, Tensor taps_spectrum, int taps, int nfft, str impl=\"stockham_r8\")"
          " -> Tensor");
    m.def("flow_stage(Tensor x, Tensor w, Tensor(a!) f0, Tensor(b!) out, Tensor derive, Tensor forcing, Tensor mask,"
          " Tensor explicit_factor, Tensor implicit_factor, Tensor(c!) work, int n, int m, float dt, int stage,"
          " str impl=\"stockham_r8\") -> ()");
    m.def("pack8(Tensor x) -> (Tensor, Tensor)");
    m.def("unpack8(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("group_norm_act(Tensor x, int groups, Tensor? weight=None, Tensor? bias=None, float eps=1e-5,"
          " str activation=\"none\", bool keep8=False) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("group_norm_act_backward(Tensor dy, Tensor? x, Tensor? codes, Tensor? scales, Tensor? weight, Tensor? bias,"
          " Tensor mean, Tensor rstd, int groups, str activation) -> (Tensor, Tensor, Tensor)");
    m.def("gated_mlp(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, str activation=\"silu\") -> Tensor");
    m.def("gated_mlp_backward(Tensor dy, Tensor? x, Tensor? codes, Tensor? scales, Tensor w_gate, Tensor w_up,"
          " Tensor w_down, str activation) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("group_norm_act_layer(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, str activation,"
          " bool checkpoint8) -> Tensor");
    m.def("gated_mlp_layer(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, str activation, bool checkpoint8)"
          " -> Tensor");
    m.def("qk_norm_rotary_layer(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, Tensor? q_positions,"
          " Tensor? k_positions, float eps, float theta, int rotated, str pairs) -> Tensor[]");
    m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? lengths=None, Tensor? mask=None, float? scale=None)"
          " -> (Tensor, Tensor, Tensor)");
    m.def("cross_attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor stats, Tensor rest,"
          " Tensor? lengths=None, Tensor? mask=None, float? scale=None) -> (Tensor, Tensor, Tensor)");
    m.def("cross_attention_layer(Tensor q, Tensor k, Tensor v, Tensor? lengths, Tensor? mask, float? scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(spectral, CUDA, m)
{
    m.impl("scale", &scale_cuda);
    m.impl("fft_c2c", &fft_c2c_cuda);
    m.impl("fft_r2c", &fft_r2c_cuda);
    m.impl("fft_c2r", &fft_c2r_cuda);
    m.impl("fft2_c2c", &fft2_c2c_cuda);
    m.impl("fft2_r2c", &fft2_r2c_cuda);
    m.impl("fft2_c2r", &fft2_c2r_cuda);
    m.impl("fft_c2c_pruned", &fft_c2c_pruned_cuda);
    m.impl("rfft2_modes", &rfft2_modes_cuda);
    m.impl("irfft2_modes", &irfft2_modes_cuda);
    m.impl("mode_contract", &mode_contract_cuda);
    m.impl("spectrum_frames", &spectrum_frames_cuda);
    m.impl("fir_overlap_save", &fir_overlap_save_cuda);
    m.impl("flow_stage", &flow_stage_cuda);
    m.impl("pack8", &pack8_cuda);
    m.impl("unpack8", &unpack8_cuda);
    m.impl("group_norm_act", &group_norm_act_cuda);
    m.impl("group_norm_act_backward", &group_norm_act_backward_cuda);
    m.impl("gated_mlp", &gated_mlp_cuda);
    m.impl("gated_mlp_backward", &gated_mlp_backward_cuda);
    m.impl("group_norm_act_layer", &group_norm_act_layer_cuda);
    m.impl("gated_mlp_layer", &gated_mlp_layer_cuda);
    m.impl("qk_norm_rotary_layer", &qk_norm_rotary_cuda);
    m.impl("cross_attention", &cross_attention_cuda);
    m.impl("cross_attention_backward", &cross_attention_backward_cuda);
    m.impl("cross_attention_layer", &cross_attention_layer_cuda);
}

TORCH_LIBRARY_IMPL(spectral, AutogradCUDA, m)
{
    m.impl("group_norm_act_layer", &group_norm_act_layer_autograd);
    m.impl("gated_mlp_layer", &gated_mlp_layer_autograd);
    m.impl("qk_norm_rotary_layer", &qk_norm_rotary_layer_autograd);
    m.impl("cross_attention_layer", &cross_attention_layer_autograd);
}

PyMODINIT_FUNC PyInit__C(void)
{
    static PyModuleDef module_def = {
        PyModuleDef_HEAD_INIT, "_C", nullptr, -1, module_methods,
    };
    return PyModule_Create(&module_def);
}
