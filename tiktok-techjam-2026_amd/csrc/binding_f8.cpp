// Python calls of the 8-bit operators (module tjkernels._f8): each checks its
// tensors and launches on the current stream of their device.
//
// On a call for a few tokens the host's share is the longer one.  Through
// ctypes, with the checks in Python, add_rmsnorm of 8 x 2048 took 8.1 us per call
// and gemm_f8 of 8 x 8192 x 2048 7.8; from here 3.5 and 6.1 (its kernel's time), of
// which 0.25 are the checks and the rest the launch.

#include "binding.h"

namespace {

// The fp32 scales of a quantised matrix: at least rows x ceil(cols / 128).
struct Scales {
  float* data = nullptr;
  int64_t ld = 0;
};

Scales block_scales(const at::Tensor* t, int64_t rows, int64_t cols, const char* name) {
  const int64_t need = (cols + 127) / 128;
  if (t && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) >= rows && t->size(1) >= need &&
      (t->stride(1) == 1 || t->size(1) == 1)) {
    const int64_t ld = t->size(0) > 1 ? t->stride(0) : need;
    if (ld >= need) return {static_cast<float*>(t->data_ptr()), ld};
  }
  refuse("%s must be a float32 [%lld, %lld] matrix with unit column stride", name, (long long)rows, (long long)need);
}

// (res, delta, gamma, eps, out, res_out, scales)
PyObject* add_rmsnorm(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 7, [&] {
    const at::Tensor &res_t = tensor(args[0], "res"), &gamma_t = tensor(args[2], "gamma"), &out_t = tensor(args[4], "out");
    const at::Tensor *delta_t = tensor_or_none(args[1], "delta"), *res_out_t = tensor_or_none(args[5], "res_out"),
                     *scales_t = tensor_or_none(args[6], "scales");
    const double eps = PyFloat_AsDouble(args[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw python_error();
    const Matrix res = matrix(res_t, "res");
    auto like = [&](const at::Tensor& t, const char* name) {
      const Matrix m = matrix(t, name);
      if (m.rows < res.rows || m.cols != res.cols)
        refuse("%s must be [%lld, %lld], got [%lld, %lld]", name, (long long)res.rows, (long long)res.cols,
               (long long)m.rows, (long long)m.cols);
      return m;
    };
    const Matrix out = like(out_t, "out");
    Matrix delta{}, res_out{};
    if (delta_t) delta = like(*delta_t, "delta");
    if (res_out_t) res_out = like(*res_out_t, "res_out");
    const float* const gamma = static_cast<const float*>(vector_of(gamma_t, res.cols, at::kFloat, "gamma"));
    Scales scales;
    if (out.dtype == TJK_E4M3) scales = block_scales(scales_t, res.rows, res.cols, "scales");
    else if (scales_t) refuse("scales belong to a float8_e4m3fn out");
    const c10::DeviceIndex device = one_device({&res_t, delta_t, &gamma_t, &out_t, res_out_t, scales_t});
    return launch(device, "tjk_add_rmsnorm", [&](void* stream) {
      return tjk_add_rmsnorm(res.data, res.dtype, res.ld, delta.data, delta.dtype, delta.ld, res_out.data, res_out.dtype,
                             res_out.ld, out.data, out.dtype, out.ld, scales.data, scales.ld, gamma, res.rows, res.cols,
                             (float)eps, stream);
    });
  });
}

// (x, out, scales, block_rows)
PyObject* quantize_f8(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 4, [&] {
    const at::Tensor &x_t = tensor(args[0], "x"), &out_t = tensor(args[1], "out"), &scales_t = tensor(args[2], "scales");
    const int block_rows = (int)integer(args[3], "block_rows");
    const Matrix x = matrix(x_t, "x"), out = matrix(out_t, "out");
    if (out.dtype != TJK_E4M3 || out.rows < x.rows || out.cols != x.cols)
      refuse("out must be a float8_e4m3fn [%lld, %lld] matrix", (long long)x.rows, (long long)x.cols);
    if (block_rows != 1 && block_rows != 128) refuse("block_rows must be 1 or 128, got %d", block_rows);
    const Scales scales = block_scales(&scales_t, (x.rows + block_rows - 1) / block_rows, x.cols, "scales");
    const c10::DeviceIndex device = one_device({&x_t, &out_t, &scales_t});
    return launch(device, "tjk_quantize_f8", [&](void* stream) {
      return tjk_quantize_f8(x.data, x.dtype, x.ld, out.data, out.ld, scales.data, scales.ld, x.rows, x.cols, block_rows,
                             stream);
    });
  });
}

// (a, a_scales, w, w_scales, bias, out, epilogue, out_scales, plan)
PyObject* gemm_f8(PyObject*, PyObject* const* args, Py_ssize_t given) {
  return guarded(given, 9, [&] {
    const at::Tensor &a_t = tensor(args[0], "a"), &as_t = tensor(args[1], "a_scales"), &w_t = tensor(args[2], "w"),
                     &ws_t = tensor(args[3], "w_scales"), &out_t = tensor(args[5], "out");
    const at::Tensor *bias_t = tensor_or_none(args[4], "bias"), *cs_t = tensor_or_none(args[7], "out_scales");
    const int epilogue = (int)integer(args[6], "epilogue"), plan = (int)integer(args[8], "plan");
    const Matrix a = matrix(a_t, "a"), w = matrix(w_t, "w"), out = matrix(out_t, "out");
    if (a.dtype != TJK_E4M3 || w.dtype != TJK_E4M3) refuse("gemm_f8 operands must be float8_e4m3fn");
    if (a.cols != w.cols || out.rows != a.rows || out.cols != w.rows)
      refuse("gemm_f8 shape mismatch a[%lld, %lld] w[%lld, %lld] out[%lld, %lld]", (long long)a.rows, (long long)a.cols,
             (long long)w.rows, (long long)w.cols, (long long)out.rows, (long long)out.cols);
    const Scales as = block_scales(&as_t, a.rows, a.cols, "a_scales");
    const Scales ws = block_scales(&ws_t, (w.rows + 127) / 128, a.cols, "w_scales");
    Scales cs;
    if (out.dtype == TJK_E4M3) cs = block_scales(cs_t, out.rows, out.cols, "out_scales");
    else if (out.dtype == TJK_F32) refuse("gemm_f8 out must be float16, bfloat16 or float8_e4m3fn");
    else if (cs_t) refuse("out_scales belong to a float8_e4m3fn out");
    const void* bias = nullptr;
    if (bias_t) bias = vector_of(*bias_t, out.cols, out.dtype == TJK_E4M3 ? at::kFloat : out_t.scalar_type(), "bias");
    const c10::DeviceIndex device = one_device({&a_t, &as_t, &w_t, &ws_t, bias_t, &out_t, cs_t});
    return launch(device, "tjk_gemm_f8", [&](void* stream) {
      return tjk_gemm_f8(a.data, a.ld, as.data, as.ld, w.data, w.ld, ws.data, ws.ld, bias, out.data, out.dtype, out.ld,
                         cs.data, cs.ld, out.rows, out.cols, a.cols, epilogue, plan, stream);
    });
  });
}

PyMethodDef methods[] = {
    {"add_rmsnorm", (PyCFunction)(void*)add_rmsnorm, METH_FASTCALL, nullptr},
    {"quantize_f8", (PyCFunction)(void*)quantize_f8, METH_FASTCALL, nullptr},
    {"gemm_f8", (PyCFunction)(void*)gemm_f8, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_f8", "Calls of the 8-bit operators.", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__f8(void) { return make_module(&module_def); }
