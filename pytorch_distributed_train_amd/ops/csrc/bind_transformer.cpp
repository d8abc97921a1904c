// Python binding of the transformer-training operators (AdamW).
// Arguments are checked here, before a launch: a kernel's bounds rest on them.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <hip/hip_runtime_api.h>

extern "C" {
void pdta_adamw(float*, const float*, void*, void*, float*, float*, long,
                long*, float, const float*, double, double, float, float,
                const unsigned char*, float, unsigned, void*, hipStream_t);
}

namespace {

// the current stream of the current device (call under a DeviceGuard)
hipStream_t cur_stream() {
  return (hipStream_t)at::hip::getCurrentHIPStreamMasqueradingAsCUDA()
      .stream();
}

void launched(const char* what) {
  hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": launch failed: ",
              hipGetErrorString(e));
}

// a flat array on `like`'s device that the 16-byte accesses may walk
void check_flat(const char* name, const at::Tensor& t, const at::Tensor& like,
                at::ScalarType dtype, long numel) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on ",
              like.device(), ", is on ", t.device());
  TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", is ",
              t.scalar_type());
  TORCH_CHECK(t.is_contiguous() && t.numel() == numel, name,
              " must be contiguous with ", numel, " elements");
  TORCH_CHECK((uintptr_t)t.data_ptr() % 16 == 0, name,
              " must start at a multiple of 16 bytes");
}

void adamw_step(at::Tensor p, at::Tensor g, at::Tensor m, at::Tensor v,
                at::Tensor step, double lr, c10::optional<at::Tensor> lr_dev,
                double beta1, double beta2, double eps, double weight_decay,
                c10::optional<at::Tensor> decay, double grad_scale,
                c10::optional<at::Tensor> m_scale,
                c10::optional<at::Tensor> v_scale, int64_t seed) {
  TORCH_CHECK(p.is_cuda(), "p must be on GPU");
  c10::DeviceGuard guard(p.device());
  long n = p.numel();
  TORCH_CHECK(n % 64 == 0, "p must have a multiple of 64 elements, has ", n);
  check_flat("p", p, p, at::kFloat, n);
  check_flat("g", g, p, at::kFloat, n);
  bool eight = m_scale.has_value();
  TORCH_CHECK(eight == v_scale.has_value(),
              "m_scale and v_scale come together");
  auto st = eight ? at::kFloat8_e4m3fn : at::kFloat;
  check_flat("m", m, p, st, n);
  check_flat("v", v, p, st, n);
  if (eight) {
    check_flat("m_scale", *m_scale, p, at::kFloat, n / 64);
    check_flat("v_scale", *v_scale, p, at::kFloat, n / 64);
  }
  if (decay.has_value()) check_flat("decay", *decay, p, at::kByte, n / 64);
  TORCH_CHECK(step.device() == p.device() &&
                  step.scalar_type() == at::kLong && step.numel() == 1,
              "step must be one int64 on ", p.device());
  if (lr_dev.has_value())
    TORCH_CHECK(lr_dev->device() == p.device() &&
                    lr_dev->scalar_type() == at::kFloat &&
                    lr_dev->numel() == 1,
                "lr must be one float32 on ", p.device());
  auto hyp = at::empty({4}, p.options());
  pdta_adamw(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr(),
             v.data_ptr(), eight ? m_scale->data_ptr<float>() : nullptr,
             eight ? v_scale->data_ptr<float>() : nullptr, n,
             (long*)step.data_ptr<int64_t>(), (float)lr,
             lr_dev.has_value() ? lr_dev->data_ptr<float>() : nullptr, beta1,
             beta2, (float)eps, (float)weight_decay,
             decay.has_value() ? decay->data_ptr<uint8_t>() : nullptr,
             (float)grad_scale, (unsigned)seed, hyp.data_ptr(),
             cur_stream());
  launched("adamw_step");
}

}  // namespace

void bind_transformer(pybind11::module_& m) {
  m.def("adamw_step", &adamw_step, py::arg("p"), py::arg("g"), py::arg("m"),
        py::arg("v"), py::arg("step"), py::arg("lr"), py::arg("lr_dev"),
        py::arg("beta1"), py::arg("beta2"), py::arg("eps"),
        py::arg("weight_decay"), py::arg("decay"), py::arg("grad_scale"),
        py::arg("m_scale"), py::arg("v_scale"), py::arg("seed"));
}
