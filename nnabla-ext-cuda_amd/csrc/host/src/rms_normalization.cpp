// RMSNormalizationHip<T> over nblahip.
#include <nbla/hip/function/rms_normalization.hpp>
#include <nbla/variable.hpp>

#include <type_traits>

namespace nbla {

template <typename T>
void RMSNormalizationHip<T>::setup_impl(const Variables &inputs, const Variables &outputs) {
  const size_t n_in = no_scale_ ? 1 : 2;
  NBLA_CHECK(inputs.size() == n_in, error_code::value,
             "RMSNormalization expects %zu inputs, given %zu.", n_in, inputs.size());
  NBLA_CHECK(outputs.size() == 1, error_code::value, "RMSNormalization has 1 output.");
  const Shape_t shape = inputs[0]->shape();
  rows_and_columns("RMSNormalization", shape, batch_axis_, rows_, cols_);
  NBLA_CHECK(no_scale_ || inputs[1]->size() == cols_, error_code::value,
             "gamma must have %lld elements.", static_cast<long long>(cols_));
  outputs[0]->reshape(shape, true);
  ms_.reshape(Shape_t{rows_}, true);
  if (format8_) x8_.reshape(rows_, cols_);
  hip_set_device(device_); // argument errors above are reported without a device
  workspace_bytes_ = nblahip_rms_bwd_workspace_bytes(rows_, cols_, HipDtype<T>::code);
  workspace_.reshape(Shape_t{static_cast<Size_t>((workspace_bytes_ + 3) / 4)}, true);
  if (std::is_same<T, Half>::value)
    stage_.reshape(Shape_t{ParamStage::capacity_for({cols_, cols_})}, true);
}

template <typename T>
void RMSNormalizationHip<T>::forward_impl(const Variables &inputs, const Variables &outputs) {
  hip_set_device(device_);
  const T *x = inputs[0]->get_data_pointer<T>(this->ctx_);
  ParamStage st;
  st.begin(this->ctx_, std::is_same<T, Half>::value, &stage_);
  const float *gamma = no_scale_ ? nullptr : st.in(inputs[1]);
  T *y = outputs[0]->cast_data_and_get_pointer<T>(this->ctx_, true);
  float *ms = ms_.cast_data_and_get_pointer<float>(this->ctx_, true);
  st.load();
  if (format8_) {
    // the step's forward with its first norm alone, which also writes the copy
    NBLA_HIP_CHECK(nblahip_resnorm_fwd(
        x, nullptr, nullptr, NBLAHIP_GATE_NONE, 0, gamma, nullptr, nullptr, nullptr, y, nullptr, nullptr,
        ms, nullptr, nullptr, x8_.codes(this->ctx_), x8_.scales(this->ctx_), nullptr, nullptr, format8_,
        rows_, cols_, 1.f, 1.f, eps_, NBLAHIP_NORM_RMS, 1, 0, HipDtype<T>::code, nullptr));
  } else {
    NBLA_HIP_CHECK(nblahip_rms_fwd(x, gamma, y, ms, rows_, cols_, eps_, HipDtype<T>::code, nullptr));
  }
}

template <typename T>
void RMSNormalizationHip<T>::backward_impl(const Variables &inputs, const Variables &outputs,
                                           const vector<bool> &propagate_down,
                                           const vector<bool> &accum) {
  hip_set_device(device_);
  const bool pd_gamma = !no_scale_ && propagate_down[1];
  if (!(propagate_down[0] || pd_gamma)) return;
  ParamStage st;
  st.begin(this->ctx_, std::is_same<T, Half>::value, &stage_);
  const float *gamma = no_scale_ ? nullptr : st.in(inputs[1]);
  const void *x = nullptr;
  const uint8_t *scales = nullptr;
  if (format8_) {
    x = x8_.kept_codes(this->ctx_);
    scales = x8_.kept_scales(this->ctx_);
  } else {
    x = inputs[0]->get_data_pointer<T>(this->ctx_);
  }
  const T *dy = outputs[0]->get_grad_pointer<T>(this->ctx_);
  const float *ms = ms_.get_data_pointer<float>(this->ctx_);
  T *dx = !propagate_down[0] ? nullptr
                             : inputs[0]->cast_grad_and_get_pointer<T>(this->ctx_, !accum[0]);
  float *dgamma = !pd_gamma ? nullptr : st.out(inputs[1], accum[1], true);
  st.load();
  float *ws = workspace_.cast_data_and_get_pointer<float>(this->ctx_, true);
  NBLA_HIP_CHECK(nblahip_rms_bwd(x, scales, format8_, dy, gamma, ms, dx, dgamma,
                                 propagate_down[0] && accum[0], pd_gamma && accum[1], rows_, cols_, eps_,
                                 HipDtype<T>::code, ws, workspace_bytes_, nullptr));
  st.store();
  workspace_.data()->array()->clear();
}

template class RMSNormalizationHip<float>;
template class RMSNormalizationHip<Half>;
} // namespace nbla
