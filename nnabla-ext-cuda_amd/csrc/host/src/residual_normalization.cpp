// ResidualNormalizationHip<T> over nblahip.
#include <nbla/hip/function/residual_normalization.hpp>
#include <nbla/variable.hpp>

#include <type_traits>

namespace nbla {

template <typename T> void ResidualNormalizationHip<T>::place_inputs() {
  const bool layer = norm_ == "layer";
  int n = 1;
  auto take = [&](bool there) { return there ? n++ : -1; };
  i_res_ = take(residual_);
  i_gate_ = take(gate_);
  i_beta_post_ = take(post_ && layer && !no_bias_);
  i_gamma_post_ = take(post_ && !no_scale_);
  i_beta_pre_ = take(pre_ && layer && !no_bias_);
  i_gamma_pre_ = take(pre_ && !no_scale_);
  n_inputs_ = n;
}

template <typename T>
void ResidualNormalizationHip<T>::setup_impl(const Variables &inputs, const Variables &outputs) {
  NBLA_CHECK(norm_ == "rms" || norm_ == "layer", error_code::value,
             "norm must be \"rms\" or \"layer\" (given \"%s\").", norm_.c_str());
  NBLA_CHECK(post_ || pre_, error_code::value, "ResidualNormalization needs post, pre or both.");
  const bool layer = norm_ == "layer";
  NBLA_CHECK(static_cast<int>(inputs.size()) == n_inputs_, error_code::value,
             "ResidualNormalization expects %d inputs, given %zu.", n_inputs_, inputs.size());
  NBLA_CHECK(outputs.size() == (pre_ ? 2u : 1u), error_code::value,
             "ResidualNormalization has %d output(s).", pre_ ? 2 : 1);
  const Shape_t shape = inputs[0]->shape();
  rows_and_columns("ResidualNormalization", shape, batch_axis_, rows_, cols_);
  NBLA_CHECK(!residual_ || inputs[i_res_]->shape() == shape, error_code::value,
             "The residual must have the shape of x.");
  for (int i : {i_beta_post_, i_gamma_post_, i_beta_pre_, i_gamma_pre_})
    NBLA_CHECK(i < 0 || inputs[i]->size() == cols_, error_code::value,
               "beta/gamma must have %lld elements.", static_cast<long long>(cols_));
  gate_kind_ = NBLAHIP_GATE_NONE;
  gate_rows_ = 0;
  if (gate_) {
    const Size_t size = inputs[i_gate_]->size();
    if (inputs[i_gate_]->shape() == shape) {
      gate_kind_ = NBLAHIP_GATE_FULL;
    } else {
      NBLA_CHECK(cols_ > 0 && size > 0 && size % cols_ == 0 && rows_ % (size / cols_) == 0,
                 error_code::value,
                 "The gate must have the shape of x, or rows of %lld elements that divide its %lld rows.",
                 static_cast<long long>(cols_), static_cast<long long>(rows_));
      gate_kind_ = NBLAHIP_GATE_ROWS;
      gate_rows_ = size / cols_;
    }
  }
  outputs[0]->reshape(shape, true);
  if (pre_) outputs[1]->reshape(shape, true);
  for (Variable *v : {&mean_post_, &var_post_, &mean_pre_, &var_pre_}) v->reshape(Shape_t{rows_}, true);
  if (format8_) {
    x8_.reshape(rows_, cols_);
    h8_.reshape(rows_, cols_);
  }
  hip_set_device(device_); // argument errors above are reported without a device
  workspace_bytes_ = nblahip_resnorm_bwd_workspace_bytes(
      rows_, cols_, gate_kind_, gate_rows_, layer ? NBLAHIP_NORM_LAYER : NBLAHIP_NORM_RMS, post_, pre_,
      HipDtype<T>::code);
  workspace_.reshape(Shape_t{static_cast<Size_t>((workspace_bytes_ + 3) / 4)}, true);
  if (std::is_same<T, Half>::value) {
    const Size_t g = gate_rows_ * cols_;
    stage_.reshape(Shape_t{ParamStage::capacity_for({cols_, cols_, cols_, cols_, cols_, cols_, cols_,
                                                     cols_, g, g})},
                   true);
  }
}

template <typename T>
void ResidualNormalizationHip<T>::forward_impl(const Variables &inputs, const Variables &outputs) {
  hip_set_device(device_);
  const Context &ctx = this->ctx_;
  const bool layer = norm_ == "layer";
  ParamStage st;
  st.begin(ctx, std::is_same<T, Half>::value, &stage_);
  auto param = [&](int i) -> const float * { return i < 0 ? nullptr : st.in(inputs[i]); };
  const T *x = inputs[0]->get_data_pointer<T>(ctx);
  const T *res = residual_ ? inputs[i_res_]->get_data_pointer<T>(ctx) : nullptr;
  const void *gate = nullptr;
  if (gate_kind_ == NBLAHIP_GATE_FULL) gate = inputs[i_gate_]->get_data_pointer<T>(ctx);
  if (gate_kind_ == NBLAHIP_GATE_ROWS) gate = param(i_gate_);
  const float *bp = param(i_beta_post_), *gp = param(i_gamma_post_);
  const float *bn = param(i_beta_pre_), *gn = param(i_gamma_pre_);
  T *h = outputs[0]->cast_data_and_get_pointer<T>(ctx, true);
  T *y = pre_ ? outputs[1]->cast_data_and_get_pointer<T>(ctx, true) : nullptr;
  auto stat = [&](Variable &v, bool on) -> float * {
    return on ? v.cast_data_and_get_pointer<float>(ctx, true) : nullptr;
  };
  const bool keep_x = format8_ && reads_x(), keep_h = format8_ && pre_;
  st.load();
  NBLA_HIP_CHECK(nblahip_resnorm_fwd(
      x, res, gate, gate_kind_, gate_rows_, gp, bp, gn, bn, h, y, stat(mean_post_, post_ && layer),
      stat(var_post_, post_), stat(mean_pre_, pre_ && layer), stat(var_pre_, pre_),
      keep_x ? x8_.codes(ctx) : nullptr, keep_x ? x8_.scales(ctx) : nullptr,
      keep_h ? h8_.codes(ctx) : nullptr, keep_h ? h8_.scales(ctx) : nullptr, format8_, rows_, cols_,
      res_scale_, branch_scale_, eps_, layer ? NBLAHIP_NORM_LAYER : NBLAHIP_NORM_RMS, post_, pre_,
      HipDtype<T>::code, nullptr));
}

template <typename T>
void ResidualNormalizationHip<T>::backward_impl(const Variables &inputs, const Variables &outputs,
                                                const vector<bool> &propagate_down,
                                                const vector<bool> &accum) {
  hip_set_device(device_);
  // One pass writes each gradient to an array of its own.  A variable that is
  // two inputs (x and the residual, say) has one array for both gradients: the
  // second is added by a pass of its own.
  vector<bool> left(propagate_down);
  for (;;) {
    vector<bool> now(left.size(), false);
    bool any = false;
    for (size_t i = 0; i < left.size(); ++i) {
      if (!left[i]) continue;
      bool shared = false;
      for (size_t k = 0; k < i; ++k)
        shared = shared || (now[k] && inputs[k]->grad().get() == inputs[i]->grad().get());
      if (shared) continue;
      now[i] = any = true;
      left[i] = false;
    }
    if (!any) return;
    backward_pass(inputs, outputs, now, accum);
  }
}

template <typename T>
void ResidualNormalizationHip<T>::backward_pass(const Variables &inputs, const Variables &outputs,
                                                const vector<bool> &propagate_down,
                                                const vector<bool> &accum) {
  const Context &ctx = this->ctx_;
  const bool layer = norm_ == "layer";
  ParamStage st;
  st.begin(ctx, std::is_same<T, Half>::value, &stage_);
  auto param = [&](int i) -> const float * { return i < 0 ? nullptr : st.in(inputs[i]); };
  auto wanted = [&](int i) { return i >= 0 && propagate_down[i]; };
  const void *gate = nullptr;
  if (gate_kind_ == NBLAHIP_GATE_FULL) gate = inputs[i_gate_]->get_data_pointer<T>(ctx);
  if (gate_kind_ == NBLAHIP_GATE_ROWS) gate = param(i_gate_);
  const float *bp = gate_ ? param(i_beta_post_) : nullptr; // (for the gate's gradient alone)
  const float *gp = param(i_gamma_post_), *gn = param(i_gamma_pre_);
  const void *x = nullptr, *h = nullptr;
  const uint8_t *xs = nullptr, *hs = nullptr;
  if (format8_) {
    if (reads_x()) {
      x = x8_.kept_codes(ctx);
      xs = x8_.kept_scales(ctx);
    }
    if (pre_) {
      h = h8_.kept_codes(ctx);
      hs = h8_.kept_scales(ctx);
    }
  } else {
    if (reads_x()) x = inputs[0]->get_data_pointer<T>(ctx);
    if (pre_) h = outputs[0]->get_data_pointer<T>(ctx);
  }
  const T *dh = outputs[0]->get_grad_pointer<T>(ctx);
  const T *dy = pre_ ? outputs[1]->get_grad_pointer<T>(ctx) : nullptr;
  auto stat = [&](Variable &v, bool on) -> const float * {
    return on ? v.get_data_pointer<float>(ctx) : nullptr;
  };
  const float *mp = stat(mean_post_, post_ && layer), *vp = stat(var_post_, post_);
  const float *mn = stat(mean_pre_, pre_ && layer), *vn = stat(var_pre_, pre_);
  unsigned flags = 0;
  auto tensor = [&](int i, unsigned flag) -> T * {
    if (!wanted(i)) return nullptr;
    if (accum[i]) flags |= flag;
    return inputs[i]->cast_grad_and_get_pointer<T>(ctx, !accum[i]);
  };
  auto pgrad = [&](int i, unsigned flag) -> float * {
    if (!wanted(i)) return nullptr;
    if (accum[i]) flags |= flag;
    return st.out(inputs[i], accum[i], true);
  };
  T *dx = tensor(0, NBLAHIP_ACCUM_DX);
  T *dres = tensor(i_res_, NBLAHIP_ACCUM_DRES);
  void *dgate = gate_kind_ == NBLAHIP_GATE_FULL
                    ? static_cast<void *>(tensor(i_gate_, NBLAHIP_ACCUM_DGATE))
                    : static_cast<void *>(pgrad(i_gate_, NBLAHIP_ACCUM_DGATE));
  float *dgp = pgrad(i_gamma_post_, NBLAHIP_ACCUM_DGAMMA_POST);
  float *dbp = pgrad(i_beta_post_, NBLAHIP_ACCUM_DBETA_POST);
  float *dgn = pgrad(i_gamma_pre_, NBLAHIP_ACCUM_DGAMMA_PRE);
  float *dbn = pgrad(i_beta_pre_, NBLAHIP_ACCUM_DBETA_PRE);
  st.load();
  float *ws = workspace_.cast_data_and_get_pointer<float>(ctx, true);
  NBLA_HIP_CHECK(nblahip_resnorm_bwd(
      x, xs, h, hs, format8_, dh, dy, gate, gate_kind_, gate_rows_, gp, bp, gn, mp, vp, mn, vn, dx, dres,
      dgate, dgp, dbp, dgn, dbn, flags, rows_, cols_, res_scale_, branch_scale_, eps_,
      layer ? NBLAHIP_NORM_LAYER : NBLAHIP_NORM_RMS, post_, pre_, HipDtype<T>::code, ws, workspace_bytes_,
      nullptr));
  st.store();
  workspace_.data()->array()->clear();
}

template class ResidualNormalizationHip<float>;
template class ResidualNormalizationHip<Half>;
} // namespace nbla
