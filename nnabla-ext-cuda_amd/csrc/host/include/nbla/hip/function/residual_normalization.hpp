// ResidualNormalization: the step between two blocks of a residual stream,
//   u = post ? norm(x) : x
//   h = res_scale * res + branch_scale * gate * u
//   y = norm(h)                                     (pre)
// over the axes that are not batch axes; norm "rms" or "layer".  No counterpart
// in the reference, whose graphs chain the functions this one fuses.
//
// Inputs, those that are there, in this order: x, res (residual), gate (gate),
// beta_post, gamma_post (post), beta_pre, gamma_pre (pre); gammas without
// no_scale, betas without no_bias and for "layer" only.  A gate of x's shape has
// an element each; else it has G rows of one element per column, each for
// rows / G successive rows (G = 1: a learned scale; a row per sample).
// Outputs [h, y], without pre [h].  checkpoint "int8" / "e4m3": the forward keeps
// 8-bit copies of x and h, and the backward reads those instead of the data.
#pragma once

#include <nbla/function_registry.hpp>
#include <nbla/hip/common.hpp>
#include <nbla/hip/hip.hpp>
#include <nbla/hip/utils/act8_copy.hpp>
#include <nbla/hip/utils/param_stage.hpp>

namespace nbla {

NBLA_REGISTER_FUNCTION_HEADER(ResidualNormalization, const vector<int> &, const string &, bool, bool,
                              bool, bool, float, float, float, bool, bool, const string &);

template <typename T> class ResidualNormalizationHip : public Function {
protected:
  int device_;
  vector<int> batch_axis_;
  string norm_;
  bool post_, pre_, residual_, gate_;
  float res_scale_, branch_scale_, eps_;
  bool no_scale_, no_bias_;
  string checkpoint_;
  int format8_;
  Size_t rows_ = 0, cols_ = 0, gate_rows_ = 0;
  int gate_kind_ = NBLAHIP_GATE_NONE;
  // number of inputs, and positions in them, -1: not there
  int n_inputs_ = 1;
  int i_res_ = -1, i_gate_ = -1, i_beta_post_ = -1, i_gamma_post_ = -1, i_beta_pre_ = -1,
      i_gamma_pre_ = -1;
  Variable mean_post_, var_post_, mean_pre_, var_pre_; // float32, kept for backward
  Act8Copy x8_, h8_;
  Variable workspace_;
  size_t workspace_bytes_ = 0;
  Variable stage_; // float32 staging of parameters stored in half (ParamStage)

public:
  ResidualNormalizationHip(const Context &ctx, const vector<int> &batch_axis, const string &norm,
                           bool post, bool pre, bool residual, bool gate, float res_scale,
                           float branch_scale, float eps, bool no_scale, bool no_bias,
                           const string &checkpoint)
      : Function(ctx), device_(std::stoi(ctx.device_id)), batch_axis_(batch_axis), norm_(norm),
        post_(post), pre_(pre), residual_(residual), gate_(gate), res_scale_(res_scale),
        branch_scale_(branch_scale), eps_(eps), no_scale_(no_scale), no_bias_(no_bias),
        checkpoint_(checkpoint), format8_(act8_format(checkpoint)) {
    place_inputs();
  }
  virtual ~ResidualNormalizationHip() {}
  virtual string name() { return "ResidualNormalizationHip"; }
  virtual int min_inputs() { return 1; }
  virtual int min_outputs() { return 1; }
  // What a core asks of a function without a class of its own in it.
  virtual vector<dtypes> in_types() { return {get_dtype<T>()}; }
  virtual vector<dtypes> out_types() { return vector<dtypes>(pre_ ? 2 : 1, get_dtype<T>()); }
  virtual std::shared_ptr<Function> copy() const {
    return std::make_shared<ResidualNormalizationHip<T>>(
        this->ctx_, batch_axis_, norm_, post_, pre_, residual_, gate_, res_scale_, branch_scale_, eps_,
        no_scale_, no_bias_, checkpoint_);
  }
  // The backward reads h for the second norm (or its 8-bit copy): it must be kept.
  virtual bool grad_depends_output_data(int i, int o) const {
    return pre_ && format8_ == NBLAHIP_ACT8_NONE && o == 0;
  }
  virtual vector<string> allowed_array_classes() {
    return SingletonManager::get<Hip>()->array_classes();
  }

protected:
  virtual void setup_impl(const Variables &inputs, const Variables &outputs);
  virtual void forward_impl(const Variables &inputs, const Variables &outputs);
  virtual void backward_impl(const Variables &inputs, const Variables &outputs,
                             const vector<bool> &propagate_down, const vector<bool> &accum);
  void backward_pass(const Variables &inputs, const Variables &outputs,
                     const vector<bool> &propagate_down, const vector<bool> &accum);
  void place_inputs();
  // The backward reads the gate, the gammas, a gated step's first beta and, without a
  // checkpoint, x for the first norm or the gate; everything else may be freed.
  virtual bool grad_depends_input_data_impl(int i, int j) const {
    if (j == 0) return reads_x() && format8_ == NBLAHIP_ACT8_NONE;
    if (j == i_res_ || j == i_beta_pre_) return false;
    return j == i_beta_post_ ? gate_ : true;
  }
  bool reads_x() const { return post_ || gate_; }
};
} // namespace nbla
