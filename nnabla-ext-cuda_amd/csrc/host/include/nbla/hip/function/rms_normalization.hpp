// RMSNormalization: y = x / sqrt(mean(x^2) + eps) * gamma over the axes that are
// not batch axes.  No counterpart in the reference; the class follows
// LayerNormalizationHip<T> (arguments, statistics kept for backward, parameters
// that may be stored in half).
//
// Inputs [x] (no_scale) or [x, gamma]; output [y].  checkpoint "int8" / "e4m3":
// the forward keeps an 8-bit copy of x, and the backward reads that instead of
// the input's data.
#pragma once

#include <nbla/function_registry.hpp>
#include <nbla/hip/common.hpp>
#include <nbla/hip/hip.hpp>
#include <nbla/hip/utils/act8_copy.hpp>
#include <nbla/hip/utils/param_stage.hpp>

namespace nbla {

NBLA_REGISTER_FUNCTION_HEADER(RMSNormalization, const vector<int> &, float, bool, const string &);

template <typename T> class RMSNormalizationHip : public Function {
protected:
  int device_;
  vector<int> batch_axis_;
  float eps_;
  bool no_scale_;
  string checkpoint_;
  int format8_;
  Size_t rows_ = 0, cols_ = 0;
  Variable ms_; // float32 mean squares kept for backward
  Act8Copy x8_;
  Variable workspace_;
  size_t workspace_bytes_ = 0;
  Variable stage_; // float32 staging of parameters stored in half (ParamStage)

public:
  RMSNormalizationHip(const Context &ctx, const vector<int> &batch_axis, float eps, bool no_scale,
                      const string &checkpoint)
      : Function(ctx), device_(std::stoi(ctx.device_id)), batch_axis_(batch_axis), eps_(eps),
        no_scale_(no_scale), checkpoint_(checkpoint),
        format8_(act8_format(checkpoint)) {}
  virtual ~RMSNormalizationHip() {}
  virtual string name() { return "RMSNormalizationHip"; }
  virtual int min_inputs() { return 1; }
  virtual int min_outputs() { return 1; }
  // What a core asks of a function without a class of its own in it.
  virtual vector<dtypes> in_types() { return {get_dtype<T>()}; }
  virtual vector<dtypes> out_types() { return vector<dtypes>(1, get_dtype<T>()); }
  virtual std::shared_ptr<Function> copy() const {
    return std::make_shared<RMSNormalizationHip<T>>(this->ctx_, batch_axis_, eps_, no_scale_, checkpoint_);
  }
  virtual vector<string> allowed_array_classes() {
    return SingletonManager::get<Hip>()->array_classes();
  }

protected:
  virtual void setup_impl(const Variables &inputs, const Variables &outputs);
  virtual void forward_impl(const Variables &inputs, const Variables &outputs);
  virtual void backward_impl(const Variables &inputs, const Variables &outputs,
                             const vector<bool> &propagate_down, const vector<bool> &accum);
  // With a checkpoint the backward reads the copy: x may be freed after the forward.
  virtual bool grad_depends_input_data_impl(int i, int j) const {
    return j == 0 ? format8_ == NBLAHIP_ACT8_NONE : true;
  }
};
} // namespace nbla
