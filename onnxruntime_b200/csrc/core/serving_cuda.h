// Shared by the GPU wrappers of the serving operators (kernels_cuda5.cc, kernels_cuda6.cc).
#pragma once
#include <ATen/ATen.h>

#include "kernel.h"
#include "ortb200_kernels.h"
#include "serving_checks.h"
#include "session.h"

namespace ortb {

inline int DtypeCode(at::ScalarType t) {
  return t == at::kHalf ? ORTB200_F16 : t == at::kBFloat16 ? ORTB200_BF16 : t == at::kFloat ? ORTB200_F32 : -1;
}
inline int Pdl(OpKernelContext& ctx) { return ctx.session()->config().Get("ortb200.pdl", "0") == "1" ? 1 : 0; }

// The bound buffer of output i where it fits and shares no memory with an input (but `in_place`, all of it), else a new tensor, which the executor
// copies to whatever is bound.
inline at::Tensor Output(OpKernelContext& ctx, int i, at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like, int in_place = -1) {
  if (i < ctx.OutputCount()) {
    const at::Tensor& b = ctx.Preallocated(i);
    if (b.defined() && b.device() == like.device() && b.scalar_type() == type && b.sizes() == sizes && b.is_contiguous()) {
      bool apart = true;
      for (int j = 0; j < ctx.InputCount(); ++j)
        if (ctx.HasInput(j) && Overlap(ctx.Input(j), b) && !(j == in_place && ctx.Input(j).data_ptr() == b.data_ptr())) apart = false;
      for (int j = 0; j < i; ++j)
        if (Overlap(ctx.Preallocated(j), b)) apart = false;
      if (apart) return b;
    }
  }
  return at::empty(sizes, like.options().dtype(type));
}

// Operands that the kernels do not take run on the device-agnostic kernel.
class WithGeneric : public OpKernel {
 public:
  explicit WithGeneric(const OpKernelInfo& info) : OpKernel(info) {
    if (const KernelDef* d = KernelRegistry::Generic().Find(info.node, info.graph)) generic_ = d->factory(info);
  }

 protected:
  void Generic(OpKernelContext& ctx) const {
    if (!generic_) ORTB_THROW(NOT_IMPLEMENTED, "no other kernel for ", node_.op_type);
    generic_->Compute(ctx);
  }
  std::unique_ptr<OpKernel> generic_;
};

inline void WantOnGpu(OpKernelContext& ctx) {
  for (int i = 0; i < ctx.InputCount(); ++i)
    ORTB_ENFORCE_ARG(!ctx.HasInput(i) || ctx.Input(i).device() == ctx.device(), ctx.node().op_type, ": input ", i, " must lie on the session's GPU");
}

template <typename K>
void RegFused(KernelRegistry& r, const std::string& op) {
  KernelDef d;
  d.domain = "com.ortb200";
  d.op_type = op;
  d.factory = [](const OpKernelInfo& info) { return std::make_unique<K>(info); };
  r.Register(std::move(d));
}

}  // namespace ortb
