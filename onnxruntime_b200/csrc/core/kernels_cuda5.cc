// GPU op wrappers, part 5: the operators around one step of a serving batch (com.ortb200 PagedBatchLayout,
// SharedPrefixPagedAttention, TokenLogProbs, TokenLogProbsGrad) on the kernels of batch_layout.cu, prefix_attn.cu and
// token_log_probs.cu.  Workspaces are taken from the allocator call by call: two captured graphs share none.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include "cuda_ops.h"
#include "kernel.h"
#include "serving_checks.h"
#include "serving_cuda.h"
#include "serving_ops.h"
#include "session.h"

namespace ortb {

namespace {

using Ctx = OpKernelContext;

class PagedBatchLayoutKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const BatchLayoutSizes z = CheckBatchLayout(ctx);
    WantOnGpu(ctx);
    if (z.B > ortb200_batch_layout_max_requests() || z.rows > ortb200_batch_layout_max_rows()) {
      Generic(ctx);
      return;
    }
    at::Tensor past = ctx.Input(0).contiguous(), fresh = ctx.Input(1).contiguous(), in = ctx.Input(2).contiguous(), pool = ctx.Input(3).contiguous();
    at::Tensor table = Output(ctx, 0, in.sizes(), at::kInt, in, 2);
    at::Tensor cum = Output(ctx, 1, {z.B + 1}, at::kInt, in), pos = Output(ctx, 2, {z.rows}, at::kLong, in), slot = Output(ctx, 3, {z.rows}, at::kLong, in);
    at::Tensor used = Output(ctx, 4, {1}, at::kInt, in);
    ortb200_batch_layout_args a{};
    a.past_seqlens = past.data_ptr<int>();
    a.new_tokens = fresh.data_ptr<int>();
    a.table_in = in.data_ptr<int>();
    a.free_blocks = pool.data_ptr<int>();
    a.table_out = table.data_ptr<int>();
    a.cum = cum.data_ptr<int>();
    a.positions = pos.data_ptr<int64_t>();
    a.slot_mapping = slot.data_ptr<int64_t>();
    a.blocks_used = used.data_ptr<int>();
    a.B = static_cast<int>(z.B); a.max_blocks = static_cast<int>(z.max_blocks); a.block_size = static_cast<int>(z.block_size);
    a.num_free = z.num_free; a.rows = z.rows;
    a.status = z.strict ? ctx.session()->StatusWord().data_ptr<int>() : nullptr;
    CheckLaunch(ortb200_batch_layout(&a, ctx.cuda_stream()), "ortb200_batch_layout");
    ctx.session()->AddLaunches(1);
    ctx.SetOutput(0, table);
    ctx.SetOutput(1, cum);
    ctx.SetOutput(2, pos);
    ctx.SetOutput(3, slot);
    ctx.SetOutput(4, used);
  }
};

class SharedPrefixPagedAttentionKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const SharedPrefixSizes z = CheckSharedPrefix(ctx);
    WantOnGpu(ctx);
    at::Tensor q = ctx.Input(0).contiguous(), k, v;
    const at::Tensor &kc = ctx.Input(3), &vc = ctx.Input(4);
    const int dt = DtypeCode(q.scalar_type());
    const bool wide = z.max_blocks * z.block_size > ortb200_prefix_attn_max_keys() || (z.N + 2 * z.Nk) * z.H > 0x7fffffffll || z.T * z.N > 0x7ffffffell;
    if (dt < 0 || z.H > 256 || wide || !kc.is_contiguous() || !vc.is_contiguous()) {
      Generic(ctx);
      return;
    }
    at::Tensor out = Output(ctx, 0, {z.T, z.N * z.H}, q.scalar_type(), q);
    if (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15) out = at::empty_like(out);   // rows are written by vectors
    if (z.T > 0 && z.max_blocks == 0) out.zero_();
    if (z.T > 0 && z.max_blocks > 0) {
      at::Tensor cum = ctx.Input(5).contiguous(), past = ctx.Input(6).contiguous(), table = ctx.Input(7).contiguous(), cos, sin, pos, slot;
      ortb200_prefix_attn_args a{};
      a.qkv = q.data_ptr();
      if (!z.packed) {
        k = ctx.Input(1).contiguous();
        v = ctx.Input(2).contiguous();
        a.k = k.data_ptr();
        a.v = v.data_ptr();
      }
      a.k_cache = kc.data_ptr();
      a.v_cache = vc.data_ptr();
      a.cu_seqlens = cum.data_ptr<int>();
      a.past_seqlens = past.data_ptr<int>();
      a.block_table = table.data_ptr<int>();
      a.shared_prefix = ctx.Input(8).data_ptr<int>();
      if (z.rotary) {
        cos = ctx.Input(9).contiguous();
        sin = ctx.Input(10).contiguous();
        a.cos_cache = cos.data_ptr();
        a.sin_cache = sin.data_ptr();
        a.cos_rows = static_cast<int>(cos.size(0));
        a.rot_dim = static_cast<int>(z.rot_dim);
        a.interleaved = z.interleaved ? 1 : 0;
      }
      if (z.placed) {
        pos = ctx.Input(11).contiguous();
        slot = ctx.Input(12).contiguous();
        a.positions = pos.data_ptr<int64_t>();
        a.slot_mapping = slot.data_ptr<int64_t>();
      }
      a.out = out.data_ptr();
      a.T = z.T;
      a.B = static_cast<int>(z.B); a.N = static_cast<int>(z.N); a.Nk = static_cast<int>(z.Nk); a.H = static_cast<int>(z.H);
      a.block_size = static_cast<int>(z.block_size); a.max_blocks = static_cast<int>(z.max_blocks); a.num_blocks = static_cast<int>(z.num_blocks);
      a.scale = z.scale;
      a.softcap = z.softcap;
      a.dtype = dt;
      // 16-bit heads of 64 or 128 over blocks that a tile of 64 keys divides, or that divide it
      const bool blocks = z.block_size % 64 == 0 || z.block_size == 8 || z.block_size == 16 || z.block_size == 32;
      const bool aligned = ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15) == 0;
      a.tensor_cores = dt != ORTB200_F32 && (z.H == 64 || z.H == 128) && blocks && aligned && z.N / z.Nk <= 128 && z.T * z.N <= (1 << 29) ? 1 : 0;
      a.use_pdl = Pdl(ctx);
      a.status = ctx.session()->StatusWord().data_ptr<int>();
      const int64_t bytes = ortb200_prefix_attn_workspace_bytes(a.T, a.B, a.N, a.Nk, a.H, a.tensor_cores);
      at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
      a.workspace = ws.data_ptr();
      a.workspace_bytes = bytes;
      CheckLaunch(ortb200_prefix_attn(&a, ctx.cuda_stream()), "ortb200_prefix_attn");
      ctx.session()->AddLaunches(a.tensor_cores ? 3 : 2);
    }
    ctx.SetOutput(0, out);
    if (ctx.OutputCount() > 1) ctx.SetOutput(1, kc);
    if (ctx.OutputCount() > 2) ctx.SetOutput(2, vc);
  }
};

class TokenLogProbsKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const TokenLogProbsSizes z = CheckTokenLogProbs(ctx);
    WantOnGpu(ctx);
    at::Tensor x = ctx.Input(0).contiguous(), tokens = ctx.Input(1).to(at::kLong).contiguous();
    const int dt = DtypeCode(x.scalar_type());
    if (dt < 0 || z.rows > 0x0fffffffll || z.vocab > ortb200_token_log_probs_max_vocab()) {
      Generic(ctx);
      return;
    }
    std::vector<int64_t> top = z.lead;
    top.push_back(z.top_k);
    const auto wanted = [&](int i) { return i < ctx.OutputCount() && ctx.OutputNeeded(i); };
    at::Tensor out[6];
    for (int i : {0, 1, 4, 5})
      if (wanted(i)) out[i] = Output(ctx, i, z.lead, at::kFloat, x);
    if (wanted(2)) out[2] = Output(ctx, 2, top, at::kFloat, x);
    if (wanted(3)) out[3] = Output(ctx, 3, top, at::kLong, x);
    ortb200_token_log_probs_args a{};
    a.logits = x.data_ptr();
    a.tokens = tokens.data_ptr<int64_t>();
    a.log_prob = wanted(0) ? out[0].data_ptr<float>() : nullptr;
    a.entropy = wanted(1) ? out[1].data_ptr<float>() : nullptr;
    a.log_sum_exp = wanted(4) ? out[4].data_ptr<float>() : nullptr;
    a.top_log_probs = wanted(2) ? out[2].data_ptr<float>() : nullptr;
    a.top_tokens = wanted(3) ? out[3].data_ptr<int64_t>() : nullptr;
    a.log_sum_exp_rest = wanted(5) ? out[5].data_ptr<float>() : nullptr;
    a.rows = z.rows;
    a.vocab = static_cast<int>(z.vocab);
    a.top_k = wanted(2) || wanted(3) ? static_cast<int>(z.top_k) : 0;
    a.dtype = dt;
    a.use_pdl = Pdl(ctx);
    CheckLaunch(ortb200_token_log_probs(&a, ctx.cuda_stream()), "ortb200_token_log_probs");
    ctx.session()->AddLaunches(z.rows > 0 ? 1 : 0);
    for (int i = 0; i < 6; ++i)
      if (out[i].defined()) ctx.SetOutput(i, out[i]);
  }
};

class TokenLogProbsGradKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const TokenLogProbsSizes z = CheckTokenLogProbsGrad(ctx);
    WantOnGpu(ctx);
    at::Tensor x = ctx.Input(0).contiguous(), tokens = ctx.Input(1).to(at::kLong).contiguous();
    const int dt = DtypeCode(x.scalar_type());
    if (dt < 0 || z.rows > 0x0fffffffll || z.vocab > ortb200_token_log_probs_max_vocab()) {
      Generic(ctx);
      return;
    }
    at::Tensor keep[10];
    auto floats = [&](int i) -> const float* {
      if (!ctx.HasInput(i)) return nullptr;
      keep[i] = ctx.Input(i).to(at::kFloat).contiguous();
      return keep[i].data_ptr<float>();
    };
    ortb200_token_log_probs_grad_args a{};
    a.logits = x.data_ptr();
    a.tokens = tokens.data_ptr<int64_t>();
    a.log_sum_exp = floats(2);
    a.entropy = floats(3);
    a.d_log_prob = floats(4);
    a.d_entropy = floats(5);
    if (ctx.HasInput(7) && z.top_k > 0) {
      keep[6] = ctx.Input(6).to(at::kLong).contiguous();
      a.top_tokens = keep[6].data_ptr<int64_t>();
      a.d_top_log_probs = floats(7);
      a.top_k = static_cast<int>(z.top_k);
    }
    a.d_log_sum_exp = floats(8);
    a.log_sum_exp_rest = floats(9);
    at::Tensor dx = Output(ctx, 0, ctx.Input(0).sizes(), x.scalar_type(), x, 0);
    a.d_logits = dx.data_ptr();
    a.rows = z.rows;
    a.vocab = static_cast<int>(z.vocab);
    a.dtype = dt;
    a.use_pdl = Pdl(ctx);
    CheckLaunch(ortb200_token_log_probs_grad(&a, ctx.cuda_stream()), "ortb200_token_log_probs_grad");
    ctx.session()->AddLaunches(z.rows > 0 ? 1 : 0);
    ctx.SetOutput(0, dx);
  }
};

}  // namespace

void RegisterCudaKernels5(KernelRegistry& r) {
  RegFused<PagedBatchLayoutKernel>(r, "PagedBatchLayout");
  RegFused<SharedPrefixPagedAttentionKernel>(r, "SharedPrefixPagedAttention");
  RegFused<TokenLogProbsKernel>(r, "TokenLogProbs");
  RegFused<TokenLogProbsGradKernel>(r, "TokenLogProbsGrad");
}

}  // namespace ortb
