// GPU op wrappers, part 6: the operators around a decode step with drafted tokens (com.ortb200 TreePagedAttention,
// PagedCacheMove, ProcessLogits) on the kernels of prefix_attn.cu, cache_move.cu and process_logits.cu.  Workspaces are taken from
// the allocator call by call: two captured graphs share none.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>

#include "cuda_ops.h"
#include "draft_ops.h"
#include "kernel.h"
#include "serving_checks.h"
#include "serving_cuda.h"
#include "session.h"

namespace ortb {

namespace {

using Ctx = OpKernelContext;

class TreePagedAttentionKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const SharedPrefixSizes z = CheckTreeAttention(ctx);
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
      at::Tensor cum = ctx.Input(5).contiguous(), past = ctx.Input(6).contiguous(), table = ctx.Input(7).contiguous(), parents = ctx.Input(8).contiguous(), cos, sin;
      ortb200_tree_attn_args t{};
      ortb200_prefix_attn_args& a = t.attn;
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
      t.parents = parents.data_ptr<int>();
      if (z.rotary) {
        cos = ctx.Input(9).contiguous();
        sin = ctx.Input(10).contiguous();
        a.cos_cache = cos.data_ptr();
        a.sin_cache = sin.data_ptr();
        a.cos_rows = static_cast<int>(cos.size(0));
        a.rot_dim = static_cast<int>(z.rot_dim);
        a.interleaved = z.interleaved ? 1 : 0;
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
      a.workspace_bytes = ortb200_tree_attn_workspace_bytes(a.T, a.B, a.N, a.Nk, a.H, a.tensor_cores);
      at::Tensor ws = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));
      a.workspace = ws.data_ptr();
      CheckLaunch(ortb200_tree_attn(&t, ctx.cuda_stream()), "ortb200_tree_attn");
      ctx.session()->AddLaunches(a.tensor_cores ? 3 : 2);
    }
    ctx.SetOutput(0, out);
    if (ctx.OutputCount() > 1) ctx.SetOutput(1, kc);
    if (ctx.OutputCount() > 2) ctx.SetOutput(2, vc);
  }
};

class PagedCacheMoveKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const CacheMoveSizes z = CheckCacheMove(ctx);
    WantOnGpu(ctx);
    std::vector<void*> caches(z.caches);
    std::vector<int64_t> bytes(z.caches);
    bool dense = z.moves <= ortb200_cache_move_max_moves();
    for (int i = 0; i < z.caches; ++i) {
      const at::Tensor& c = ctx.Input(2 + i);
      dense = dense && c.is_contiguous();
      caches[i] = c.data_ptr();
      bytes[i] = z.units > 0 ? c.numel() / z.units * static_cast<int64_t>(c.element_size()) : 0;
    }
    if (!dense) {
      Generic(ctx);
      return;
    }
    at::Tensor sources = ctx.Input(0).contiguous(), targets = ctx.Input(1).contiguous();
    ortb200_cache_move_args a{};
    a.caches = caches.data();
    a.unit_bytes = bytes.data();
    a.num_caches = z.caches;
    a.units = z.units;
    a.sources = sources.data_ptr<int64_t>();
    a.targets = targets.data_ptr<int64_t>();
    a.moves = z.moves;
    a.use_pdl = Pdl(ctx);
    a.status = ctx.session()->StatusWord().data_ptr<int>();
    CheckLaunch(ortb200_cache_move(&a, ctx.cuda_stream()), "ortb200_cache_move");
    ctx.session()->AddLaunches(z.moves > 0 ? 1 : 0);
    for (int i = 0; i < z.caches && i < ctx.OutputCount(); ++i) ctx.SetOutput(i, ctx.Input(2 + i));
  }
};

class ProcessLogitsKernel final : public WithGeneric {
 public:
  using WithGeneric::WithGeneric;
  void Compute(Ctx& ctx) const override {
    const ProcessLogitsSizes z = CheckProcessLogits(ctx);
    WantOnGpu(ctx);
    at::Tensor x = ctx.Input(0).contiguous();
    const int dt = DtypeCode(x.scalar_type());
    if (dt < 0 || z.vocab > ortb200_process_logits_max_vocab() || z.history + z.drafted > (1 << 30) - 1 || z.rows > (1 << 28) || z.drafted > 0x7fffffff) {
      Generic(ctx);
      return;
    }
    at::Tensor keep[15];
    const auto given = [&](int i, at::ScalarType type) -> void* {
      if (!ctx.HasInput(i)) return nullptr;
      keep[i] = ctx.Input(i).to(type).contiguous();
      // an input without elements is there all the same
      return keep[i].numel() > 0 ? keep[i].data_ptr() : x.data_ptr();
    };
    at::Tensor out = Output(ctx, 0, x.sizes(), at::kFloat, x);   // (biased tokens are read twice: not in place)
    ortb200_process_logits_args a{};
    a.logits = x.data_ptr();
    a.scores = out.data_ptr<float>();
    a.history = static_cast<int64_t*>(given(1, at::kLong));
    a.history_starts = static_cast<int64_t*>(given(2, at::kLong));
    a.generated_starts = static_cast<int64_t*>(given(3, at::kLong));
    a.row_list = static_cast<int*>(given(4, at::kInt));
    a.drafted = z.drafted > 0 ? static_cast<int64_t*>(given(5, at::kLong)) : nullptr;
    a.repetition = static_cast<float*>(given(6, at::kFloat));
    a.presence = static_cast<float*>(given(7, at::kFloat));
    a.frequency = static_cast<float*>(given(8, at::kFloat));
    if (z.biases > 0) {
      a.bias_tokens = static_cast<int64_t*>(given(9, at::kLong));
      a.bias_values = static_cast<float*>(given(10, at::kFloat));
    }
    a.bias_starts = static_cast<int64_t*>(given(11, at::kLong));   // without biases, too: starts that are none are reported
    a.allowed = static_cast<int*>(given(12, at::kInt));
    a.row_mask = static_cast<int*>(given(13, at::kInt));
    a.temperature = static_cast<float*>(given(14, at::kFloat));
    a.rows = z.rows;
    a.history_len = z.history;
    a.bias_len = z.biases;
    a.lists = z.lists;
    a.vocab = static_cast<int>(z.vocab);
    a.drafted_width = static_cast<int>(z.drafted);
    a.masks = static_cast<int>(z.masks);
    a.mask_words = static_cast<int>(z.mask_words);
    a.dtype = dt;
    a.use_pdl = Pdl(ctx);
    a.status = ctx.session()->StatusWord().data_ptr<int>();
    if (z.rows > 0) {
      CheckLaunch(ortb200_process_logits(&a, ctx.cuda_stream()), "ortb200_process_logits");
      ctx.session()->AddLaunches(1);
    }
    ctx.SetOutput(0, out);
  }
};

}  // namespace

void RegisterCudaKernels6(KernelRegistry& r) {
  RegFused<TreePagedAttentionKernel>(r, "TreePagedAttention");
  RegFused<PagedCacheMoveKernel>(r, "PagedCacheMove");
  RegFused<ProcessLogitsKernel>(r, "ProcessLogits");
}

}  // namespace ortb
