// com.ortb200 operators around one step of a serving batch, device-agnostic versions (tensor library): PagedBatchLayout (block
// table, positions and cache slots out of request lengths), SharedPrefixPagedAttention (sequences that begin with the same
// tokens), TreePagedAttention (sequences that bring a tree of drafted tokens), TokenLogProbs and TokenLogProbsGrad (log probabilities, entropy and alternatives, and their gradient).  The GPU
// provider has its own kernels (kernels_cuda5.cc).
#include <ATen/ATen.h>

#include <cmath>
#include <limits>

#include "kernel.h"
#include "serving_checks.h"

namespace ortb {

namespace {

using Ctx = OpKernelContext;
constexpr int kMax = 1 << 30;
constexpr const char* FUSED = "com.ortb200";

std::vector<int64_t> HostInts(const at::Tensor& t) {
  at::Tensor c = t.to(at::kCPU, at::kLong).contiguous();
  return std::vector<int64_t>(c.data_ptr<int64_t>(), c.data_ptr<int64_t>() + c.numel());
}
at::Tensor F32(const at::Tensor& t) { return t.to(at::kFloat); }
int64_t BlocksOf(int64_t tokens, int64_t size) { return (tokens + size - 1) / size; }

void WantInts(Ctx& ctx, int i, at::ScalarType type, int64_t dim, const char* what) {
  const at::Tensor& t = ctx.RequiredInput(i);
  ORTB_ENFORCE_ARG(t.scalar_type() == type && (dim < 0 || t.dim() == dim), ctx.node().op_type, ": ", what, " must be ", c10::toString(type), " of rank ", dim);
}

void PagedBatchLayoutImpl(Ctx& ctx) {
  const BatchLayoutSizes z = CheckBatchLayout(ctx);
  const at::Tensor& table_in = ctx.Input(2);
  const std::vector<int64_t> past = HostInts(ctx.Input(0)), fresh = HostInts(ctx.Input(1)), pool = HostInts(ctx.Input(3));
  at::Tensor table = table_in.to(at::kCPU).contiguous().clone();
  at::Tensor cum = at::zeros({z.B + 1}, at::kInt), pos = at::full({z.rows}, -1, at::kLong), slot = at::full({z.rows}, -1, at::kLong), used = at::zeros({1}, at::kInt);
  int64_t tokens = 0, blocks = 0;
  int refused = 0;
  for (int64_t b = 0; b < z.B; ++b) {
    if (past[b] < 0 || fresh[b] < 0) {
      refused = 4;
      continue;
    }
    const int64_t held = BlocksOf(past[b], z.block_size), all = BlocksOf(past[b] + fresh[b], z.block_size);
    if (fresh[b] > 0 && all > z.max_blocks) refused = std::max(refused, 2);
    tokens += fresh[b];
    blocks += all - held;
  }
  if (refused < 4 && tokens > z.rows) refused = 3;
  if (refused < 2 && blocks > z.num_free) refused = 1;
  ORTB_ENFORCE_ARG(!refused || !z.strict, "PagedBatchLayout: the batch cannot be laid out (", -refused, ": ",
                   refused == 1 ? "too few free blocks" : refused == 2 ? "the table is too narrow" : refused == 3 ? "more tokens than rows" : "a negative length", ")");
  if (!refused) {
    int* tb = table.data_ptr<int>();
    int64_t row = 0, next = 0;
    for (int64_t b = 0; b < z.B; ++b) {
      int* mine = tb + b * z.max_blocks;
      for (int64_t j = BlocksOf(past[b], z.block_size); j < BlocksOf(past[b] + fresh[b], z.block_size); ++j) mine[j] = static_cast<int>(pool[next++]);
      for (int64_t s = 0; s < fresh[b]; ++s, ++row) {
        const int64_t p = past[b] + s;
        pos.data_ptr<int64_t>()[row] = p;
        slot.data_ptr<int64_t>()[row] = static_cast<int64_t>(mine[p / z.block_size]) * z.block_size + p % z.block_size;
      }
      cum.data_ptr<int>()[b + 1] = static_cast<int>(row);
    }
  }
  used.data_ptr<int>()[0] = refused ? -refused : static_cast<int>(blocks);
  const c10::Device dev = table_in.device();
  ctx.SetOutput(0, table.to(dev));
  ctx.SetOutput(1, cum.to(dev));
  ctx.SetOutput(2, pos.to(dev));
  ctx.SetOutput(3, slot.to(dev));
  ctx.SetOutput(4, used.to(dev));
}

// Of the rows of a sequence: which ones each sees, [S, S], and how deep each lies; undefined where the rows form a prompt.
std::pair<at::Tensor, at::Tensor> TreeOf(const std::vector<int64_t>& parents, int64_t t0, int64_t S, int64_t b) {
  for (int64_t i = 0; i < S; ++i) {
    const int64_t p = parents[t0 + i];
    ORTB_ENFORCE_ARG(p >= -1 && p < i && (S <= kMostTreeNodes || p == i - 1), "TreePagedAttention: the parent of row ", i, " of sequence ", b,
                     S > kMostTreeNodes ? " must be the row before it: the sequence has more rows than a tree" : " must be a row in front of it, or -1");
  }
  if (S > kMostTreeNodes) return {};
  at::Tensor sees = at::zeros({S, S}, at::kBool), depth = at::zeros({S}, at::kLong);
  for (int64_t i = 0; i < S; ++i) {
    const int64_t p = parents[t0 + i];
    if (p >= 0) {
      sees[i].copy_(sees[p]);
      depth.data_ptr<int64_t>()[i] = depth.data_ptr<int64_t>()[p] + 1;
    }
    sees.data_ptr<bool>()[i * S + i] = true;
  }
  return {sees, depth};
}

// The promise about the first tokens changes nothing here: every sequence reads its own row of the table.
void PagedQueries(Ctx& ctx, const SharedPrefixSizes& z) {
  const std::string& op = ctx.node().op_type;
  at::Tensor q = ctx.Input(0), k, v;
  at::Tensor kc = ctx.Input(3), vc = ctx.Input(4);
  if (z.packed) {
    k = q.narrow(1, z.N * z.H, z.Nk * z.H);
    v = q.narrow(1, (z.N + z.Nk) * z.H, z.Nk * z.H);
    q = q.narrow(1, 0, z.N * z.H);
  } else {
    k = ctx.Input(1);
    v = ctx.Input(2);
  }
  q = q.reshape({z.T, z.N, z.H});
  k = k.reshape({z.T, z.Nk, z.H});
  v = v.reshape({z.T, z.Nk, z.H});
  const std::vector<int64_t> cum = HostInts(ctx.Input(5)), past = HostInts(ctx.Input(6));
  const at::Tensor table = ctx.Input(7).to(at::kCPU, at::kLong);
  const std::vector<int64_t> parents = z.tree ? HostInts(ctx.Input(8)) : std::vector<int64_t>();
  at::Tensor given_pos, given_slot;
  if (z.placed) {
    given_pos = ctx.Input(11).to(at::kCPU);
    given_slot = ctx.Input(12).to(at::kCPU);
  }
  const double scale = z.scale != 0.f ? z.scale : 1.0 / std::sqrt(static_cast<double>(z.H));
  auto rotate = [&](const at::Tensor& x, const at::Tensor& pos) {   // x [L, heads, H]
    if (!z.rotary) return x;
    const int64_t half = z.rot_dim / 2;
    at::Tensor c = F32(ctx.Input(9).index_select(0, pos.to(x.device()))).unsqueeze(1), s = F32(ctx.Input(10).index_select(0, pos.to(x.device()))).unsqueeze(1);
    at::Tensor xf = F32(x), turned = xf.narrow(2, 0, z.rot_dim);
    if (z.interleaved) {
      at::Tensor pairs = turned.reshape({x.size(0), x.size(1), half, 2}), u = pairs.select(3, 0), w = pairs.select(3, 1);
      turned = at::stack({u * c - w * s, w * c + u * s}, 3).reshape({x.size(0), x.size(1), z.rot_dim});
    } else {
      at::Tensor u = turned.narrow(2, 0, half), w = turned.narrow(2, half, half);
      turned = at::cat({u * c - w * s, w * c + u * s}, 2);
    }
    return at::cat({turned, xf.narrow(2, z.rot_dim, z.H - z.rot_dim)}, 2).to(x.scalar_type());
  };
  at::Tensor out = at::zeros({z.T, z.N, z.H}, q.options());
  for (int64_t b = 0; b < z.B; ++b) {
    const int64_t t0 = cum[b], S = cum[b + 1] - t0, pl = past[b], L = pl + S;
    ORTB_ENFORCE_ARG(t0 >= 0 && S >= 0 && t0 + S <= z.T && pl >= 0 && (S == 0 || L <= z.max_blocks * z.block_size),
                     op, ": lengths of sequence ", b, " do not fit the batch or the block table");
    if (S == 0) continue;
    std::pair<at::Tensor, at::Tensor> tree;
    if (z.tree) tree = TreeOf(parents, t0, S, b);
    at::Tensor pos = z.placed ? given_pos.narrow(0, t0, S) : (tree.second.defined() ? tree.second : at::arange(S, at::kLong)) + pl;
    ORTB_ENFORCE_ARG(!z.rotary || (pos.min().item<int64_t>() >= 0 && pos.max().item<int64_t>() < ctx.Input(9).size(0)),
                     op, ": a position of sequence ", b, " lies outside the rotary tables");
    at::Tensor qb = rotate(q.narrow(0, t0, S), pos), kb = rotate(k.narrow(0, t0, S), pos), vb = v.narrow(0, t0, S);
    const int64_t nblk = BlocksOf(L, z.block_size);
    at::Tensor blocks = table[b].narrow(0, 0, nblk);
    ORTB_ENFORCE_ARG(blocks.min().item<int64_t>() >= 0 && blocks.max().item<int64_t>() < z.num_blocks,
                     op, ": the table of sequence ", b, " names a block outside the cache");
    for (int64_t s = 0; s < S; ++s) {
      const int64_t p = pl + s, slot = z.placed ? given_slot[t0 + s].item<int64_t>() : blocks[p / z.block_size].item<int64_t>() * z.block_size + p % z.block_size;
      ORTB_ENFORCE_ARG(slot >= 0 && slot < z.num_blocks * z.block_size, op, ": the slot of a token of sequence ", b, " lies outside the cache");
      kc[slot / z.block_size][slot % z.block_size].copy_(kb[s]);
      vc[slot / z.block_size][slot % z.block_size].copy_(vb[s]);
    }
    blocks = blocks.to(kc.device());
    auto gather = [&](const at::Tensor& c) {
      return F32(c.index_select(0, blocks).reshape({nblk * z.block_size, z.Nk, z.H}).narrow(0, 0, L)).permute({1, 0, 2}).repeat_interleave(z.N / z.Nk, 0);
    };
    at::Tensor s = at::matmul(F32(qb).permute({1, 0, 2}), gather(kc).transpose(1, 2)) * scale;   // [N, S, L]
    if (z.softcap > 0.f) s = at::tanh(s / z.softcap) * z.softcap;
    at::Tensor qpos = (at::arange(S, s.options().dtype(at::kLong)) + pl).unsqueeze(1), kpos = at::arange(L, s.options().dtype(at::kLong)).unsqueeze(0);
    at::Tensor hidden = kpos.gt(qpos);
    if (tree.first.defined()) hidden.narrow(1, pl, S).copy_(tree.first.logical_not());
    s = s.masked_fill(hidden.unsqueeze(0), -std::numeric_limits<float>::infinity());
    at::Tensor values = gather(vc), weights = at::softmax(s, -1), product;
    if (z.tree && !at::isfinite(values.narrow(1, pl, S)).all().item<bool>()) {
      // values that are not finite count for rows that see them, and 0 times them not for the others
      at::Tensor finite = at::isfinite(values).all(2, true);   // [N, L, 1]
      finite.narrow(1, 0, pl).fill_(true);
      product = at::matmul(weights, at::where(finite, values, at::zeros_like(values)));
      at::Tensor spoilt = at::matmul(hidden.logical_not().to(values.scalar_type()).unsqueeze(0), finite.logical_not().to(values.scalar_type()));   // [N, S, 1]
      product = product.masked_fill(spoilt.gt(0), std::numeric_limits<float>::quiet_NaN());
    } else {
      product = at::matmul(weights, values);
    }
    out.narrow(0, t0, S).copy_(product.permute({1, 0, 2}));
  }
  ctx.SetOutput(0, out.reshape({z.T, z.N * z.H}));
  if (ctx.OutputCount() > 1) ctx.SetOutput(1, kc);
  if (ctx.OutputCount() > 2) ctx.SetOutput(2, vc);
}

void SharedPrefixPagedAttentionImpl(Ctx& ctx) { PagedQueries(ctx, CheckSharedPrefix(ctx)); }
void TreePagedAttentionImpl(Ctx& ctx) { PagedQueries(ctx, CheckTreeAttention(ctx)); }

at::Tensor WideLogits(const at::Tensor& x, const TokenLogProbsSizes& z) {
  return (x.scalar_type() == at::kDouble ? x : F32(x)).reshape({z.rows, z.vocab});
}

void TokenLogProbsImpl(Ctx& ctx) {
  const TokenLogProbsSizes z = CheckTokenLogProbs(ctx);
  at::Tensor x = WideLogits(ctx.Input(0), z), tokens = ctx.Input(1).to(at::kLong).reshape({z.rows});
  const double inf = std::numeric_limits<double>::infinity();
  at::Tensor m = z.rows > 0 ? x.amax(1, true) : x.narrow(1, 0, 1);
  at::Tensor empty = m.eq(-inf);                                     // nothing in the row is possible
  at::Tensor from = at::where(empty, at::zeros_like(m), m), d = x - from, e = at::exp(d), s = e.sum(1, true);
  at::Tensor log_s = at::log(s), lse = at::where(empty, m, m + log_s);
  at::Tensor w = (e * d.clamp_min(-1000.0)).sum(1, true);             // (exp(-1000) is 0, and 0 times -inf has to count as 0)
  at::Tensor entropy = at::where(empty, at::zeros_like(s), log_s - w / s);
  at::Tensor in = tokens.ge(0).logical_and(tokens.lt(z.vocab));
  // (from the largest logit: m + log S is rounded by 2^-24 of m)
  auto log_prob_of = [&](const at::Tensor& idx) { return at::where(empty, at::full_like(lse, -inf), x.gather(1, idx) - from - log_s); };
  at::Tensor lp = log_prob_of(at::where(in, tokens, at::zeros_like(tokens)).unsqueeze(1)).squeeze(1);
  std::vector<int64_t> top = z.lead;
  top.push_back(z.top_k);
  ctx.SetOutput(0, F32(at::where(in, lp, at::zeros_like(lp))).reshape(z.lead));
  if (ctx.OutputCount() > 1) ctx.SetOutput(1, F32(entropy).reshape(z.lead));
  if (ctx.OutputCount() > 2 && (ctx.OutputNeeded(2) || (ctx.OutputCount() > 3 && ctx.OutputNeeded(3)))) {
    at::Tensor order = std::get<1>(at::sort(x, /*stable=*/true, 1, /*descending=*/true)).narrow(1, 0, z.top_k);
    ctx.SetOutput(2, F32(z.top_k ? log_prob_of(order) : x.narrow(1, 0, 0)).reshape(top));
    if (ctx.OutputCount() > 3) ctx.SetOutput(3, order.reshape(top).contiguous());
  }
  if (ctx.OutputCount() > 4) ctx.SetOutput(4, F32(lse).reshape(z.lead));
  if (ctx.OutputCount() > 5) {   // what rounding to 32 bits takes from m + log S
    at::Tensor sum = lse.to(at::kFloat).to(at::kDouble), rest = (m.to(at::kDouble) - sum) + log_s.to(at::kDouble);
    ctx.SetOutput(5, F32(at::where(at::isfinite(sum), rest, at::zeros_like(rest))).reshape(z.lead));
  }
}

void TokenLogProbsGradImpl(Ctx& ctx) {
  const TokenLogProbsSizes z = CheckTokenLogProbsGrad(ctx);
  at::Tensor x = WideLogits(ctx.Input(0), z), tokens = ctx.Input(1).to(at::kLong).reshape({z.rows, 1});
  const double inf = std::numeric_limits<double>::infinity();
  auto column = [&](int i) { return ctx.HasInput(i) ? ctx.Input(i).to(x.scalar_type()).reshape({z.rows, 1}) : at::zeros({z.rows, 1}, x.options()); };
  at::Tensor lse = column(2), empty = lse.eq(-inf);
  at::Tensor lp = x - at::where(empty, at::zeros_like(lse), lse) - column(9), gone = x.eq(-inf);
  at::Tensor in = tokens.ge(0).logical_and(tokens.lt(z.vocab));
  at::Tensor g = at::where(in, column(4), at::zeros_like(lse)), all = column(8) - g, h = column(5);
  at::Tensor top;
  if (ctx.HasInput(7)) {
    top = ctx.Input(7).to(x.scalar_type()).reshape({z.rows, z.top_k});
    all = all - top.sum(1, true);
  }
  at::Tensor dx = at::exp(lp) * all;
  if (ctx.HasInput(5)) dx = dx - at::exp(lp) * h * (lp.clamp_min(-1000.0) + column(3));   // (exp(-1000) is 0: the factor needs no more than a finite value)
  dx = at::where(gone, at::zeros_like(dx), dx);
  dx = dx.scatter_add(1, at::where(in, tokens, at::zeros_like(tokens)), g);
  if (top.defined() && z.top_k > 0) dx = dx.scatter_add(1, ctx.Input(6).to(at::kLong).reshape({z.rows, z.top_k}), top);
  dx = at::where(empty, at::zeros_like(dx), dx);
  ctx.SetOutput(0, dx.to(ctx.Input(0).scalar_type()).reshape(ctx.Input(0).sizes()));
}

}  // namespace

BatchLayoutSizes CheckBatchLayout(Ctx& ctx) {
  BatchLayoutSizes z;
  const char* op = "PagedBatchLayout";
  z.block_size = ctx.node().attr_i("block_size", 0);
  ORTB_ENFORCE_ARG(z.block_size > 0 && z.block_size <= (1 << 30), op, ": block_size must be positive");
  z.strict = ctx.node().attr_i("strict", 0) != 0;
  WantInts(ctx, 0, at::kInt, 1, "past_seqlens");
  WantInts(ctx, 1, at::kInt, 1, "new_tokens");
  WantInts(ctx, 2, at::kInt, 2, "block_table");
  WantInts(ctx, 3, at::kInt, 1, "free_blocks");
  const at::Tensor& rows = ctx.RequiredInput(4);
  z.B = ctx.Input(0).size(0);
  z.max_blocks = ctx.Input(2).size(1);
  z.num_free = ctx.Input(3).size(0);
  ORTB_ENFORCE_ARG(rows.dim() >= 1, op, ": rows must have a first dimension, the packed tokens");
  z.rows = rows.size(0);
  ORTB_ENFORCE_ARG(ctx.Input(1).size(0) == z.B && ctx.Input(2).size(0) == z.B, op, ": lengths and block table disagree about the number of requests");
  ORTB_ENFORCE_ARG(z.rows < (int64_t(1) << 31) && z.max_blocks < (int64_t(1) << 31), op, ": a dimension beyond 32 bits");
  return z;
}

namespace {
SharedPrefixSizes PagedQuerySizes(Ctx& ctx, const char* no_window) {
  SharedPrefixSizes z;
  const Node& n = ctx.node();
  const std::string& op = n.op_type;
  z.N = n.attr_i("num_heads", 0);
  z.Nk = n.attr_i("kv_num_heads", 0);
  z.scale = n.attr_f("scale", 0.f);
  z.softcap = n.attr_f("softcap", 0.f);
  z.rotary = n.attr_i("do_rotary", 0) != 0;
  z.interleaved = n.attr_i("rotary_interleaved", 0) != 0;
  const at::Tensor &q = ctx.RequiredInput(0), &kc = ctx.RequiredInput(3), &vc = ctx.RequiredInput(4);
  ORTB_ENFORCE_ARG(n.attr_i("local_window_size", -1) <= 0, op, no_window);
  ORTB_ENFORCE_ARG(z.N > 0 && z.Nk > 0 && z.N % z.Nk == 0, op, ": num_heads must be a multiple of kv_num_heads");
  ORTB_ENFORCE_ARG(z.softcap >= 0.f && std::isfinite(z.softcap), op, ": softcap must be finite and not negative");
  ORTB_ENFORCE_ARG(z.scale >= 0.f && std::isfinite(z.scale), op, ": scale must be finite and not negative");
  ORTB_ENFORCE_ARG(q.dim() == 2 && kc.dim() == 4 && vc.sizes() == kc.sizes() && kc.size(2) == z.Nk, op, ": query must be [tokens, width] and the caches [blocks, block size, ",
                   z.Nk, ", head size]");
  ORTB_ENFORCE_ARG(q.is_floating_point() && kc.scalar_type() == q.scalar_type() && vc.scalar_type() == q.scalar_type(), op, ": query and caches must have one floating type");
  z.T = q.size(0);
  z.num_blocks = kc.size(0);
  z.block_size = kc.size(1);
  z.H = kc.size(3);
  z.packed = !ctx.HasInput(1);
  ORTB_ENFORCE_ARG(z.num_blocks > 0 && z.block_size > 0 && z.H > 0 && z.num_blocks < (int64_t(1) << 31), op, ": an empty cache");
  ORTB_ENFORCE_ARG(q.size(1) == (z.packed ? z.N + 2 * z.Nk : z.N) * z.H, op, ": the query's width does not fit its heads");
  if (!z.packed) {
    for (int i : {1, 2}) {
      const at::Tensor& t = ctx.RequiredInput(i);
      ORTB_ENFORCE_ARG(t.dim() == 2 && t.size(0) == z.T && t.size(1) == z.Nk * z.H && t.scalar_type() == q.scalar_type(), op, ": key and value must be [tokens, ",
                       z.Nk * z.H, "] of the query's type");
    }
  }
  WantInts(ctx, 5, at::kInt, 1, "cumulative_sequence_length");
  WantInts(ctx, 6, at::kInt, 1, "past_seqlens");
  WantInts(ctx, 7, at::kInt, 2, "block_table");
  z.B = ctx.Input(6).size(0);
  z.max_blocks = ctx.Input(7).size(1);
  ORTB_ENFORCE_ARG(ctx.Input(5).size(0) == z.B + 1 && ctx.Input(7).size(0) == z.B, op, ": lengths and block table disagree about the number of sequences");
  ORTB_ENFORCE_ARG(z.T == 0 || z.B == 0 || z.max_blocks > 0, op, ": a block table without columns");
  if (z.rotary) {
    const at::Tensor &c = ctx.RequiredInput(9), &s = ctx.RequiredInput(10);
    ORTB_ENFORCE_ARG(c.dim() == 2 && c.sizes() == s.sizes() && c.size(0) > 0 && c.size(1) > 0 && 2 * c.size(1) <= z.H && c.scalar_type() == q.scalar_type() &&
                         s.scalar_type() == q.scalar_type(),
                     op, ": the rotary tables must be [positions, up to ", z.H / 2, "] of the query's type");
    z.rot_dim = 2 * c.size(1);
  }
  return z;
}
}  // namespace

SharedPrefixSizes CheckTreeAttention(Ctx& ctx) {
  SharedPrefixSizes z = PagedQuerySizes(ctx, ": no window is known for trees; use PagedAttention");
  WantInts(ctx, 8, at::kInt, 1, "parents");
  ORTB_ENFORCE_ARG(ctx.Input(8).size(0) == z.T, "TreePagedAttention: parents have one entry per token");
  const at::Tensor &kc = ctx.Input(3), &vc = ctx.Input(4);   // (views that lie side by side in one tensor are not contiguous)
  ORTB_ENFORCE_ARG(!kc.is_contiguous() || !vc.is_contiguous() || !Overlap(kc, vc), "TreePagedAttention: key and value caches share memory");
  z.tree = true;
  return z;
}

SharedPrefixSizes CheckSharedPrefix(Ctx& ctx) {
  const char* op = "SharedPrefixPagedAttention";
  SharedPrefixSizes z = PagedQuerySizes(ctx, ": a window excludes the shared tokens; use PagedAttention");
  WantInts(ctx, 8, at::kInt, -1, "shared_prefix");
  ORTB_ENFORCE_ARG(ctx.Input(8).numel() == 1, op, ": shared_prefix is one number");
  z.placed = ctx.HasInput(11);
  ORTB_ENFORCE_ARG(z.placed == ctx.HasInput(12), op, ": positions and slot_mapping come together");
  for (int i : {11, 12})
    if (z.placed) {
      WantInts(ctx, i, at::kLong, 1, i == 11 ? "positions" : "slot_mapping");
      ORTB_ENFORCE_ARG(ctx.Input(i).size(0) == z.T, op, ": positions and slot_mapping have one entry per token");
    }
  return z;
}

namespace {
TokenLogProbsSizes LogitsAndTokens(Ctx& ctx) {
  TokenLogProbsSizes z;
  const std::string& op = ctx.node().op_type;
  const at::Tensor &x = ctx.RequiredInput(0), &t = ctx.RequiredInput(1);
  ORTB_ENFORCE_ARG(x.dim() >= 1 && x.is_floating_point(), op, ": logits must be floating with the vocabulary as the last dimension");
  z.vocab = x.size(-1);
  ORTB_ENFORCE_ARG(z.vocab > 0 && z.vocab < (int64_t(1) << 31), op, ": an empty vocabulary, or one beyond 32 bits");
  z.lead = x.sizes().vec();
  z.lead.pop_back();
  z.rows = x.numel() / z.vocab;
  ORTB_ENFORCE_ARG((t.scalar_type() == at::kLong || t.scalar_type() == at::kInt) && t.sizes() == at::IntArrayRef(z.lead), op,
                   ": tokens must be int64 or int32 of the shape of the logits without the vocabulary");
  return z;
}
}  // namespace

TokenLogProbsSizes CheckTokenLogProbs(Ctx& ctx) {
  TokenLogProbsSizes z = LogitsAndTokens(ctx);
  z.top_k = ctx.node().attr_i("top_k", 0);
  ORTB_ENFORCE_ARG(z.top_k >= 0 && z.top_k <= 32 && z.top_k <= z.vocab, "TokenLogProbs: top_k must lie between 0 and 32 and within the vocabulary");
  return z;
}

TokenLogProbsSizes CheckTokenLogProbsGrad(Ctx& ctx) {
  TokenLogProbsSizes z = LogitsAndTokens(ctx);
  ctx.RequiredInput(2);
  ORTB_ENFORCE_ARG(!ctx.HasInput(5) || ctx.HasInput(3), "TokenLogProbsGrad: the gradient of the entropy needs the entropy");
  for (int i : {2, 3, 4, 5, 8, 9})
    ORTB_ENFORCE_ARG(!ctx.HasInput(i) || (ctx.Input(i).is_floating_point() && ctx.Input(i).numel() == z.rows), "TokenLogProbsGrad: input ", i, " must hold one floating value per row");
  if (ctx.HasInput(7)) {
    const at::Tensor& k = ctx.RequiredInput(6);
    ORTB_ENFORCE_ARG(k.dim() >= 1 && (k.scalar_type() == at::kLong || k.scalar_type() == at::kInt) && ctx.Input(7).is_floating_point() && ctx.Input(7).sizes() == k.sizes() &&
                         k.numel() == z.rows * k.size(-1) && k.size(-1) <= 32 && k.size(-1) <= z.vocab,
                     "TokenLogProbsGrad: top_tokens and their gradients must be [rows, up to 32]");
    z.top_k = k.size(-1);
  }
  return z;
}

void RegisterServingKernels(KernelRegistry& r) {
  r.RegisterFn(FUSED, "PagedBatchLayout", 1, kMax, PagedBatchLayoutImpl);
  r.RegisterFn(FUSED, "SharedPrefixPagedAttention", 1, kMax, SharedPrefixPagedAttentionImpl);
  r.RegisterFn(FUSED, "TreePagedAttention", 1, kMax, TreePagedAttentionImpl);
  r.RegisterFn(FUSED, "TokenLogProbs", 1, kMax, TokenLogProbsImpl);
  r.RegisterFn(FUSED, "TokenLogProbsGrad", 1, kMax, TokenLogProbsGradImpl);
}

}  // namespace ortb
