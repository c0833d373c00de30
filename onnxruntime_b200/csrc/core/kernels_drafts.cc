// com.ortb200 operators around a decode step with drafted tokens, device-agnostic versions: PagedCacheMove (cache entries to other
// places) and ProcessLogits (penalties, biases, masks and temperatures).  TreePagedAttention stands beside its relative in
// kernels_serving.cc; the GPU provider has its own kernels (kernels_cuda6.cc).
#include <ATen/ATen.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <set>

#include "kernel.h"
#include "serving_checks.h"

namespace ortb {

namespace {

using Ctx = OpKernelContext;
constexpr int kMax = 1 << 30;
constexpr const char* FUSED = "com.ortb200";

void PagedCacheMoveImpl(Ctx& ctx) {
  const CacheMoveSizes z = CheckCacheMove(ctx);
  const at::Tensor s = ctx.Input(0).to(at::kCPU).contiguous(), t = ctx.Input(1).to(at::kCPU).contiguous();
  std::vector<int64_t> sources, targets;
  std::set<int64_t> named;
  for (int64_t m = 0; m < z.moves; ++m) {
    const int64_t from = s.data_ptr<int64_t>()[m], to = t.data_ptr<int64_t>()[m];
    if (to < 0) continue;
    ORTB_ENFORCE_ARG(to < z.units && from >= 0 && from < z.units, "PagedCacheMove: move ", m, " from ", from, " to ", to, " leaves the cache of ", z.units);
    ORTB_ENFORCE_ARG(named.insert(to).second, "PagedCacheMove: ", to, " is the target of two moves");
    sources.push_back(from);
    targets.push_back(to);
  }
  const at::Tensor from = at::tensor(sources, at::kLong), to = at::tensor(targets, at::kLong);
  for (int i = 0; i < z.caches; ++i) {
    at::Tensor cache = ctx.Input(2 + i);
    if (!targets.empty()) {
      const c10::Device dev = cache.device();
      c10::List<c10::optional<at::Tensor>> read, write;
      if (z.blocks) {
        read.push_back(from.to(dev));
        write.push_back(to.to(dev));
      } else {
        const int64_t size = cache.size(1);
        read.push_back(from.div(size, "floor").to(dev));
        read.push_back(from.remainder(size).to(dev));
        write.push_back(to.div(size, "floor").to(dev));
        write.push_back(to.remainder(size).to(dev));
      }
      cache.index_put_(write, at::index(cache, read));
    }
    if (i < ctx.OutputCount()) ctx.SetOutput(i, cache);
  }
}

template <typename V>
std::vector<V> Host(Ctx& ctx, int i, at::ScalarType type) {
  if (!ctx.HasInput(i)) return {};
  const at::Tensor t = ctx.Input(i).to(at::kCPU, type).contiguous();
  return std::vector<V>(t.data_ptr<V>(), t.data_ptr<V>() + t.numel());
}

void ProcessLogitsImpl(Ctx& ctx) {
  const ProcessLogitsSizes z = CheckProcessLogits(ctx);
  const at::Tensor x = ctx.Input(0).to(at::kCPU, at::kFloat).contiguous();
  at::Tensor out = at::empty_like(x);
  const auto history = Host<int64_t>(ctx, 1, at::kLong), starts = Host<int64_t>(ctx, 2, at::kLong), generated = Host<int64_t>(ctx, 3, at::kLong);
  const auto lists = Host<int>(ctx, 4, at::kInt), row_mask = Host<int>(ctx, 13, at::kInt), allowed = Host<int>(ctx, 12, at::kInt);
  const auto drafted = Host<int64_t>(ctx, 5, at::kLong), bias_tokens = Host<int64_t>(ctx, 9, at::kLong), bias_starts = Host<int64_t>(ctx, 11, at::kLong);
  const auto repetition = Host<float>(ctx, 6, at::kFloat), presence = Host<float>(ctx, 7, at::kFloat), frequency = Host<float>(ctx, 8, at::kFloat);
  const auto bias_values = Host<float>(ctx, 10, at::kFloat), temperature = Host<float>(ctx, 14, at::kFloat);
  const char* op = "ProcessLogits";
  constexpr float kNever = -std::numeric_limits<float>::infinity();
  // of the tokens that a row touches, which are few beside its vocabulary; all 0 between rows
  std::vector<int64_t> count(z.vocab), sum_of(z.vocab), touched, banned;
  std::vector<char> seen(z.vocab);
  for (int64_t r = 0; r < z.rows; ++r) {
    const float* from = x.data_ptr<float>() + r * z.vocab;
    float* to = out.data_ptr<float>() + r * z.vocab;
    const float rep = repetition.empty() ? 1.f : repetition[r], pres = presence.empty() ? 0.f : presence[r], freq = frequency.empty() ? 0.f : frequency[r];
    std::copy(from, from + z.vocab, to);
    touched.clear();
    banned.clear();
    const auto add = [&](int64_t v, bool counts) {
      if (v < 0 || v >= z.vocab) return;
      if (!seen[v]) touched.push_back(v);
      seen[v] = 1;
      count[v] += counts;
    };
    if (rep != 1.f || pres != 0.f || freq != 0.f) {   // a row without penalties has no use for its text
      if (ctx.HasInput(1)) {
        const int64_t l = lists.empty() ? r : lists[r];
        ORTB_ENFORCE_ARG(l < z.lists, op, ": row ", r, " names list ", l, " of ", z.lists);
        if (l >= 0) {
          ORTB_ENFORCE_ARG(starts[l] >= 0 && starts[l] <= starts[l + 1] && starts[l + 1] <= z.history, op, ": list ", l, " leaves the history");
          for (int64_t i = starts[l]; i < starts[l + 1]; ++i) add(history[i], generated.empty() || i >= generated[l]);
        }
      }
      for (int64_t d = 0; d < z.drafted; ++d) add(drafted[r * z.drafted + d], true);
    }
    for (const int64_t v : touched) {
      to[v] = to[v] < 0.f ? to[v] * rep : to[v] / rep;
      if (count[v]) to[v] -= freq * static_cast<float>(count[v]) + pres;
      seen[v] = 0;
      count[v] = 0;
    }
    if (!bias_tokens.empty() || ctx.HasInput(9)) {
      ORTB_ENFORCE_ARG(bias_starts[r] >= 0 && bias_starts[r] <= bias_starts[r + 1] && bias_starts[r + 1] <= z.biases, op, ": the biases of row ", r, " leave their list");
      std::vector<std::pair<int64_t, float>> sums;   // of each token, its biases in their order
      for (int64_t i = bias_starts[r]; i < bias_starts[r + 1]; ++i) {
        const int64_t v = bias_tokens[i];
        if (v < 0 || v >= z.vocab) continue;
        if (sum_of[v] == 0) {
          sums.emplace_back(v, bias_values[i]);
          sum_of[v] = static_cast<int64_t>(sums.size());
        } else {
          sums[sum_of[v] - 1].second += bias_values[i];
        }
      }
      for (const auto& [v, s] : sums) {
        if (s == kNever) banned.push_back(v);   // holds for logits that are infinite or NaN, too
        else to[v] += s;
        sum_of[v] = 0;
      }
    }
    if (!temperature.empty() && temperature[r] > 0.f && temperature[r] != 1.f) {
      const float t = temperature[r];
      for (int64_t v = 0; v < z.vocab; ++v) to[v] /= t;
    }
    for (const int64_t v : banned) to[v] = kNever;
    if (!row_mask.empty()) {
      ORTB_ENFORCE_ARG(row_mask[r] < z.masks, op, ": row ", r, " names mask ", row_mask[r], " of ", z.masks);
      for (int64_t w = 0; w < z.mask_words && row_mask[r] >= 0; ++w) {
        const unsigned bits = static_cast<unsigned>(allowed[row_mask[r] * z.mask_words + w]);
        float* const of = to + 32 * w;
        const int n = static_cast<int>(std::min<int64_t>(32, z.vocab - 32 * w));
        for (int b = 0; b < n && bits != ~0u; ++b) {   // (without a branch, which masks give no way to foresee)
          uint32_t f, never;
          std::memcpy(&f, of + b, 4);
          std::memcpy(&never, &kNever, 4);
          const uint32_t keep = 0u - (bits >> b & 1);
          f = (f & keep) | (never & ~keep);
          std::memcpy(of + b, &f, 4);
        }
      }
    }
  }
  ctx.SetOutput(0, out.to(ctx.Input(0).device()));
}

}  // namespace

CacheMoveSizes CheckCacheMove(Ctx& ctx) {
  CacheMoveSizes z;
  const char* op = "PagedCacheMove";
  const at::Tensor &s = ctx.RequiredInput(0), &t = ctx.RequiredInput(1);
  ORTB_ENFORCE_ARG(s.scalar_type() == at::kLong && t.scalar_type() == at::kLong && s.dim() == 1 && s.sizes() == t.sizes(), op,
                   ": sources and targets must be int64 of rank 1, one of each per move");
  z.moves = s.size(0);
  z.blocks = ctx.node().attr_i("whole_blocks", 0) != 0;
  z.caches = ctx.InputCount() - 2;
  ORTB_ENFORCE_ARG(z.caches > 0, op, ": no cache is given");
  std::vector<std::pair<const char*, const char*>> places;
  for (int i = 0; i < z.caches; ++i) {
    const at::Tensor &c = ctx.RequiredInput(2 + i), &first = ctx.Input(2);
    ORTB_ENFORCE_ARG(c.dim() >= 2 && c.size(0) == first.size(0) && (z.blocks || c.size(1) == first.size(1)), op,
                     ": caches must be [blocks, block size, ...], with the same number of blocks and, where tokens move, of tokens in a block");
    if (c.is_contiguous() && c.numel() > 0) {
      const char* at = static_cast<const char*>(c.data_ptr());
      places.emplace_back(at, at + c.numel() * c.element_size());
    }
  }
  std::sort(places.begin(), places.end());
  for (size_t i = 1; i < places.size(); ++i) ORTB_ENFORCE_ARG(places[i].first >= places[i - 1].second, op, ": two caches share memory");
  z.units = ctx.Input(2).size(0) * (z.blocks ? 1 : ctx.Input(2).size(1));
  return z;
}

ProcessLogitsSizes CheckProcessLogits(Ctx& ctx) {
  ProcessLogitsSizes z;
  const char* op = "ProcessLogits";
  const at::Tensor& x = ctx.RequiredInput(0);
  ORTB_ENFORCE_ARG(x.dim() == 2 && x.is_floating_point() && x.size(1) > 0 && x.size(1) < (int64_t(1) << 31), op, ": logits must be floating, [rows, vocabulary]");
  z.rows = x.size(0);
  z.vocab = x.size(1);
  const auto want = [&](int i, at::ScalarType type, int64_t size, const char* what) {
    const at::Tensor& t = ctx.RequiredInput(i);
    const bool typed = t.scalar_type() == type || (type == at::kLong && t.scalar_type() == at::kInt);
    ORTB_ENFORCE_ARG(typed && t.dim() == 1 && (size < 0 || t.size(0) == size), op, ": ", what, " must be ", c10::toString(type), " of rank 1",
                     size < 0 ? "" : ", " + std::to_string(size) + " long");
  };
  ORTB_ENFORCE_ARG(ctx.HasInput(1) == ctx.HasInput(2), op, ": history and history_starts come together");
  if (ctx.HasInput(1)) {
    want(1, at::kLong, -1, "history");
    want(2, at::kLong, -1, "history_starts");
    z.history = ctx.Input(1).size(0);
    z.lists = ctx.Input(2).size(0) - 1;
    ORTB_ENFORCE_ARG(z.lists >= 0, op, ": history_starts has one entry more than there are lists");
    ORTB_ENFORCE_ARG(ctx.HasInput(4) || z.lists == z.rows, op, ": without row_list there is a list for every row");
  }
  if (ctx.HasInput(3)) {
    ORTB_ENFORCE_ARG(ctx.HasInput(1), op, ": generated_starts are places in a history");
    want(3, at::kLong, z.lists, "generated_starts");
  }
  if (ctx.HasInput(4)) {
    ORTB_ENFORCE_ARG(ctx.HasInput(1), op, ": row_list names lists of a history");
    want(4, at::kInt, z.rows, "row_list");
  }
  if (ctx.HasInput(5)) {
    const at::Tensor& d = ctx.Input(5);
    ORTB_ENFORCE_ARG(d.dim() == 2 && d.size(0) == z.rows && (d.scalar_type() == at::kLong || d.scalar_type() == at::kInt), op,
                     ": drafted must be int64 or int32, a row for every row of logits");
    z.drafted = d.size(1);
  }
  for (int i : {6, 7, 8, 14})
    if (ctx.HasInput(i)) want(i, at::kFloat, z.rows, i == 6 ? "repetition" : i == 7 ? "presence" : i == 8 ? "frequency" : "temperature");
  ORTB_ENFORCE_ARG(ctx.HasInput(9) == ctx.HasInput(10) && ctx.HasInput(9) == ctx.HasInput(11), op, ": bias_tokens, bias_values and bias_starts come together");
  if (ctx.HasInput(9)) {
    want(9, at::kLong, -1, "bias_tokens");
    z.biases = ctx.Input(9).size(0);
    want(10, at::kFloat, z.biases, "bias_values");
    want(11, at::kLong, z.rows + 1, "bias_starts");
  }
  ORTB_ENFORCE_ARG(ctx.HasInput(12) == ctx.HasInput(13), op, ": allowed and row_mask come together");
  if (ctx.HasInput(12)) {
    const at::Tensor& m = ctx.Input(12);
    ORTB_ENFORCE_ARG(m.scalar_type() == at::kInt && m.dim() == 2 && m.size(1) == (z.vocab + 31) / 32, op, ": allowed must be int32, [masks, ", (z.vocab + 31) / 32, "]");
    z.masks = m.size(0);
    z.mask_words = m.size(1);
    want(13, at::kInt, z.rows, "row_mask");
  }
  return z;
}

void RegisterDraftKernels(KernelRegistry& r) {
  r.RegisterFn(FUSED, "PagedCacheMove", 1, kMax, PagedCacheMoveImpl);
  r.RegisterFn(FUSED, "ProcessLogits", 1, kMax, ProcessLogitsImpl);
}

}  // namespace ortb
