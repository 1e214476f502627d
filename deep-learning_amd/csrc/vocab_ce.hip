// Entry points of the vocabulary cross entropy (vocab_ce.hpp).
#include "vocab_ce.hpp"

using namespace dlmi;

static char const *ce_check(dlmi_dtype type, size_t B, size_t K, size_t V) {
  if (type != DLMI_F32 && type != DLMI_BF16) return "unknown type";
  if (B > DLMI_VOCAB_CE_MAX_ROWS) return "too many rows";
  if (K > DLMI_VOCAB_CE_MAX_FEATURES) return "too many features";
  if (V > 0x7fffffffu) return "too many classes";
  return nullptr;
}

extern "C" {

int dlmi_vocab_ce_fwd(dlmi_ctx *ctx, dlmi_dtype type, size_t B, size_t K, size_t V, void const *X, void const *W, float const *bias,
                      int32_t const *labels, float *loss, float *lse) {
  if (ctx == nullptr) return DLMI_E_INVALID;
  char const *const wrong = ce_check(type, B, K, V);
  DLMI_REQUIRE(ctx, wrong == nullptr, wrong);
  if (B == 0) return DLMI_OK;
  DLMI_REQUIRE_DEVICE(ctx);
  DLMI_REQUIRE(ctx, K != 0 && V != 0, "no features or no classes");
  DLMI_REQUIRE(ctx, X != nullptr && W != nullptr && labels != nullptr && loss != nullptr && lse != nullptr, "null pointer");
  size_t const e = type == DLMI_F32 ? 4 : 2;
  dlmi_span const spans[] = {{loss, B * 4, false}, {lse, B * 4, false}, {X, B * K * e, false}, {W, V * K * e, false}, {bias, V * 4, false},
                             {labels, B * 4, false}};
  DLMI_REQUIRE(ctx, !dlmi_spans_collide(spans, 2, 6), "an output must not be written over another array");
  CeArgs a = {};
  a.B = B;
  a.K = K;
  a.V = V;
  a.X = X;
  a.W = W;
  a.bias = bias;
  a.labels = labels;
  a.loss = loss;
  a.lse = lse;
  return type == DLMI_F32 ? ce_forward<float>(ctx, a) : ce_forward<__bf16>(ctx, a);
}

int dlmi_vocab_ce_bwd(dlmi_ctx *ctx, dlmi_dtype type, size_t B, size_t K, size_t V, void const *X, void const *W, float const *bias,
                      int32_t const *labels, float const *lse, float const *dloss, float scale, void *dX, void *dW, float *db,
                      int accumulate) {
  if (ctx == nullptr) return DLMI_E_INVALID;
  char const *const wrong = ce_check(type, B, K, V);
  DLMI_REQUIRE(ctx, wrong == nullptr, wrong);
  DLMI_REQUIRE(ctx, B != 0 && K != 0 && V != 0, "no rows, no features or no classes");
  DLMI_REQUIRE_DEVICE(ctx);
  DLMI_REQUIRE(ctx, X != nullptr && W != nullptr && labels != nullptr && lse != nullptr, "null pointer");
  DLMI_REQUIRE(ctx, dX != nullptr || dW != nullptr || db != nullptr, "no gradient asked for");
  size_t const e = type == DLMI_F32 ? 4 : 2;
  dlmi_span const spans[] = {{dX, B * K * e, false}, {dW, V * K * e, false}, {db, V * 4, false},   {X, B * K * e, false}, {W, V * K * e, false},
                             {bias, V * 4, false},   {labels, B * 4, false}, {lse, B * 4, false}, {dloss, B * 4, false}};
  DLMI_REQUIRE(ctx, !dlmi_spans_collide(spans, 3, 9), "a gradient must not be written over another array");
  CeArgs a = {};
  a.B = B;
  a.K = K;
  a.V = V;
  a.X = X;
  a.W = W;
  a.bias = bias;
  a.labels = labels;
  a.lse_in = lse;
  a.dloss = dloss;
  a.scale = scale;
  a.dX = dX;
  a.dW = dW;
  a.db = db;
  a.accumulate = accumulate;
  return type == DLMI_F32 ? ce_backward<float>(ctx, a) : ce_backward<__bf16>(ctx, a);
}

}  // extern "C"
