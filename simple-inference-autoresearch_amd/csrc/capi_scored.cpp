// The score options of the scored entry points: checks, and the kernels' arguments.
#include <math.h>
#include <string.h>

#include "host_util.hpp"
#include "scored.hpp"

namespace sia {

namespace {

// A device array of int32, one entry for all or one per sequence.
int per_sequence(const sia_tensor* t, const char* name, int64_t B, const int32_t** data, int32_t* per_seq) {
  if (t == nullptr) return SIA_OK;
  if (t->data == nullptr || t->dtype != SIA_I32 || t->ndim > 1)
    return fail(SIA_ERR_INVALID_ARGUMENT, "%s must be an int32 scalar, (1,) or (B,) tensor", name);
  const int64_t n = t->ndim == 0 ? 1 : t->shape[0];
  if (n != 1 && n != B) return fail(SIA_ERR_INVALID_ARGUMENT, "%s must have 1 or B elements, got %lld", name, (long long)n);
  if (n > 1 && t->stride[0] != 1) return fail(SIA_ERR_INVALID_ARGUMENT, "%s must be contiguous", name);
  *data = (const int32_t*)t->data;
  *per_seq = n > 1;
  return SIA_OK;
}

}  // namespace

int fill_score(const sia_score_options* o, bool prompt, int64_t B, int64_t Hq, float sm_scale, int causal, ScoreArgs& s) {
  memset(&s, 0, sizeof(s));
  // (no window: the largest one; prompts, whose positions lie below 2^30, add it to them in 32 bits)
  s.window = prompt ? 1 << 30 : 0x7fffffff;
  s.causal = causal != 0;
  if (o == nullptr) return SIA_OK;
  for (int i = 0; i < 4; ++i)
    if (o->reserved[i] != 0) return fail(SIA_ERR_INVALID_ARGUMENT, "sia_score_options reserved fields must be zero");
  if (o->softcap != 0.f) {
    s.cap_in = 2.0f * kLog2e * sm_scale / o->softcap;
    s.cap_out = o->softcap * kLog2e;
    s.cap_inv = sm_scale / o->softcap;
    s.cap_log2 = 2.0f / o->softcap;
    if (!(o->softcap > 0.f) || !isfinite(s.cap_in) || !isfinite(s.cap_out) || !isfinite(s.cap_log2))
      return fail(SIA_ERR_INVALID_ARGUMENT, "softcap must be a positive finite number");
  }
  if (o->window < 0) return fail(SIA_ERR_INVALID_ARGUMENT, "window must be positive");
  if (o->window > 0 && o->window < s.window) s.window = o->window;
  if (const sia_tensor* t = o->alibi_slopes) {
    if (t->data == nullptr || t->dtype != SIA_F32 || t->ndim != 1 || t->shape[0] != Hq)
      return fail(SIA_ERR_INVALID_ARGUMENT, "alibi_slopes must be a float32 (Hq,) tensor");
    if (Hq > 1 && t->stride[0] != 1) return fail(SIA_ERR_INVALID_ARGUMENT, "alibi_slopes must be contiguous");
    s.slopes = (const float*)t->data;
  }
  int rc;
  if ((rc = per_sequence(o->kv_start, "kv_start", B, &s.start, &s.start_per_seq))) return rc;
  if (!prompt) {
    if (o->kv_len != nullptr || o->prefix_len != nullptr || o->cu_seqlens != nullptr)
      return fail(SIA_ERR_INVALID_ARGUMENT, "kv_len, prefix_len and cu_seqlens of the score options are for prompts");
    return SIA_OK;
  }
  if ((rc = per_sequence(o->kv_len, "kv_len", B, &s.len, &s.len_per_seq))) return rc;
  if ((rc = per_sequence(o->prefix_len, "prefix_len", B, &s.prefix, &s.prefix_per_seq))) return rc;
  if (const sia_tensor* t = o->cu_seqlens) {
    if (t->dtype != SIA_I32 || (t->ndim != 1 && t->ndim != 2))
      return fail(SIA_ERR_INVALID_ARGUMENT, "cu_seqlens must be an int32 (n,) or (B, n) tensor");
    const int64_t n = t->shape[t->ndim - 1];
    if (t->ndim == 2 && t->shape[0] != B) return fail(SIA_ERR_INVALID_ARGUMENT, "cu_seqlens must have a row per sequence");
    if (n > 0x7fffffff) return fail(SIA_ERR_UNSUPPORTED, "too many documents");
    if (n > 1 && t->stride[t->ndim - 1] != 1) return fail(SIA_ERR_INVALID_ARGUMENT, "cu_seqlens must be contiguous");
    if (n > 0) {
      if (t->data == nullptr) return fail(SIA_ERR_INVALID_ARGUMENT, "cu_seqlens has no data pointer");
      s.cuts = (const int32_t*)t->data;
      s.ncuts = (int32_t)n;
      s.cuts_sb = t->ndim == 2 ? t->stride[0] : 0;
    }
  }
  return SIA_OK;
}

}  // namespace sia
