// C ABI of the 4-bit key/value cache: argument checks (kernels: cache4_store.cu, cache4_attn.cu).
#include <cstring>

#include "cache4.cuh"
#include "host_util.h"

namespace ra {
namespace {

int check_cache(const ra_cache4_t* c, const char* name, CacheView* out) {
  if (!c) return fail(-60, "%s is NULL", name);
  if (c->b < 1 || c->hkv < 1 || (int64_t)c->b * c->hkv > INT32_MAX)
    return fail(-61, "%s: b and hkv must be >= 1 and b * hkv below 2^31 (got %d, %d)", name, c->b, c->hkv);
  if (c->capacity < kCacheAlign || c->capacity % kCacheAlign || c->capacity > (1 << 30))
    return fail(-62, "%s: capacity must be a multiple of %d up to 2^30 (got %d)", name, kCacheAlign, c->capacity);
  if (c->d != 64 && c->d != 128 && c->d != 256) return fail(-63, "%s: head dim must be 64, 128 or 256 (got %d)", name, c->d);
  const void* arrays[] = {c->k, c->v, c->k_limits, c->v_limits, c->positions, c->weights, c->lengths, c->seen};
  for (const void* p : arrays)
    if (!p) return fail(-64, "%s: an array is NULL", name);
  for (int i = 0; i < 5; ++i)
    if (reinterpret_cast<uintptr_t>(arrays[i]) % 16) return fail(-65, "%s: k, v, k_limits, v_limits and positions must lie on 16-byte boundaries", name);
  *out = CacheView{(uint8_t*)c->k, (uint8_t*)c->v, (uint32_t*)c->k_limits, (uint32_t*)c->v_limits, c->positions, c->weights, c->lengths,
                   c->seen, c->b, c->hkv, c->capacity, c->d};
  return 0;
}

int check_rows(const ra_tensor_t* k, const ra_tensor_t* v, int dtype, int t) {
  int rc;
  if ((rc = check_tensor(k, "k")) || (rc = check_tensor(v, "v"))) return rc;
  if (dtype != RA_DTYPE_F32 && dtype != RA_DTYPE_BF16) return fail(-4, "dtype must be RA_DTYPE_F32 or RA_DTYPE_BF16 (got %d)", dtype);
  if (t < 1) return fail(-66, "at least one row is needed (got %d)", t);
  return 0;
}

TensorView view(const ra_tensor_t* t) { return TensorView{t->ptr, t->stride_b, t->stride_l, t->stride_h}; }

int check_heads(const CacheView& c, int h, int lq, int dtype) {
  if (h < 1 || h % c.hkv) return fail(-67, "h must be a multiple of the cache's %d key/value heads (got %d)", c.hkv, h);
  if (lq < 1 || (int64_t)c.b * h * lq > INT32_MAX) return fail(-68, "lq must be >= 1 and b * h * lq below 2^31 (got lq %d)", lq);
  if (dtype != RA_DTYPE_F32 && dtype != RA_DTYPE_BF16) return fail(-4, "dtype must be RA_DTYPE_F32 or RA_DTYPE_BF16 (got %d)", dtype);
  return 0;
}

}  // namespace
}  // namespace ra

using namespace ra;

extern "C" {

int ra_cache4_append(const ra_cache4_t* cache, const ra_tensor_t* k, const ra_tensor_t* v, int32_t dtype, int32_t t,
                     const int32_t* counts, const int32_t* start, const int32_t* positions, void* stream) {
  CacheView c;
  int rc;
  if ((rc = check_cache(cache, "cache", &c)) || (rc = check_rows(k, v, dtype, t))) return rc;
  if (t > c.cap) return fail(-69, "%d rows do not fit a capacity of %d", t, c.cap);
  cudaError_t e = launch_cache_append(c, view(k), view(v), dtype, t, counts, start, positions, (cudaStream_t)stream);
  return e == cudaSuccess ? 0 : fail_cuda(e, "cache append");
}

int ra_cache4_read(const ra_cache4_t* cache, const ra_tensor_t* k, const ra_tensor_t* v, int32_t dtype, int32_t t,
                   const int32_t* start, void* stream) {
  CacheView c;
  int rc;
  if ((rc = check_cache(cache, "cache", &c)) || (rc = check_rows(k, v, dtype, t))) return rc;
  cudaError_t e = launch_cache_read(c, view(k), view(v), dtype, t, start, (cudaStream_t)stream);
  return e == cudaSuccess ? 0 : fail_cuda(e, "cache read");
}

int64_t ra_cache4_evict_workspace(const ra_cache4_t* cache, int32_t keep) {
  CacheView c;
  int rc;
  if ((rc = check_cache(cache, "cache", &c))) return rc;
  if (keep < 1 || keep > c.cap) return fail(-70, "keep must be between 1 and the capacity %d (got %d)", c.cap, keep);
  return 2ll * c.b * c.hkv * keep * (int64_t)sizeof(int32_t);
}

int ra_cache4_evict(const ra_cache4_t* cache, int32_t keep, int32_t recent, const ra_cache4_t* out, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  CacheView c, o;
  int rc;
  const int64_t need = ra_cache4_evict_workspace(cache, keep);
  if (need < 0) return (int)need;
  if ((rc = check_cache(cache, "cache", &c))) return rc;
  if (!out) out = cache;
  if ((rc = check_cache(out, "out", &o))) return rc;
  if (o.b != c.b || o.hkv != c.hkv || o.d != c.d || o.cap < keep)
    return fail(-71, "out must have the cache's b, hkv and d and room for %d rows", keep);
  const void* from[] = {c.k, c.v, c.kl, c.vl, c.pos, c.weight, c.len, c.seen};
  const void* to[] = {o.k, o.v, o.kl, o.vl, o.pos, o.weight, o.len, o.seen};
  int shared = 0;
  for (int i = 0; i < 8; ++i) shared += from[i] == to[i];
  if (shared && (shared < 8 || o.cap != c.cap))
    return fail(-72, "out must be the cache itself or share nothing with it");
  if (recent < 0 || recent > keep) return fail(-73, "recent must be between 0 and keep (got %d)", recent);
  if (!workspace || workspace_bytes < need) return fail(-74, "evict needs a workspace of %lld bytes", (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 4) return fail(-75, "workspace must lie on a 4-byte boundary");
  cudaError_t e = launch_cache_evict(c, o, keep, recent, (int32_t*)workspace, (cudaStream_t)stream);
  return e == cudaSuccess ? 0 : fail_cuda(e, "cache evict");
}

int64_t ra_cache4_attention_workspace(const ra_cache4_t* cache, int32_t h, int32_t lq, int32_t dtype) {
  CacheView c;
  int rc;
  if ((rc = check_cache(cache, "cache", &c)) || (rc = check_heads(c, h, lq, dtype))) return rc;
  size_t bytes = 0;
  cudaError_t e = cache_attn_workspace(c.b, c.hkv, c.cap, c.d, h, lq, dtype, &bytes);
  if (e != cudaSuccess) return -fail_cuda(e, "cache attention workspace");
  return (int64_t)bytes;
}

int ra_cache4_attention(const ra_cache4_t* cache, const ra_tensor_t* q, const ra_tensor_t* out, float* lse, int32_t h,
                        int32_t lq, int32_t dtype, float sm_scale, const ra_score_mod_t* mod, float* weights_out,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  CacheAttnParams p;
  memset(&p, 0, sizeof(p));
  int rc;
  if ((rc = check_cache(cache, "cache", &p.c)) || (rc = check_heads(p.c, h, lq, dtype))) return rc;
  if ((rc = check_tensor(q, "q")) || (rc = check_tensor(out, "out"))) return rc;
  if (!(sm_scale == sm_scale)) return fail(-5, "sm_scale is NaN");
  if (mod) {
    const uint32_t known = RA_MOD_CAUSAL | RA_MOD_WINDOW | RA_MOD_ALIBI;
    if (mod->kinds & ~known) return fail(-76, "cache attention takes the causal, window and ALiBi kinds only (got 0x%x)", mod->kinds);
    if ((mod->kinds & RA_MOD_WINDOW) && mod->window < 1) return fail(-13, "score_mod: window must be >= 1");
    if ((mod->kinds & RA_MOD_ALIBI) && !mod->alibi_slopes) return fail(-12, "score_mod: alibi_slopes is NULL");
    p.kinds = mod->kinds;
    p.window = mod->window;
    p.q_pos = mod->q_pos;
    p.slopes = mod->alibi_slopes;
  }
  const int64_t need = ra_cache4_attention_workspace(cache, h, lq, dtype);
  if (need < 0) return (int)(need < -3 ? need : -need);
  if (!workspace || workspace_bytes < need) return fail(-74, "cache attention needs a workspace of %lld bytes", (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(-75, "workspace must lie on a 16-byte boundary");
  p.q = view(q);
  p.out = view(out);
  p.lse = lse;
  p.h = h;
  p.lq = lq;
  p.dtype = dtype;
  p.scale = sm_scale;
  p.weights_out = weights_out;
  p.ws = workspace;
  cudaError_t e = launch_cache_attn(p, (cudaStream_t)stream);
  return e == cudaSuccess ? 0 : fail_cuda(e, "cache attention");
}

}  // extern "C"
