// C entry points of the cross attention (kernels: cross_fwd.hip, cross_bwd.hip).
#include "cross.h"

namespace vsa {

int64_t cross_fwd_parts(const vsa_cross* c);
int64_t cross_bwd_parts(const vsa_cross* c);
int cross_fwd(const vsa_cross* c, CrossArgs a, char* scratch, hipStream_t s);
int cross_bwd(const vsa_cross* c, const CrossArgs& a, char* scratch, hipStream_t s);
int cross_words(const vsa_cross* c, uint32_t* words, int nwords, hipStream_t s);

namespace {

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// rows start 16-byte aligned, and a tile's rows lie within 30 bits of its first
bool rows_ok(const void* p, const int64_t* stride, int es) {
  int64_t low = 0;
  for (int x = 0; x < 3; ++x) {
    if (stride[x] < 0) return false;
    low |= stride[x] * es;
  }
  return (((uint64_t)(uintptr_t)p | (uint64_t)low) & 15) == 0 && stride[2] <= (1LL << 30) / (64 * es);
}

int check(const vsa_cross* c) {
  if (!c || !c->q || !c->k || !c->v) return VSA_ERR_NULL;
  if (c->dtype != VSA_BF16 && c->dtype != VSA_F16 && c->dtype != VSA_F32) return VSA_ERR_DTYPE;
  if (c->batch <= 0 || c->batch > 65535 || c->heads <= 0 || c->kv_heads <= 0 ||
      c->heads % c->kv_heads || c->heads > 65535 || c->head_dim <= 0 || c->head_dim > 256 ||
      c->head_dim % 8 || c->sq <= 0 || c->skv <= 0 || c->skv > (1LL << 31) - 256 ||
      c->sq > ((1LL << 31) - 256) / (c->heads / c->kv_heads) || !(fabsf(c->scale) <= 0x1p127f) ||
      (c->key_mask && c->mask_stride < 0) || c->q_stride[2] < c->head_dim ||
      c->k_stride[2] < c->head_dim || c->v_stride[2] < c->head_dim)
    return VSA_ERR_SHAPE;
  const int es = c->dtype == VSA_F32 ? 4 : 2;
  if (!rows_ok(c->q, c->q_stride, es) || !rows_ok(c->k, c->k_stride, es) ||
      !rows_ok(c->v, c->v_stride, es) || !vsa_aligned<4>(c->kv_lens))
    return VSA_ERR_ALIGN;
  return VSA_OK;
}

CrossArgs args(const vsa_cross* c) {
  CrossArgs a = {};
  a.q = {c->q, c->q_stride[0], c->q_stride[1], c->q_stride[2]};
  a.k = {c->k, c->k_stride[0], c->k_stride[1], c->k_stride[2]};
  a.v = {c->v, c->v_stride[0], c->v_stride[1], c->v_stride[2]};
  a.lens = c->kv_lens;
  a.batch = c->batch, a.heads = c->heads, a.kv_heads = c->kv_heads;
  a.group = c->heads / c->kv_heads;
  a.sq = (int)c->sq, a.skv = (int)c->skv, a.dim = c->head_dim;
  a.spread = c->batch > 1 && (c->kv_lens || c->key_mask) &&
             2 * c->skv * c->head_dim * (c->dtype == VSA_F32 ? 4 : 2) <= 1 << 20;
  a.scale = c->scale;
  a.c2 = c->scale * kLog2e;
  if (a.c2 == 0.f) a.c2 = 1.17549435e-38f;   // masked scores stay -inf, all others 2^0
  return a;
}

int words_of(const vsa_cross* c) { return (int)((c->skv + 63) / 64 * 2); }
int64_t words_bytes(const vsa_cross* c) {
  return c->key_mask ? round256((int64_t)c->batch * words_of(c) * 4) : 0;
}

// the mask's words, at the start of the scratch
int prepare(const vsa_cross* c, CrossArgs& a, char*& scratch, hipStream_t s) {
  if (!c->key_mask) return VSA_OK;
  a.words = (const uint32_t*)scratch;
  a.nwords = words_of(c);
  const int rc = cross_words(c, (uint32_t*)scratch, a.nwords, s);
  scratch += words_bytes(c);
  return rc;
}

}  // namespace
}  // namespace vsa

using namespace vsa;

extern "C" int vsa_cross_sizes(const vsa_cross* c, int64_t* scratch_fwd, int64_t* scratch_bwd) {
  if (!scratch_fwd || !scratch_bwd) return VSA_ERR_NULL;
  const int rc = check(c);
  if (rc) return rc;
  *scratch_fwd = words_bytes(c) + round256(cross_fwd_parts(c));
  *scratch_bwd = words_bytes(c) + round256((int64_t)c->batch * c->heads * c->sq * 4) +
                 round256(cross_bwd_parts(c));
  return VSA_OK;
}

extern "C" int vsa_cross_fwd(const vsa_cross* c, void* out, const int64_t* out_stride, void* lo,
                             float* lse, void* scratch, void* stream) {
  int rc = check(c);
  if (rc) return rc;
  if (!out || !out_stride) return VSA_ERR_NULL;
  if (!scratch && (c->key_mask || cross_fwd_parts(c))) return VSA_ERR_NULL;
  if (!rows_ok(out, out_stride, c->dtype == VSA_F32 ? 4 : 2) || !vsa_aligned<4>(lse) ||
      !vsa_aligned<8>(lo) || !vsa_aligned<256>(scratch))
    return VSA_ERR_ALIGN;
  CrossArgs a = args(c);
  a.out = out;
  a.lo = (uint8_t*)lo;
  for (int x = 0; x < 3; ++x) a.out_s[x] = out_stride[x];
  a.lse = lse;
  if (a.c2 < 0) {   // the running max wants a scale that keeps the order
    a.c2 = -a.c2;
    a.qsign = c->dtype == VSA_F32 ? 0x80000000u : 0x80008000u;
  }
  char* at = (char*)scratch;
  if ((rc = prepare(c, a, at, (hipStream_t)stream))) return rc;
  return cross_fwd(c, a, at, (hipStream_t)stream);
}

extern "C" int vsa_cross_bwd(const vsa_cross* c, const void* out, const int64_t* out_stride,
                             const void* lo, const void* dout, const int64_t* dout_stride,
                             const float* lse, void* dq, const int64_t* dq_stride, void* dk, const int64_t* dk_stride,
                             void* dv, const int64_t* dv_stride, void* scratch, void* stream) {
  int rc = check(c);
  if (rc) return rc;
  if (!out || !out_stride || !dout || !dout_stride || !lse || !dq || !dq_stride || !dk ||
      !dk_stride || !dv || !dv_stride || !scratch)
    return VSA_ERR_NULL;
  const int es = c->dtype == VSA_F32 ? 4 : 2;
  if (!rows_ok(out, out_stride, es) || !rows_ok(dout, dout_stride, es) ||
      !rows_ok(dq, dq_stride, es) || !rows_ok(dk, dk_stride, es) || !rows_ok(dv, dv_stride, es) ||
      !vsa_aligned<8>(lo) || !vsa_aligned<4>(lse) || !vsa_aligned<256>(scratch))
    return VSA_ERR_ALIGN;
  CrossArgs a = args(c);
  a.o = {out, out_stride[0], out_stride[1], out_stride[2]};
  a.dout = {dout, dout_stride[0], dout_stride[1], dout_stride[2]};
  a.dq = dq, a.dk = dk, a.dv = dv;
  for (int x = 0; x < 3; ++x)
    a.dq_s[x] = dq_stride[x], a.dk_s[x] = dk_stride[x], a.dv_s[x] = dv_stride[x];
  a.lo = (uint8_t*)const_cast<void*>(lo);
  a.lse = const_cast<float*>(lse);
  char* at = (char*)scratch;
  if ((rc = prepare(c, a, at, (hipStream_t)stream))) return rc;
  a.delta = (float*)at;
  at += round256((int64_t)c->batch * c->heads * c->sq * 4);
  return cross_bwd(c, a, at, (hipStream_t)stream);
}
