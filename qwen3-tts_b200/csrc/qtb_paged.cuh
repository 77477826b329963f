// qtb_paged.cuh -- shared pieces of the paged-cache operators (qtb_paged.cu):
// the attention problem as the kernels see it, its per-request bounds, and the
// element-type helpers.
#pragma once
#include "qtb_device.cuh"
#include "../../include/qwen3tts_b200.h"

namespace qtb {

// Status bits that a kernel ORs into the caller's word (QTB_PS_* of the header).
QTB_DEV void raise_status(int *status, int bits) {
  if (status && bits) atomicOr(status, bits);
}

// One attention call.  Strides are in elements; the innermost one is 1.
struct AttnCall {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  float *lse;              // [n_tokens][n_heads], or null
  const int *cu;           // [n_req + 1] packed offsets of the requests' new tokens
  const int *kv_len;       // [n_req] visible keys of the last new token (paged form)
  const int *table;        // [n_req][table_stride] pages (paged form)
  int *status;
  long long q_st, q_sh, o_st, o_sh;
  long long k_st[3], v_st[3];   // paged: page, head, position; packed: token, head, -
  long long table_stride;
  int n_req, n_tokens, n_heads, n_kv, group, page, n_pages, table_cols;
  int causal, window;
  float scale_log2;        // scale * log2(e): scores are kept in units of log2
};

// What a request asks for.  Token i of its n new ones sits at position
// first + i, sees keys up to there (causal) and none at or before
// first + i - window (window > 0); keys outside [lo, hi) concern none of them.
struct AttnReq {
  int t0, n, first, lo, hi;
};

template <bool PAGED>
QTB_DEV AttnReq attn_request(const AttnCall &c, int r) {
  AttnReq a;
  a.t0 = min(max(c.cu[r], 0), c.n_tokens);
  const int t1 = min(max(c.cu[r + 1], 0), c.n_tokens);
  a.n = max(t1 - a.t0, 0);
  const long long room = (long long)c.table_cols * c.page;
  a.hi = PAGED ? max((int)min((long long)c.kv_len[r], room), 0) : a.n;
  a.first = a.hi - a.n;
  a.lo = c.window > 0 ? max(a.first - c.window + 1, 0) : 0;   // positions and windows are below 2^30
  return a;
}

// -------------------------------------------------------- element types ----
template <bool F16>
QTB_DEV uint32_t pack2(float lo, float hi) {   // round to nearest even
  uint32_t r;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool F16>
QTB_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16) mma_f16(d, a, b0, b1);
  else mma_bf16(d, a, b0, b1);
}
QTB_DEV float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
QTB_DEV void ldsm_x4(uint32_t (&r)[4], const void *row_addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(row_addr))
               : "memory");
}
// 16 bytes global -> shared, or 16 zero bytes when !ok (nothing is read then).
QTB_DEV void cp16_zfill(void *dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
QTB_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
QTB_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A launch marked programmatic may start while its predecessor still runs:
// pdl_wait returns when that one's writes are visible, pdl_release lets the
// successor start.
QTB_DEV void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
QTB_DEV void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace qtb
