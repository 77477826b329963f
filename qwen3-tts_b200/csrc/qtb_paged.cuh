// qtb_paged.cuh -- shared pieces of the paged-cache operators (qtb_paged.cu):
// the attention problem as the kernels see it, its per-request bounds, and the
// element-type helpers.
#pragma once
#include "qtb_device.cuh"
#include "../../include/qwen3tts_b200.h"
#include <cuda.h>

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
// Over pages the new tokens are the request's last, so that the packed token
// cu[r + 1] - 1 is at position kv_len - 1, whether or not the table has room for
// that key (hi) and the packed tensors for that token (t0, n): those that exist
// keep their positions.  Positions are at most 2^30, as the host bounds the room,
// and longer lengths are taken as that.
struct AttnReq {
  int t0, n, first, lo, hi;
};
constexpr int POS_MAX = 1 << 30;

template <bool PAGED>
QTB_DEV AttnReq attn_request(const AttnCall &c, int r) {
  AttnReq a;
  a.t0 = min(max(c.cu[r], 0), c.n_tokens);
  const int t1 = min(max(c.cu[r + 1], 0), c.n_tokens);
  a.n = max(t1 - a.t0, 0);
  a.hi = a.n;
  a.first = 0;
  if (PAGED) {
    const int len = min(max(c.kv_len[r], 0), POS_MAX);
    a.hi = min(len, c.table_cols * c.page);                   // the host has bounded the product
    a.first = (int)max((long long)len - c.cu[r + 1] + a.t0, -(long long)POS_MAX);   // farther before the keys is as far
  }
  a.lo = c.window > 0 ? max(a.first - c.window + 1, 0) : 0;   // positions and windows are at most 2^30
  return a;
}

// What is wrong with a request's offsets and length (QTB_PS_* bits); the kernels'
// first block reports it.
template <bool PAGED>
QTB_DEV int attn_wrong(const AttnCall &c, int r) {
  const int a = c.cu[r], b = c.cu[r + 1], len = PAGED ? c.kv_len[r] : 0;
  return (a < 0 || b < a || b > c.n_tokens || len < 0 ? QTB_PS_LENGTH : 0) |
         (PAGED && len > c.table_cols * c.page ? QTB_PS_ROW_FULL : 0);
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
// Tiled TMA loads of a 4- or 5-dimensional box (no multicast).
QTB_DEV void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
QTB_DEV void tma_load_5d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, int v, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
      : "memory");
}
QTB_DEV void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A launch marked programmatic may start while its predecessor still runs:
// pdl_wait returns when that one's writes are visible, pdl_release lets the
// successor start.
QTB_DEV void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
QTB_DEV void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ----------------------------------------------------------------- join ----
// Work that several blocks share leaves its parts in the workspace: block b has
// room for two, part 0 of an item that began in an earlier block and part 1 of
// one that goes on in the next.  A part is, for each of its 1 or 2 tiles of M
// rows, the outputs O [M][HD] and (m, l) [M][2] in f32.  What block b began and
// did not finish:
struct AttnCut {
  int last;                // the last block with a part of it (-1: nothing was cut)
  int t0, n;               // the request's first packed token, its tokens
  int head0, row0;         // first query head; index of row 0 among the request's rows of the key head
  int per_tile;            // rows in use in a tile
  int pad[2];
};
constexpr int JOIN_WARPS = 8;

// Adds the parts of the item that block blockIdx.x cut: part 1 of that block,
// then part 0 of the following ones.  WPR warps share a row (they take every
// WPR-th part and join theirs in warp order), or a warp has RPW rows side by
// side; a lane has HD / 32 dims of each.  Bounded by the latency of a part's
// loads for few parts (those of UNROLL parts of all its rows are in flight
// together), by their bytes for many: 148 cut items of 256 rows are about 40 MB
// and 14 us.  Its blocks may be up while the grid that writes parts and cuts still
// runs, so neither is read-only to it: they are not declared const __restrict__,
// which would let the compiler read them through the read-only path, and ahead of
// pdl_wait.
template <int HD, bool F16, int M, int TILES, int WPR, int RPW>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
join_kernel(const AttnCall c, const float *parts, const AttnCut *cuts) {
  static_assert(WPR == 1 || RPW == 1, "rows of a warp");
  constexpr int TF = M * (HD + 2), V = HD / 32, UNROLL = 4, ROWS = JOIN_WARPS / WPR * RPW;
  __shared__ float s_o[WPR > 1 ? JOIN_WARPS : 1][HD];
  __shared__ float2 s_ml[JOIN_WARPS];
  pdl_wait();
  const AttnCut cut = cuts[blockIdx.x];
  if (cut.last < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b0 = blockIdx.x, n = cut.last - b0 + 1, sub = warp % WPR;
  for (int r0 = blockIdx.y * ROWS; r0 < M * TILES; r0 += gridDim.y * ROWS) {
    const int row = r0 + warp / WPR * RPW, tile = row / M, rr = row - tile * M;
    const float *base = parts + (long long)(2 * b0) * TILES * TF + tile * TF + rr * HD + V * lane;   // part 0 of b0
    const float *base_ml = parts + (long long)(2 * b0) * TILES * TF + tile * TF + M * HD + 2 * rr;
    const int at0 = cut.row0 + tile * cut.per_tile + rr;
    if (rr >= cut.per_tile || at0 / c.group >= cut.n) {   // the rows of a warp run on: its first one tells
      if (WPR > 1) return;                 // all warps have this row
      continue;
    }
    float m[RPW], l[RPW], o[RPW][V];
#pragma unroll
    for (int r = 0; r < RPW; r++) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) o[r][v] = 0.f;
    }
    for (int i0 = sub; i0 < n; i0 += WPR * UNROLL) {
      float x[UNROLL][RPW][V];
      float2 ml[UNROLL][RPW];
#pragma unroll
      for (int i = 0; i < UNROLL; i++) {
        const int k = min(i0 + i * WPR, n - 1);
        const long long off = (long long)(2 * k + (k == 0 ? 1 : 0)) * TILES * TF;
#pragma unroll
        for (int r = 0; r < RPW; r++) {
          ml[i][r] = *reinterpret_cast<const float2 *>(base_ml + off + 2 * r);
#pragma unroll
          for (int v = 0; v < V; v += 2) {
            const float2 y = *reinterpret_cast<const float2 *>(base + off + r * HD + v);
            x[i][r][v] = y.x; x[i][r][v + 1] = y.y;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < UNROLL; i++)
#pragma unroll
        for (int r = 0; r < RPW; r++) {
          // a part without a visible key has m = -inf, and O that was never written
          if (i0 + i * WPR >= n || ml[i][r].x == -INFINITY) continue;
          const float m2 = fmaxf(m[r], ml[i][r].x), f = exp2_approx(m[r] - m2), w = exp2_approx(ml[i][r].x - m2);
          m[r] = m2;
          l[r] = l[r] * f + ml[i][r].y * w;
#pragma unroll
          for (int v = 0; v < V; v++) o[r][v] = o[r][v] * f + x[i][r][v] * w;
        }
    }
    if (WPR > 1) {
#pragma unroll
      for (int v = 0; v < V; v++) s_o[warp][V * lane + v] = o[0][v];
      if (lane == 0) s_ml[warp] = make_float2(m[0], l[0]);
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int i = 1; i < WPR; i++) {
          const float2 z = s_ml[warp + i];
          if (z.x == -INFINITY) continue;
          const float m2 = fmaxf(m[0], z.x), f = exp2_approx(m[0] - m2), w = exp2_approx(z.x - m2);
          m[0] = m2;
          l[0] = l[0] * f + z.y * w;
#pragma unroll
          for (int v = 0; v < V; v++) o[0][v] = o[0][v] * f + s_o[warp + i][V * lane + v] * w;
        }
      }
      __syncthreads();
      if (sub != 0) continue;
    }
#pragma unroll
    for (int r = 0; r < RPW; r++) {
      const int at = at0 + r, tok = at / c.group, head = cut.head0 + at - tok * c.group;
      if (rr + r >= cut.per_tile || tok >= cut.n) continue;
      const float inv = l[r] > 0.f || l[r] != l[r] ? 1.f / l[r] : 0.f;   // no visible key: zeros
      const long long tk = cut.t0 + tok;
      uint16_t *op = c.out + tk * c.o_st + head * c.o_sh + V * lane;
#pragma unroll
      for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t *>(op + v) = pack2<F16>(o[r][v] * inv, o[r][v + 1] * inv);
      if (c.lse && lane == 0) c.lse[tk * c.n_heads + head] = l[r] == 0.f ? -INFINITY : (m[r] + log2f(l[r])) * 0.6931471805599453f;
    }
  }
}

// ------------------------------------------------------------------ host ---
// A launch that may come up before its predecessor in the stream has ended (it
// calls pdl_wait before it reads that one's results).
template <typename... P, typename... A>
static cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

typedef CUresult (*TensorMapFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The map of a tensor of two-byte values (extents and strides innermost first,
// the innermost stride 1) in boxes with the 128-byte swizzle; what lies outside
// reads as zeros.
static inline bool tensor_map(TensorMapFn fn, CUtensorMap *out, const void *base, bool f16, int rank, const long long *ext,
                              const long long *stride, const int *box) {
  cuuint64_t dims[5], bytes[4];
  cuuint32_t b[5], one[5];
  for (int i = 0; i < rank; i++) {
    dims[i] = (cuuint64_t)ext[i];
    b[i] = (cuuint32_t)box[i];
    one[i] = 1;
    if (i) bytes[i - 1] = ext[i] > 1 ? (cuuint64_t)stride[i] * 2 : 128;   // of an axis of one, any will do
  }
  return fn && fn(out, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void *>(base),
                  dims, bytes, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace qtb
