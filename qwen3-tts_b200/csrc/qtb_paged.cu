// qtb_paged.cu -- the operators of a serving step over a paged KV cache, on
// device memory and the caller's stream: block tables and slot maps from
// request lengths (qtb_paged_plan), the append of new keys and values through
// the slot map (qtb_paged_append), attention of each request's new tokens over
// its pages (qtb_paged_attention) and over packed prompts
// (qtb_prompt_attention).  No call allocates, synchronises or keeps state.
#include "qtb_paged.cuh"
#include "qtb_attn_rows.cuh"
#include "qtb_attn_tile.cuh"

#include <cuda_runtime.h>
#include <cstdint>
#include <limits.h>
#include <mutex>

using namespace qtb;

extern int qtb_fail(int code, const char *fmt, ...);   // qtb_engine.cu: records the thread's message

#define PAGED_TRY(call)                                                                       \
  do {                                                                                        \
    cudaError_t e_ = (call);                                                                  \
    if (e_ != cudaSuccess) return qtb_fail(QTB_E_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
  } while (0)

namespace {

// ------------------------------------------------------------------ plan ---
// With cu the exclusive sum of new and f that of the pages each request has to
// take, token t of request r (cu[r] <= t < cu[r + 1]) sits at position
// p = past[r] + t - cu[r], in page p / P of its row: an old page, or
// free[head + f[r] + p / P - ceil(past[r] / P)].  Neither needs another
// request's table row, so one launch does it all: every block walks the
// request lengths (from L2) in tiles with a block-wide scan, and serves the
// tokens of its own range and every grid-th request's row.  Tokens past
// max_tokens are dropped before pages are counted for them: where the packed
// offsets pass it, the tile is scanned again.  What bounds it is a launch and the
// latency of lengths, scan, divisions and stores, not bytes: 7.1 us for 64 requests
// of a token each, 6.8 for 1024 with 38000 tokens.
constexpr int PLAN_THREADS = 256, PLAN_PER = 4, PLAN_TILE = PLAN_THREADS * PLAN_PER;

struct PlanCall {
  const int *past, *fresh, *free_pages, *free_head;
  int *table, *cu, *kv_len, *pos, *req, *head_out, *status;
  long long *slot;
  long long table_stride;
  int n_req, table_cols, page, n_free, max_tokens;
};

// Inclusive block scan of a pair; every thread also gets the block's total.
QTB_DEV void scan_pair(long long &a, long long &b, long long (*s_w)[2], long long &ta, long long &tb) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long xa = __shfl_up_sync(0xffffffffu, a, o), xb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += xa; b += xb; }
  }
  __syncthreads();
  if (lane == 31) { s_w[w][0] = a; s_w[w][1] = b; }
  __syncthreads();
  long long pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll
  for (int i = 0; i < PLAN_THREADS / 32; i++) {
    if (i == w) { pa = ta; pb = tb; }
    ta += s_w[i][0]; tb += s_w[i][1];
  }
  a += pa; b += pb;
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const PlanCall c) {
  __shared__ long long s_w[PLAN_THREADS / 32][2];
  __shared__ int s_cu[PLAN_TILE + 1];    // packed offsets of the tile's requests, clipped to max_tokens
  __shared__ int s_first[PLAN_TILE];     // list index of the request's first new page, clipped to n_free
  __shared__ int s_past[PLAN_TILE];
  const int tid = threadIdx.x, nb = gridDim.x;
  const int t0 = (int)((long long)c.max_tokens * blockIdx.x / nb);
  const int t1 = (int)((long long)c.max_tokens * (blockIdx.x + 1) / nb);
  const long long cap = (long long)c.table_cols * c.page;
  const int head = c.free_head ? max(*c.free_head, 0) : 0;
  long long tok = 0, pages = head;       // packed offset and list index at the tile's start
  int bad = 0;
  for (int base = 0; base < c.n_req; base += PLAN_TILE) {
    int past[PLAN_PER], n[PLAN_PER], need[PLAN_PER];
    long long a = 0, b = 0;
    bool full = false;
    auto pages_for = [&](int p, int m) {     // that m tokens behind p cached ones have to take
      const long long end = min((long long)p + m, cap);
      if ((long long)p + m > cap) full = true;
      return (int)max((end + c.page - 1) / c.page - ((long long)p + c.page - 1) / c.page, 0ll);
    };
#pragma unroll
    for (int i = 0; i < PLAN_PER; i++) {
      const int r = base + tid * PLAN_PER + i;
      int p = r < c.n_req ? c.past[r] : 0, m = r < c.n_req ? c.fresh[r] : 0;
      if (p < 0 || m < 0) { bad |= QTB_PS_LENGTH; p = max(p, 0); m = max(m, 0); }
      past[i] = p; n[i] = m;
      need[i] = pages_for(p, m);
      a += m; b += need[i];
    }
    long long mine_a = a, mine_b = b;
    long long ta, tb;
    scan_pair(a, b, s_w, ta, tb);
    if (tok + ta > c.max_tokens) {           // the same for the whole block
      // the tokens past max_tokens are dropped, and take no pages
      long long at = tok + a - mine_a;
      b = 0;
      full = false;
#pragma unroll
      for (int i = 0; i < PLAN_PER; i++) {
        const int m = (int)max(min((long long)n[i], c.max_tokens - at), 0ll);
        at += n[i];
        need[i] = pages_for(past[i], m);
        b += need[i];
      }
      mine_b = b;
      long long x = 0, tx;
      scan_pair(x, b, s_w, tx, tb);
    }
    if (full) bad |= QTB_PS_ROW_FULL;
    a += tok - mine_a; b += pages - mine_b;   // exclusive, from the call's start
#pragma unroll
    for (int i = 0; i < PLAN_PER; i++) {
      const int j = tid * PLAN_PER + i;
      s_cu[j] = (int)min(a, (long long)c.max_tokens);
      s_first[j] = (int)min(b, (long long)c.n_free);
      s_past[j] = past[i];
      a += n[i]; b += need[i];
      if (j == PLAN_TILE - 1) s_cu[PLAN_TILE] = (int)min(a, (long long)c.max_tokens);
    }
    __syncthreads();
    const int here = min(PLAN_TILE, c.n_req - base);
    // rows: offsets, lengths and new table entries, a warp to a request
    for (int j = blockIdx.x * (PLAN_THREADS / 32) + (tid >> 5); j < here; j += nb * (PLAN_THREADS / 32)) {
      const int r = base + j, p = s_past[j], m = s_cu[j + 1] - s_cu[j];
      const long long end = min((long long)p + m, cap);
      const int have = (int)min(((long long)p + c.page - 1) / c.page, (long long)c.table_cols);
      const int want = (int)((end + c.page - 1) / c.page);
      for (int e = have + (tid & 31); e < want; e += 32) {
        const long long at = (long long)s_first[j] + (e - have);
        const bool ok = at < c.n_free;
        if (!ok) bad |= QTB_PS_NO_PAGES;
        c.table[r * c.table_stride + e] = ok ? c.free_pages[at] : -1;
      }
      if ((tid & 31) == 0) {
        c.cu[r] = s_cu[j];
        c.kv_len[r] = (int)min((long long)p + m, (long long)INT_MAX);
        if (r == c.n_req - 1) c.cu[c.n_req] = s_cu[j + 1];
      }
    }
    // tokens of this block's range that belong to the tile's requests
    const int lo = max(t0, s_cu[0]), hi = min(t1, s_cu[here]);
    for (int t = lo + tid; t < hi; t += PLAN_THREADS) {
      int j = 0, k = here;               // s_cu[j] <= t < s_cu[k]
      while (k - j > 1) {
        const int mid = (j + k) >> 1;
        if (s_cu[mid] <= t) j = mid; else k = mid;
      }
      const int r = base + j;
      const long long p = (long long)s_past[j] + t - s_cu[j];
      const int e = (int)(p / c.page), have = (int)(((long long)s_past[j] + c.page - 1) / c.page);
      int page = -1;
      if (p < cap) {
        const long long at = (long long)s_first[j] + (e - have);
        if (e < have) page = c.table[r * c.table_stride + e];
        else if (at < c.n_free) page = c.free_pages[at];
        if (page < 0) bad |= e < have ? QTB_PS_PAGE : QTB_PS_NO_PAGES;
      }
      c.slot[t] = page < 0 ? -1 : (long long)page * c.page + p % c.page;
      c.pos[t] = (int)min(p, (long long)INT_MAX);
      c.req[t] = r;
    }
    tok += ta; pages += tb;
    __syncthreads();
  }
  if (tok > c.max_tokens) bad |= QTB_PS_ROOM;
  // room behind the last token
  for (int t = max(t0, (int)min(tok, (long long)c.max_tokens)) + tid; t < t1; t += PLAN_THREADS) {
    c.slot[t] = -1;
    c.pos[t] = -1;
    c.req[t] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    if (c.n_req == 0) c.cu[0] = 0;
    if (c.head_out) *c.head_out = (int)min(pages, max((long long)c.n_free, (long long)head));
  }
  raise_status(c.status, bad);
}

// ---------------------------------------------------------------- append ---
// pool[slot / P][head][slot % P][:] = round(x[token][head][:]), for keys and
// values.  A thread has a fixed place of 8 values (16 bytes of cache) in a
// token's row and moves it for APP_UNROLL tokens at a time, all loads first;
// bounded by the bytes read and written: 32768 tokens of 8 heads of 128, f16, into
// pages of 64 take 45 us, 5.95 TB/s (55 us when each thread divided its way to its
// place for every vector).  64 tokens are a launch, 2.2 us.
constexpr int APP_THREADS = 256, APP_UNROLL = 4;

struct AppendCall {
  const void *k, *v;
  uint16_t *kpool, *vpool;
  const long long *slot;
  int *status;
  long long k_st, k_sh, v_st, v_sh;
  long long kp_st[3], vp_st[3];
  long long n_slots;
  int n_tokens, page;
  int row_vec, head_vec;    // vectors of 8 values in a token, in a head
  int side;                 // tokens that a block's threads stand side by side for
};

template <bool F16, bool SRC32>
QTB_DEV uint4 load8(const void *base, long long at) {
  if (!SRC32) return ld_nc_u4(static_cast<const uint16_t *>(base) + at);
  const uint4 a = ld_nc_u4(static_cast<const float *>(base) + at);
  const uint4 b = ld_nc_u4(static_cast<const float *>(base) + at + 4);
  uint4 r;
  r.x = pack2<F16>(__uint_as_float(a.x), __uint_as_float(a.y));
  r.y = pack2<F16>(__uint_as_float(a.z), __uint_as_float(a.w));
  r.z = pack2<F16>(__uint_as_float(b.x), __uint_as_float(b.y));
  r.w = pack2<F16>(__uint_as_float(b.z), __uint_as_float(b.w));
  return r;
}

template <bool F16, bool SRC32>
__global__ void __launch_bounds__(APP_THREADS) append_kernel(const AppendCall c) {
  const int beside = c.side > 1 ? threadIdx.x / c.row_vec : 0;
  if (beside >= c.side) return;
  int bad = 0;
  for (int vec = threadIdx.x - beside * c.row_vec; vec < c.row_vec; vec += APP_THREADS) {
    const int h = vec / c.head_vec, d = (vec - h * c.head_vec) * 8;
    const long long ks = h * c.k_sh + d, vs = h * c.v_sh + d, kp = h * c.kp_st[1] + d, vp = h * c.vp_st[1] + d;
    const int step = gridDim.x * c.side;
    for (int t0 = blockIdx.x * c.side + beside; t0 < c.n_tokens; t0 += step * APP_UNROLL) {
      long long s[APP_UNROLL];
      uint4 kx[APP_UNROLL], vx[APP_UNROLL];
#pragma unroll
      for (int u = 0; u < APP_UNROLL; u++) {
        const long long t = t0 + (long long)u * step;
        s[u] = t < c.n_tokens ? c.slot[t] : -1;
        if (s[u] >= c.n_slots) { bad |= QTB_PS_PAGE; s[u] = -1; }
      }
#pragma unroll
      for (int u = 0; u < APP_UNROLL; u++) {
        if (s[u] < 0) continue;
        const long long t = t0 + (long long)u * step;
        kx[u] = load8<F16, SRC32>(c.k, t * c.k_st + ks);
        vx[u] = load8<F16, SRC32>(c.v, t * c.v_st + vs);
      }
#pragma unroll
      for (int u = 0; u < APP_UNROLL; u++) {
        if (s[u] < 0) continue;
        const long long pg = c.n_slots <= 0x7fffffffll ? (long long)((unsigned)s[u] / (unsigned)c.page) : s[u] / c.page;
        const long long off = s[u] - pg * c.page;
        *reinterpret_cast<uint4 *>(c.kpool + pg * c.kp_st[0] + off * c.kp_st[2] + kp) = kx[u];
        *reinterpret_cast<uint4 *>(c.vpool + pg * c.vp_st[0] + off * c.vp_st[2] + vp) = vx[u];
      }
    }
  }
  raise_status(c.status, bad);
}

// ------------------------------------------------------------------ host ---
constexpr int MAX_DEV = 64;
struct DevInfo {
  int sms = 0;
  TensorMapFn encode = nullptr;            // cuTensorMapEncodeTiled
  cudaError_t err = cudaSuccess;
};

// The current device's SM count, with the kernels' shared-memory limits set,
// once per device.
int device_info(const DevInfo **out) {
  *out = nullptr;
  static DevInfo info[MAX_DEV];
  static std::once_flag once[MAX_DEV];
  int dev = 0;
  PAGED_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= MAX_DEV) return qtb_fail(QTB_E_UNSUPPORTED, "device index %d", dev);
  DevInfo &d = info[dev];
  std::call_once(once[dev], [&] {
    int major = 0;
    d.err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (d.err == cudaSuccess && major != 10) d.err = cudaErrorNoKernelImageForDevice;
    if (d.err == cudaSuccess) d.err = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    if (d.err == cudaSuccess) d.err = rows_prepare();
    if (d.err == cudaSuccess) d.err = tile_prepare();
    if (d.err == cudaSuccess) {
      void *p = nullptr;
      cudaDriverEntryPointQueryResult q;
      d.err = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
      if (q == cudaDriverEntryPointSuccess) d.encode = reinterpret_cast<TensorMapFn>(p);
    }
  });
  if (d.err != cudaSuccess) return qtb_fail(QTB_E_CUDA, "paged operators on device %d: %s", dev, cudaGetErrorString(d.err));
  *out = &d;
  return QTB_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Strides of whole 16 bytes; that of an axis of one is never used, and may be any.
bool rows16(const int64_t *st, const int64_t *ext, int n, int elem) {
  for (int i = 0; i < n; i++)
    if (ext[i] > 1 && (st[i] < 0 || st[i] % (16 / elem))) return false;
  return true;
}
// Strides that a tensor map can hold: an expanded axis (stride 0) it cannot.
bool spread(const int64_t *st, const int64_t *ext, int n) {
  for (int i = 0; i < n; i++)
    if (ext[i] > 1 && (st[i] <= 0 || st[i] >= (1ll << 39))) return false;
  return true;
}

// Checks what both attention forms share and fills the kernels' view of it.
int attn_call(const qtb_attn_t *d, bool paged, AttnCall &c) {
  if (!d) return qtb_fail(QTB_E_INVALID, "null descriptor");
  if (d->dtype != QTB_T_BF16 && d->dtype != QTB_T_F16) return qtb_fail(QTB_E_UNSUPPORTED, "dtype %lld: bf16 or f16", (long long)d->dtype);
  if (d->head_dim != 64 && d->head_dim != 128) return qtb_fail(QTB_E_UNSUPPORTED, "head_dim %lld: 64 or 128", (long long)d->head_dim);
  if (d->n_heads < 1 || d->n_kv < 1 || d->n_heads % d->n_kv || d->n_heads > 1024)
    return qtb_fail(QTB_E_INVALID, "%lld query heads over %lld key heads", (long long)d->n_heads, (long long)d->n_kv);
  if (d->n_heads / d->n_kv > 128) return qtb_fail(QTB_E_UNSUPPORTED, "%lld query heads to a key head: at most 128", (long long)(d->n_heads / d->n_kv));
  if (d->n_req < 0 || d->n_req >= (1 << 24) || d->n_tokens < 0 || d->n_tokens * (d->n_heads / d->n_kv) >= (1ll << 30))
    return qtb_fail(QTB_E_INVALID, "%lld requests, %lld tokens", (long long)d->n_req, (long long)d->n_tokens);
  if (d->n_tokens / (TILE_M / (d->n_heads / d->n_kv)) + d->n_req >= (1ll << 31) / d->n_kv)   // units of work are counted in 32 bits
    return qtb_fail(QTB_E_UNSUPPORTED, "%lld requests and %lld tokens over %lld key heads", (long long)d->n_req, (long long)d->n_tokens, (long long)d->n_kv);
  if (d->window < 0 || d->max_new < 0) return qtb_fail(QTB_E_INVALID, "window %lld, max_new %lld", (long long)d->window, (long long)d->max_new);
  if (!(d->scale == d->scale) || d->scale > 3e38 || d->scale < -3e38) return qtb_fail(QTB_E_INVALID, "scale is not finite");
  if (!d->cu_new || (d->n_tokens && (!d->q || !d->out)) || (d->n_tokens && !paged && (!d->k || !d->v)))
    return qtb_fail(QTB_E_INVALID, "null pointer");
  if (!aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out))
    return qtb_fail(QTB_E_INVALID, "q, k, v and out must start on 16 bytes");
  const int64_t qx[2] = {d->n_tokens, d->n_heads}, px[3] = {d->n_pages, d->n_kv, d->page}, tx[2] = {d->n_tokens, d->n_kv};
  const int64_t *kx = paged ? px : tx;
  const int kn = paged ? 3 : 2;
  if (!rows16(d->q_stride, qx, 2, 2) || !rows16(d->k_stride, kx, kn, 2) || !rows16(d->v_stride, kx, kn, 2) || !rows16(d->out_stride, qx, 2, 2))
    return qtb_fail(QTB_E_INVALID, "strides must be non-negative multiples of 16 bytes");
  if (paged) {
    if (d->page < 16 || d->page % 16 || d->page > 65536) return qtb_fail(QTB_E_INVALID, "page %lld: a multiple of 16", (long long)d->page);
    if (d->n_pages < 1 || d->n_pages >= INT_MAX || d->table_cols < 0 || d->table_cols > (1 << 30) || d->table_cols * d->page > (1 << 30) || d->table_stride < 0)
      return qtb_fail(QTB_E_INVALID, "%lld pages, %lld table columns", (long long)d->n_pages, (long long)d->table_cols);
    if ((d->n_req && !d->kv_len) || (d->n_req && d->table_cols && !d->table) || (d->n_pages && (!d->k || !d->v)))
      return qtb_fail(QTB_E_INVALID, "null pointer");
  }
  if (!spread(d->q_stride, qx, 2) || !spread(d->out_stride, qx, 2) || !spread(d->k_stride, kx, kn) || !spread(d->v_stride, kx, kn))
    return qtb_fail(QTB_E_INVALID, "an axis of q, k, v or out is expanded (stride 0)");
  c = AttnCall{};
  c.q = static_cast<const uint16_t *>(d->q); c.k = static_cast<const uint16_t *>(d->k); c.v = static_cast<const uint16_t *>(d->v);
  c.out = static_cast<uint16_t *>(d->out); c.lse = d->lse; c.cu = d->cu_new; c.status = d->status;
  c.q_st = d->q_stride[0]; c.q_sh = d->q_stride[1]; c.o_st = d->out_stride[0]; c.o_sh = d->out_stride[1];
  for (int i = 0; i < 3; i++) { c.k_st[i] = d->k_stride[i]; c.v_st[i] = d->v_stride[i]; }
  c.n_req = (int)d->n_req; c.n_tokens = (int)d->n_tokens; c.n_heads = (int)d->n_heads; c.n_kv = (int)d->n_kv;
  c.group = c.n_heads / c.n_kv;
  c.causal = d->causal != 0; c.window = (int)(d->window < (1 << 30) ? d->window : 1 << 30);
  c.scale_log2 = (float)(d->scale * 1.4426950408889634);
  c.page = 16;
  if (paged) {
    c.kv_len = d->kv_len; c.table = d->table; c.table_stride = d->table_stride;
    c.page = (int)d->page; c.n_pages = (int)d->n_pages; c.table_cols = (int)d->table_cols;
  }
  return QTB_OK;
}

// Which kernel has the call.  The rows kernel, where every request has few query
// rows to a key head, as max_new tells (and in the forms that the tile kernel does
// not read); the tile kernel, where any has many, and for prompts, which have no
// long cache to split.  A mixed call goes to the tiles as a whole: single tokens
// fill them badly, but their keys stream at the same rate, and a second pair of
// launches costs more (us, tiles / rows and tiles: 16 requests of up to 7000 keys,
// every fourth with 400 new tokens, 204 / 236; 64 of 1000, every fourth with 64,
// 64 / 74; 4 of 500, one with 64, 15 / 26).
struct AttnPlan {
  long long rows;          // query rows of a request to a key head, at most (0: not known)
  bool tiles;
  bool cut;                // items may be cut between blocks
  size_t ws;               // bytes of workspace
};
AttnPlan attn_plan(const AttnCall &c, const qtb_attn_t *d, bool paged, int sms) {
  AttnPlan p;
  p.rows = (d->max_new < (1 << 30) ? d->max_new : 1 << 30) * c.group;   // max_new may be any number
  p.tiles = tile_form(c) && !(paged && p.rows > 0 && p.rows <= ROWS_M);
  // no second launch for a few key tiles, nor where one request's items are seen to fill the blocks
  const long long pair = 2 * (TILE_M / c.group), items = (c.n_tokens + pair - 1) / pair * c.n_kv;
  p.cut = p.tiles && !(d->max_kv > 0 && d->max_kv <= 4 * TILE_N) && !(c.n_req == 1 && tile_whole(items, sms));
  p.ws = !p.tiles ? rows_workspace((int)d->head_dim, sms) : p.cut ? tile_workspace((int)d->head_dim, sms) : 0;
  return p;
}

int attend(const qtb_attn_t *d, bool paged, void *stream) {
  AttnCall c;
  int rc = attn_call(d, paged, c);
  if (rc) return rc;
  if (!c.n_req || !c.n_tokens) return QTB_OK;
  const DevInfo *dev;
  if ((rc = device_info(&dev))) return rc;
  const AttnPlan p = attn_plan(c, d, paged, dev->sms);
  const int64_t need = (int64_t)p.ws;
  if (d->workspace_bytes < need || (need && !d->workspace))
    return qtb_fail(QTB_E_WORKSPACE, "workspace of %lld bytes: %lld needed", (long long)d->workspace_bytes, (long long)need);
  if (!aligned16(d->workspace)) return qtb_fail(QTB_E_INVALID, "the workspace must start on 16 bytes");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = d->dtype == QTB_T_F16;
  const int hd = (int)d->head_dim;
  static const char *const no_map = "q, k or v have strides or extents that a tensor map cannot hold";
  if (p.tiles) {
    TileMaps m;
    if (!tile_maps(c, paged, f16, hd, dev->encode, m)) return qtb_fail(QTB_E_UNSUPPORTED, no_map);
    PAGED_TRY(tile_launch(c, paged, f16, hd, m, dev->sms, p.cut ? d->workspace : nullptr, st));
  } else {
    RowsMaps m;
    const int max_rows = p.rows > 0 && p.rows < ROWS_M ? (int)p.rows : ROWS_M;
    if (!rows_maps(c, paged, f16, hd, dev->encode, m)) return qtb_fail(QTB_E_UNSUPPORTED, no_map);
    PAGED_TRY(rows_launch(c, paged, f16, hd, m, dev->sms, max_rows, d->workspace, st));
  }
  return QTB_OK;
}

}  // namespace

extern "C" int qtb_paged_plan(const qtb_paged_plan_t *d, void *stream) {
  if (!d) return qtb_fail(QTB_E_INVALID, "null descriptor");
  if (d->n_req < 0 || d->n_req >= (1 << 24) || d->max_tokens < 0 || d->max_tokens >= (1ll << 30) || d->n_free < 0 ||
      d->n_free > INT_MAX || d->page < 1 || d->page > 65536 || d->table_cols < 0 || d->table_cols > (1 << 30) || d->table_cols * d->page > (1 << 30) || d->table_stride < 0)
    return qtb_fail(QTB_E_INVALID, "%lld requests, room for %lld tokens, %lld free pages of %lld, %lld table columns", (long long)d->n_req,
                    (long long)d->max_tokens, (long long)d->n_free, (long long)d->page, (long long)d->table_cols);
  if (!d->cu_new || (d->n_req && (!d->past_len || !d->new_len || !d->kv_len || (d->table_cols && !d->table))) ||
      (d->n_free && !d->free_pages) || (d->max_tokens && (!d->slot || !d->pos || !d->req)))
    return qtb_fail(QTB_E_INVALID, "null pointer");
  if (d->free_head && d->free_head == d->free_head_out)
    return qtb_fail(QTB_E_INVALID, "free_head_out must be another word than free_head");
  const DevInfo *dev;
  if (int rc = device_info(&dev)) return rc;
  PlanCall c = {};
  c.past = d->past_len; c.fresh = d->new_len; c.free_pages = d->free_pages; c.free_head = d->free_head;
  c.table = d->table; c.cu = d->cu_new; c.kv_len = d->kv_len; c.pos = d->pos; c.req = d->req;
  c.head_out = d->free_head_out; c.status = d->status; c.slot = reinterpret_cast<long long *>(d->slot);
  c.table_stride = d->table_stride;
  c.n_req = (int)d->n_req; c.table_cols = (int)d->table_cols; c.page = (int)d->page; c.n_free = (int)d->n_free;
  c.max_tokens = (int)d->max_tokens;
  const long long want = (d->max_tokens + 2 * d->n_req + 511) / 512;
  const int grid = (int)(want < 1 ? 1 : want > dev->sms ? dev->sms : want);
  plan_kernel<<<grid, PLAN_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(c);
  PAGED_TRY(cudaGetLastError());
  return QTB_OK;
}

extern "C" int qtb_paged_append(const qtb_paged_append_t *d, void *stream) {
  if (!d) return qtb_fail(QTB_E_INVALID, "null descriptor");
  const bool src32 = d->src_dtype == QTB_T_F32;
  if ((d->dtype != QTB_T_BF16 && d->dtype != QTB_T_F16) || (!src32 && d->src_dtype != d->dtype))
    return qtb_fail(QTB_E_UNSUPPORTED, "type %lld into a cache of type %lld: bf16 or f16 from the same or from f32", (long long)d->src_dtype, (long long)d->dtype);
  if (d->n_tokens < 0 || d->n_tokens >= (1ll << 30) || d->n_kv < 1 || d->n_kv > 1024 || d->head_dim < 8 || d->head_dim % 8 || d->head_dim > 1024)
    return qtb_fail(QTB_E_INVALID, "%lld tokens, %lld heads of %lld (a multiple of 8)", (long long)d->n_tokens, (long long)d->n_kv, (long long)d->head_dim);
  if (d->page < 1 || d->page > 65536 || d->n_pages < 0 || d->n_pages > INT_MAX)
    return qtb_fail(QTB_E_INVALID, "%lld pages of %lld", (long long)d->n_pages, (long long)d->page);
  if (!d->n_tokens) return QTB_OK;
  if (!d->k || !d->v || !d->slot || (d->n_pages && (!d->kpool || !d->vpool))) return qtb_fail(QTB_E_INVALID, "null pointer");
  const int es = src32 ? 4 : 2;
  const int64_t sx[2] = {d->n_tokens, d->n_kv}, px[3] = {d->n_pages, d->n_kv, d->page};
  if (!aligned16(d->k) || !aligned16(d->v) || !aligned16(d->kpool) || !aligned16(d->vpool) || !rows16(d->k_stride, sx, 2, es) ||
      !rows16(d->v_stride, sx, 2, es) || !rows16(d->kpool_stride, px, 3, 2) || !rows16(d->vpool_stride, px, 3, 2))
    return qtb_fail(QTB_E_INVALID, "pointers and strides must be multiples of 16 bytes");
  const DevInfo *dev;
  if (int rc = device_info(&dev)) return rc;
  AppendCall c = {};
  c.k = d->k; c.v = d->v; c.kpool = static_cast<uint16_t *>(d->kpool); c.vpool = static_cast<uint16_t *>(d->vpool);
  c.slot = reinterpret_cast<const long long *>(d->slot); c.status = d->status;
  c.k_st = d->k_stride[0]; c.k_sh = d->k_stride[1]; c.v_st = d->v_stride[0]; c.v_sh = d->v_stride[1];
  for (int i = 0; i < 3; i++) { c.kp_st[i] = d->kpool_stride[i]; c.vp_st[i] = d->vpool_stride[i]; }
  c.head_vec = (int)d->head_dim / 8;
  c.row_vec = (int)d->n_kv * c.head_vec;
  c.n_tokens = (int)d->n_tokens;
  c.side = c.row_vec < APP_THREADS ? APP_THREADS / c.row_vec : 1;
  c.n_slots = d->n_pages * d->page;
  c.page = (int)d->page;
  // as many blocks as tokens side by side, up to eight to an SM
  const long long want = (d->n_tokens + c.side - 1) / c.side;
  const int grid = (int)(want < dev->sms * 8ll ? want : dev->sms * 8ll);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = d->dtype == QTB_T_F16;
  if (f16 && src32) append_kernel<true, true><<<grid, APP_THREADS, 0, st>>>(c);
  else if (f16) append_kernel<true, false><<<grid, APP_THREADS, 0, st>>>(c);
  else if (src32) append_kernel<false, true><<<grid, APP_THREADS, 0, st>>>(c);
  else append_kernel<false, false><<<grid, APP_THREADS, 0, st>>>(c);
  PAGED_TRY(cudaGetLastError());
  return QTB_OK;
}

extern "C" int64_t qtb_attn_workspace(const qtb_attn_t *d, int paged) {
  AttnCall c;
  if (int rc = attn_call(d, paged != 0, c)) return rc;
  if (!c.n_req || !c.n_tokens) return 0;
  const DevInfo *dev;
  if (int rc = device_info(&dev)) return rc;
  return (int64_t)attn_plan(c, d, paged != 0, dev->sms).ws;
}

extern "C" int qtb_paged_attention(const qtb_attn_t *d, void *stream) { return attend(d, true, stream); }
extern "C" int qtb_prompt_attention(const qtb_attn_t *d, void *stream) { return attend(d, false, stream); }
