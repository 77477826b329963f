// qtb_attn_rows.cuh -- attention of few query rows over many keys.
//
// A query row is one (token, query head); the rows of a request that share a
// key head (token-major, the group's heads inside) are taken 16 at a time, the
// M of mma.m16n8k16, so that grouped heads and the tokens of a short chunk read
// K and V once.  Scores are in units of log2 (scale * log2 e folded in), and
// each warp keeps the running maximum m, sum l and output O of its own keys:
//   m' = max(m, s),  l' = l 2^(m - m') + sum 2^(s - m'),  O' likewise.
// States of any two key sets join the same way, so the key axis is cut freely:
// the (request, row group, key head, 64-key chunk) units of the whole call are
// dealt out to the grid in equal runs, whatever the requests' lengths.  An item
// that a block holds whole is written at once; one that is cut leaves its parts
// (O, m, l in f32) in the workspace, and rows_join_kernel adds them in block
// order, so results do not depend on timing.
//
// Keys outside the request, pages outside the pool and rows past the request's
// last are filled with zeros on the way to shared memory and their scores set
// to -inf, so nothing that lies there (NaN, infinities) reaches a sum.
#pragma once
#include "qtb_paged.cuh"

namespace qtb {

constexpr int ROWS_THREADS = 128, ROWS_WARPS = 4, ROWS_M = 16, ROWS_CHUNK = 64, ROWS_STAGES = 3, ROWS_PER_SM = 2;

// Where a cut item's parts are, per block: the request, row group and head of
// the item that the block starts and does not finish, and the last block that
// holds a part of it (-1: none).
struct RowsCut {
  int r, rg, h, last;
};

template <int HD>
constexpr int rows_part_floats() { return ROWS_M * (HD + 2); }   // O rows, then (m, l) pairs
template <int HD>
constexpr int rows_smem() {
  return ROWS_STAGES * 2 * ROWS_CHUNK * HD * 2 + 2 * 32 * (HD / 2) * 4 + ROWS_WARPS * ROWS_M * 2 * 4;
}

// A position in the call's sequence of units.
template <bool PAGED>
struct RowsCursor {
  AttnReq a;
  int r, rg, h, ch;      // request, row group, key head, chunk within the item
  int groups, chunks, c0;

  QTB_DEV void load(const AttnCall &c, int row_limit) {   // the request's counts
    a = attn_request<PAGED>(c, r);
    const int rows = a.n * c.group;
    groups = rows > row_limit ? 0 : (rows + ROWS_M - 1) / ROWS_M;
    c0 = a.lo / ROWS_CHUNK;
    chunks = max((a.hi + ROWS_CHUNK - 1) / ROWS_CHUNK - c0, 1);
  }
  QTB_DEV long long units(const AttnCall &c) const { return (long long)groups * c.n_kv * chunks; }
  QTB_DEV void next(const AttnCall &c, int row_limit) {
    if (++ch < chunks) return;
    ch = 0;
    if (++h < c.n_kv) return;
    h = 0;
    if (++rg < groups) return;
    rg = 0;
    do {
      r++;
      if (r >= c.n_req) { groups = 1; chunks = 1; return; }   // past the end: never served
      load(c, row_limit);
    } while (groups == 0);
  }
};

template <int HD, bool F16, bool PAGED>
__global__ void __launch_bounds__(ROWS_THREADS, ROWS_PER_SM)
rows_kernel(const AttnCall c, int row_limit, float *__restrict__ parts, RowsCut *__restrict__ cuts) {
  constexpr int KS = HD / 16;              // k-steps of Q K^T
  constexpr int NT = HD / 8;               // 8-wide output tiles
  constexpr int UPR = HD / 8;              // 16-byte units of a key row
  constexpr int PASS_ROWS = ROWS_THREADS / UPR, PASSES = ROWS_CHUNK / PASS_ROWS;
  constexpr int KEYS_B = ROWS_CHUNK * HD * 2;
  extern __shared__ __align__(128) unsigned char smem[];
  float *s_red = reinterpret_cast<float *>(smem + ROWS_STAGES * 2 * KEYS_B);   // [2][HD / 2][32]
  float2 *s_ml = reinterpret_cast<float2 *>(s_red + 2 * 32 * (HD / 2));        // [warp][16] (m, l)
  __shared__ long long s_sum[ROWS_WARPS];
  __shared__ long long s_off;              // first unit's index within its request
  __shared__ int s_req;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;

  // --- this block's run of units: thread i counts requests [i n / 128, (i + 1) n / 128)
  RowsCursor<PAGED> cur;
  const int ra = (int)((long long)c.n_req * tid / ROWS_THREADS), rb = (int)((long long)c.n_req * (tid + 1) / ROWS_THREADS);
  long long sum = 0;
  for (cur.r = ra; cur.r < rb; cur.r++) {
    cur.load(c, row_limit);
    sum += cur.units(c);
  }
  long long pre = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, pre, o);
    if (lane >= o) pre += x;
  }
  if (lane == 31) s_sum[warp] = pre;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < ROWS_WARPS; w++) {
    if (w < warp) pre += s_sum[w];
    total += s_sum[w];
  }
  pre -= sum;
  const long long blocks = min((long long)gridDim.x, total);
  if (tid == 0) cuts[blockIdx.x].last = -1;
  if (blockIdx.x >= blocks) return;
  const long long u0 = total * blockIdx.x / blocks, u1 = total * (blockIdx.x + 1) / blocks;
  if (u0 >= pre && u0 < pre + sum) {
    long long at = pre;
    for (cur.r = ra; cur.r < rb; cur.r++) {
      cur.load(c, row_limit);
      const long long n = cur.units(c);
      if (u0 < at + n) break;
      at += n;
    }
    s_req = cur.r;
    s_off = u0 - at;
  }
  __syncthreads();
  cur.r = s_req;
  cur.load(c, row_limit);
  {
    long long off = s_off;
    cur.ch = (int)(off % cur.chunks);
    off /= cur.chunks;
    cur.h = (int)(off % c.n_kv);
    cur.rg = (int)(off / c.n_kv);
  }
  RowsCursor<PAGED> ld = cur;              // runs ahead of `cur` by the copies in flight
  int bad = 0;

  auto copy_unit = [&](int stage) {
    unsigned char *ks = smem + stage * 2 * KEYS_B, *vs = ks + KEYS_B;
    const int row0 = tid / UPR, unit = tid % UPR, pos0 = (ld.c0 + ld.ch) * ROWS_CHUNK;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
      const int row = p * PASS_ROWS + row0, pos = pos0 + row;
      bool ok = pos >= ld.a.lo && pos < ld.a.hi;
      const uint16_t *kp = c.k, *vp = c.v;
      if (ok) {
        if (PAGED) {
          const int e = pos / c.page, pg = c.table[ld.r * c.table_stride + e];
          if (pg < 0 || pg >= c.n_pages) { ok = false; bad |= QTB_PS_PAGE; }
          else {
            const long long off = pos - e * c.page;
            kp += pg * c.k_st[0] + ld.h * c.k_st[1] + off * c.k_st[2] + unit * 8;
            vp += pg * c.v_st[0] + ld.h * c.v_st[1] + off * c.v_st[2] + unit * 8;
          }
        } else {
          const long long t = ld.a.t0 + pos;
          kp += t * c.k_st[0] + ld.h * c.k_st[1] + unit * 8;
          vp += t * c.v_st[0] + ld.h * c.v_st[1] + unit * 8;
        }
      }
      const int at = row * (HD * 2) + ((unit ^ (row & 7)) << 4);
      cp16_zfill(ks + at, kp, ok);
      cp16_zfill(vs + at, vp, ok);
    }
  };

  const long long n_units = u1 - u0;
#pragma unroll
  for (int s = 0; s < ROWS_STAGES - 1; s++) {
    if (s < n_units) { copy_unit(s); ld.next(c, row_limit); }
    cp_commit();
  }

  uint32_t q[KS][4];
  float o[NT][4], m[2], l[2];
  int last_key[2], first_key[2], tok[2];   // per row: the keys it sees, its token (-1: no row)
  bool starts = cur.ch == 0;               // this block holds the current item from its first chunk
  bool fresh = true;

  for (long long u = 0; u < n_units; u++) {
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int row = cur.rg * ROWS_M + gid + 8 * i, t = row / c.group, g = row - t * c.group;
        const bool live = t < cur.a.n;
        tok[i] = live ? t : -1;
        last_key[i] = !live ? -1 : c.causal ? cur.a.first + t : cur.a.hi - 1;
        first_key[i] = c.window > 0 ? max(cur.a.first + t - c.window + 1, 0) : 0;
        const uint16_t *qp = c.q + (long long)(cur.a.t0 + t) * c.q_st + (long long)(cur.h * c.group + g) * c.q_sh + 2 * tig;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          q[k][i] = live ? __ldg(reinterpret_cast<const uint32_t *>(qp + 16 * k)) : 0u;
          q[k][2 + i] = live ? __ldg(reinterpret_cast<const uint32_t *>(qp + 16 * k + 8)) : 0u;
        }
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[n][i] = 0.f;
    }
    cp_wait<ROWS_STAGES - 2>();
    __syncthreads();
    if (u + ROWS_STAGES - 1 < n_units) {
      copy_unit((int)((u + ROWS_STAGES - 1) % ROWS_STAGES));
      ld.next(c, row_limit);
    }
    cp_commit();

    // --- this warp's 16 keys of the chunk
    const unsigned char *ks = smem + (int)(u % ROWS_STAGES) * 2 * KEYS_B, *vs = ks + KEYS_B;
    const int key0 = (cur.c0 + cur.ch) * ROWS_CHUNK + warp * 16;
    float s[2][4] = {};
    {
      const int row = warp * 16 + (lane & 7) + ((lane & 16) >> 1), half = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        uint32_t b[4];
        ldsm_x4(b, ks + row * (HD * 2) + (((2 * k + half) ^ (row & 7)) << 4));
        mma16<F16>(s[0], q[k], b[0], b[1]);
        mma16<F16>(s[1], q[k], b[2], b[3]);
      }
    }
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int key = key0 + 8 * t + 2 * tig + (i & 1), w = i >> 1;
        s[t][i] = key <= last_key[w] && key >= first_key[w] ? s[t][i] * c.scale_log2 : -INFINITY;
        mx[w] = fmaxf(mx[w], s[t][i]);
      }
#pragma unroll
    for (int w = 0; w < 2; w++) {
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
    }
    if (__any_sync(0xffffffffu, mx[0] != m[0] || mx[1] != m[1])) {
#pragma unroll
      for (int w = 0; w < 2; w++) {
        const float f = mx[w] == -INFINITY ? 1.f : exp2_approx(m[w] - mx[w]);
        m[w] = mx[w];
        l[w] *= f;
#pragma unroll
        for (int n = 0; n < NT; n++) { o[n][2 * w] *= f; o[n][2 * w + 1] *= f; }
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[t][i] = exp2_approx(s[t][i] - base[i >> 1]);
        l[i >> 1] += s[t][i];
      }
    // probabilities are rounded to the cache's type for the product with V, as
    // large as the result's own rounding; their sum l is of the unrounded ones
    const uint32_t pa[4] = {pack2<F16>(s[0][0], s[0][1]), pack2<F16>(s[0][2], s[0][3]),
                            pack2<F16>(s[1][0], s[1][1]), pack2<F16>(s[1][2], s[1][3])};
    {
      const int row = warp * 16 + (lane & 15), half = lane >> 4;
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t b[4];
        ldsm_x4_trans(b, vs + row * (HD * 2) + (((n + half) ^ (row & 7)) << 4));
        mma16<F16>(o[n], pa, b[0], b[1]);
        mma16<F16>(o[n + 1], pa, b[2], b[3]);
      }
    }

    const bool ends = cur.ch == cur.chunks - 1;
    if (ends || u + 1 == n_units) {
      // --- join the four warps' states
#pragma unroll
      for (int w = 0; w < 2; w++) {
        l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
        l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
        if (tig == 0) s_ml[warp * ROWS_M + gid + 8 * w] = make_float2(m[w], l[w]);
      }
      __syncthreads();
      float mt[2], lt[2];
#pragma unroll
      for (int w = 0; w < 2; w++) {
        mt[w] = -INFINITY;
        lt[w] = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS_WARPS; i++) mt[w] = fmaxf(mt[w], s_ml[i * ROWS_M + gid + 8 * w].x);
        const float b = mt[w] == -INFINITY ? 0.f : mt[w];
#pragma unroll
        for (int i = 0; i < ROWS_WARPS; i++) {
          const float2 x = s_ml[i * ROWS_M + gid + 8 * w];
          lt[w] += x.y * exp2_approx(x.x - b);
        }
        const float f = exp2_approx(m[w] - b);
#pragma unroll
        for (int n = 0; n < NT; n++) { o[n][2 * w] *= f; o[n][2 * w + 1] *= f; }
      }
#pragma unroll
      for (int half = 2; half >= 1; half >>= 1) {   // warps half .. 2 half - 1 hand over to 0 .. half - 1
        if (warp >= half && warp < 2 * half) {
          float *d = s_red + (warp - half) * 32 * (HD / 2);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) d[(n * 4 + i) * 32 + lane] = o[n][i];
        }
        __syncthreads();
        if (warp < half) {
          const float *d = s_red + warp * 32 * (HD / 2);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[n][i] += d[(n * 4 + i) * 32 + lane];
        }
        __syncthreads();
      }
      if (warp == 0) {
        if (starts && ends) {
#pragma unroll
          for (int w = 0; w < 2; w++) {
            if (tok[w] < 0) continue;
            const int row = cur.rg * ROWS_M + gid + 8 * w, h = cur.h * c.group + row - tok[w] * c.group;
            const long long t = cur.a.t0 + tok[w];
            const float inv = lt[w] > 0.f || lt[w] != lt[w] ? 1.f / lt[w] : 0.f;   // no visible key: zeros
            uint16_t *op = c.out + t * c.o_st + h * c.o_sh + 2 * tig;
#pragma unroll
            for (int n = 0; n < NT; n++)
              *reinterpret_cast<uint32_t *>(op + 8 * n) = pack2<F16>(o[n][2 * w] * inv, o[n][2 * w + 1] * inv);
            if (c.lse && tig == 0)
              c.lse[t * c.n_heads + h] = lt[w] == 0.f ? -INFINITY : (mt[w] + log2f(lt[w])) * 0.6931471805599453f;
          }
        } else {
          // a block's first item may come from the block before (part 0), its last go on in the next (part 1)
          float *d = parts + (long long)(2 * blockIdx.x + (starts ? 1 : 0)) * rows_part_floats<HD>();
#pragma unroll
          for (int w = 0; w < 2; w++) {
            const int row = gid + 8 * w;
#pragma unroll
            for (int n = 0; n < NT; n++)
              *reinterpret_cast<float2 *>(d + row * HD + 8 * n + 2 * tig) = make_float2(o[n][2 * w], o[n][2 * w + 1]);
            if (tig == 0) *reinterpret_cast<float2 *>(d + ROWS_M * HD + 2 * row) = make_float2(mt[w], lt[w]);
          }
          if (starts && lane == 0) {
            // the block of the item's last unit: b with total b / blocks <= that unit
            const long long end = u0 + u + (cur.chunks - 1 - cur.ch);
            int b = (int)((end * blocks) / total);
            while (b + 1 < blocks && total * (b + 1) / blocks <= end) b++;
            cuts[blockIdx.x] = RowsCut{cur.r, cur.rg, cur.h, b};
          }
        }
      }
      fresh = true;
      starts = true;
    }
    cur.next(c, row_limit);
  }
  cp_wait<0>();
  raise_status(c.status, bad);
}

// Joins the parts of the item that block blockIdx.x cut: part 1 of that block,
// then part 0 of the following ones, in that order.
template <int HD, bool F16, bool PAGED>
__global__ void __launch_bounds__(HD)
rows_join_kernel(const AttnCall c, const float *__restrict__ parts, const RowsCut *__restrict__ cuts) {
  pdl_wait();
  const RowsCut cut = cuts[blockIdx.x];
  if (cut.last < 0) return;
  const AttnReq a = attn_request<PAGED>(c, cut.r);
  const int d = threadIdx.x, b0 = blockIdx.x;
  constexpr int PF = rows_part_floats<HD>();
  auto part = [&](int b) { return parts + (long long)(2 * b + (b == b0 ? 1 : 0)) * PF; };
  for (int i = 0; i < ROWS_M; i++) {
    const int row = cut.rg * ROWS_M + i, t = row / c.group, h = cut.h * c.group + row - t * c.group;
    if (t >= a.n) return;
    float m = -INFINITY;
    for (int b = b0; b <= cut.last; b++) m = fmaxf(m, part(b)[ROWS_M * HD + 2 * i]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
    for (int b = b0; b <= cut.last; b++) {
      const float *p = part(b), f = exp2_approx(p[ROWS_M * HD + 2 * i] - base);
      l += p[ROWS_M * HD + 2 * i + 1] * f;
      o += p[i * HD + d] * f;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const long long at = a.t0 + t;
    c.out[at * c.o_st + h * c.o_sh + d] = (uint16_t)pack2<F16>(o * inv, 0.f);
    if (c.lse && d == 0) c.lse[at * c.n_heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}

// ------------------------------------------------------------------ host ---
static inline size_t rows_workspace(int hd, int sms) {
  const size_t grid = (size_t)sms * ROWS_PER_SM;
  return grid * 16 + grid * 2 * (size_t)(hd == 128 ? rows_part_floats<128>() : rows_part_floats<64>()) * 4;
}

template <int HD, bool F16, bool PAGED>
static cudaError_t rows_prepare_one() {
  return cudaFuncSetAttribute(rows_kernel<HD, F16, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, rows_smem<HD>());
}
static inline cudaError_t rows_prepare() {
  cudaError_t e;
  if ((e = rows_prepare_one<128, false, false>()) != cudaSuccess) return e;
  if ((e = rows_prepare_one<128, false, true>()) != cudaSuccess) return e;
  if ((e = rows_prepare_one<128, true, false>()) != cudaSuccess) return e;
  if ((e = rows_prepare_one<128, true, true>()) != cudaSuccess) return e;
  if ((e = rows_prepare_one<64, false, false>()) != cudaSuccess) return e;
  if ((e = rows_prepare_one<64, false, true>()) != cudaSuccess) return e;
  if ((e = rows_prepare_one<64, true, false>()) != cudaSuccess) return e;
  return rows_prepare_one<64, true, true>();
}

template <int HD, bool F16, bool PAGED>
static cudaError_t rows_launch_one(const AttnCall &c, int sms, int row_limit, void *ws, cudaStream_t st) {
  const int grid = sms * ROWS_PER_SM;
  RowsCut *cuts = static_cast<RowsCut *>(ws);
  float *parts = reinterpret_cast<float *>(static_cast<char *>(ws) + (size_t)grid * sizeof(RowsCut));
  rows_kernel<HD, F16, PAGED><<<grid, ROWS_THREADS, rows_smem<HD>(), st>>>(c, row_limit, parts, cuts);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(HD);
  cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rows_join_kernel<HD, F16, PAGED>, c, (const float *)parts, (const RowsCut *)cuts);
}
// Requests with at most row_limit query rows to a key head are served.
static inline cudaError_t rows_launch(const AttnCall &c, bool paged, bool f16, int hd, int sms, int row_limit, void *ws,
                                      cudaStream_t st) {
  if (hd == 128) {
    if (f16) return paged ? rows_launch_one<128, true, true>(c, sms, row_limit, ws, st) : rows_launch_one<128, true, false>(c, sms, row_limit, ws, st);
    return paged ? rows_launch_one<128, false, true>(c, sms, row_limit, ws, st) : rows_launch_one<128, false, false>(c, sms, row_limit, ws, st);
  }
  if (f16) return paged ? rows_launch_one<64, true, true>(c, sms, row_limit, ws, st) : rows_launch_one<64, true, false>(c, sms, row_limit, ws, st);
  return paged ? rows_launch_one<64, false, true>(c, sms, row_limit, ws, st) : rows_launch_one<64, false, false>(c, sms, row_limit, ws, st);
}

}  // namespace qtb
