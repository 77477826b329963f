// qtb_attn_rows.cuh -- attention of few query rows over many keys.
//
// A query row is one (token, query head); the rows of a request that share a
// key head (token-major, the group's heads inside) are taken 16 at a time, the
// M of mma.m16n8k16, so that grouped heads and the tokens of a short chunk read
// K and V once.  Scores are in units of log2 (scale * log2 e folded in), and
// each warp keeps a maximum m, the sum l of 2^(s - m) and the output O of its
// own keys.  States of any two key sets join (m the larger, the other's l and O
// scaled), so the key axis is cut freely: the (request, row group, key head,
// 64-key chunk) units of the whole call are dealt out to the grid in equal
// runs, whatever the requests' lengths.  An item that a block holds whole is
// written at once; one that is cut leaves its parts (O, m, l in f32) in the
// workspace, and join_kernel adds them in block order, so results do not depend
// on timing.
//
// m is renewed lazily, when a score passes it by 8: until then the
// probabilities are at most 2^8 and the quotient O / l does not care.
//
// What bounds it is the stream of K and V.  One warp copies by TMA (a box is a
// run of a page's positions with all of its dims, 128-byte swizzle), four
// compute; two blocks of three 64-key stages on an SM keep up to 192 KB in
// flight.  (Copies of 16 bytes issued by the computing warps themselves reached
// half the rate.)  Keys outside the request may hold anything: their scores
// become -inf and their V is masked to zero in registers.
//
// Measured, with the join: 128 requests of 4096 to 16384 keys, 32 / 4 heads, pages
// of 64: 423 to 430 us, 6.5 TB/s, the rate of a plain copy; 64 requests of 256 to
// 4096 keys, 16 / 8 heads, pages of 16: 85 us, 5.75 TB/s; one request of 4096
// keys: 11 us, the latency of two dependent launches.
#pragma once
#include "qtb_paged.cuh"
#include <cuda.h>

namespace qtb {

constexpr int ROWS_WARPS = 4, ROWS_THREADS = 32 * (ROWS_WARPS + 1), ROWS_M = 16, ROWS_CHUNK = 64, ROWS_PER_SM = 2;
constexpr long long ROWS_WAIT = 4000000000ll;   // cycles: about two seconds
// Units of work, which a block counts in 32 bits: as many keys as this take a quarter
// of an hour.  Requests that offsets which fall let share their tokens could ask for more.
constexpr long long ROWS_UNITS = 1ll << 38;

struct RowsMaps {
  CUtensorMap k, v;
};

template <int HD>
constexpr int rows_part_floats() { return ROWS_M * (HD + 2); }   // O rows, then (m, l) pairs
template <int HD>
constexpr int rows_stages() { return HD == 128 ? 3 : 6; }
template <int HD>
constexpr int rows_keys_bytes() { return ROWS_CHUNK * HD * 2; }
template <int HD>
constexpr int rows_smem() { return rows_stages<HD>() * 2 * rows_keys_bytes<HD>() + 2 * 32 * (HD / 2) * 4; }

// A position in the call's sequence of units.
template <bool PAGED>
struct RowsCursor {
  AttnReq a;
  int r, rg, h, ch;      // request, row group, key head, chunk within the item
  int groups, chunks, c0;

  QTB_DEV void load(const AttnCall &c) {   // the request's counts
    a = attn_request<PAGED>(c, r);
    groups = (a.n * c.group + ROWS_M - 1) / ROWS_M;
    c0 = a.lo / ROWS_CHUNK;
    chunks = max((a.hi + ROWS_CHUNK - 1) / ROWS_CHUNK - c0, 1);
  }
  QTB_DEV long long units(const AttnCall &c) const { return (long long)groups * c.n_kv * chunks; }
  QTB_DEV void next(const AttnCall &c) {
    if (++ch < chunks) return;
    ch = 0;
    if (++h < c.n_kv) return;
    h = 0;
    if (++rg < groups) return;
    rg = 0;
    do {
      r++;
      if (r >= c.n_req) { groups = 1; chunks = 1; return; }   // past the end: never served
      load(c);
    } while (groups == 0);
  }
};

struct RowsShared {
  uint64_t full[8], empty[8];
  long long sum[ROWS_WARPS + 1], off;      // off: the first unit's index within its request
  int req, abort;
  float2 ml[ROWS_WARPS][ROWS_M];
};

template <int HD, bool F16, bool PAGED>
__global__ void __launch_bounds__(ROWS_THREADS, ROWS_PER_SM)
rows_kernel(const AttnCall c, const __grid_constant__ RowsMaps maps, int box, float *__restrict__ parts,
            AttnCut *__restrict__ cuts) {
  constexpr int KS = HD / 16;              // k-steps of Q K^T
  constexpr int NT = HD / 8;               // 8-wide output tiles
  constexpr int STAGES = rows_stages<HD>(), KEYS_B = rows_keys_bytes<HD>();
  extern __shared__ __align__(1024) unsigned char rows_smem_base[];
  unsigned char *smem = rows_smem_base;
  float *s_red = reinterpret_cast<float *>(smem + STAGES * 2 * KEYS_B);   // [2][HD / 2][32]
  __shared__ RowsShared sh;

  const int tid = threadIdx.x, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  pdl_release();                           // the join kernel's blocks may come up; they wait for this grid's end

  // --- this block's run of units: thread i counts requests [i n / 160, (i + 1) n / 160)
  if (tid == 0) {
    for (int i = 0; i < STAGES; i++) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], ROWS_WARPS); }
    sh.abort = 0;
    fence_mbar_init();
  }
  RowsCursor<PAGED> cur;
  const int ra = (int)((long long)c.n_req * tid / ROWS_THREADS), rb = (int)((long long)c.n_req * (tid + 1) / ROWS_THREADS);
  long long sum = 0;
  int wrong = 0;
  for (cur.r = ra; cur.r < rb; cur.r++) {
    cur.load(c);
    sum = min(sum + cur.units(c), ROWS_UNITS);
    if (blockIdx.x == 0) wrong |= attn_wrong<PAGED>(c, cur.r);
  }
  raise_status(c.status, wrong);
  long long pre = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, pre, o);
    if (lane >= o) pre += x;
  }
  if (lane == 31) sh.sum[warp] = pre;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w <= ROWS_WARPS; w++) {
    if (w < warp) pre += sh.sum[w];
    total += sh.sum[w];
  }
  pre -= sum;
  if (total >= ROWS_UNITS) {               // no work
    if (blockIdx.x == 0 && tid == 0) raise_status(c.status, QTB_PS_LENGTH);
    total = 0;
  }
  const long long blocks = min((long long)gridDim.x, total);
  if (tid == 0) cuts[blockIdx.x].last = -1;
  if (blockIdx.x >= blocks) return;
  const long long u0 = total * blockIdx.x / blocks, u1 = total * (blockIdx.x + 1) / blocks;
  if (u0 >= pre && u0 < pre + sum) {
    long long at = pre;
    for (cur.r = ra; cur.r < rb; cur.r++) {
      cur.load(c);
      const long long n = cur.units(c);
      if (u0 < at + n) break;
      at += n;
    }
    sh.req = cur.r;
    sh.off = u0 - at;
  }
  __syncthreads();
  cur.r = sh.req;
  cur.load(c);
  {
    unsigned long long off = (unsigned long long)sh.off;
    cur.ch = (int)(off % (unsigned)cur.chunks);
    off /= (unsigned)cur.chunks;
    cur.h = (int)(off % (unsigned)c.n_kv);
    cur.rg = (int)(off / (unsigned)c.n_kv);
  }
  const int n_units = (int)(u1 - u0);

  // Bounded wait; one that runs out lets the block run on without data, so that
  // its own barriers are met, and reports it.
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (mbar_wait(bar, parity, 20000)) return true;
    const long long t0 = clock64();
    while (!*reinterpret_cast<volatile int *>(&sh.abort)) {
      if (mbar_wait(bar, parity, 20000)) return true;
      if (clock64() - t0 > ROWS_WAIT) {
        *reinterpret_cast<volatile int *>(&sh.abort) = 1;
        raise_status(c.status, QTB_PS_TIMEOUT);
      }
    }
    return false;
  };

  if (warp == ROWS_WARPS) {
    // ------------------------------------------------------------- loads ---
    // Lanes 0-3 have the chunk's boxes of K, lanes 4-7 of V.
    const int boxes = ROWS_CHUNK / box, bi = lane & 3, kv = (lane >> 2) & 1;
    const uint32_t bytes = (uint32_t)(box * HD * 2);
    unsigned char *dst0 = smem + kv * KEYS_B + bi * bytes;
    const CUtensorMap *map = kv ? &maps.v : &maps.k;
    int bad = 0, u = 0, pg = 0, off = 0;
    bool mine = false;
    auto find = [&]() {                    // this lane's box of the cursor's chunk
      const int pos = (cur.c0 + cur.ch) * ROWS_CHUNK + bi * box;
      mine = lane < 8 && bi < boxes && pos < cur.a.hi && pos + box > cur.a.lo;
      if (PAGED) {
        if (mine) {
          const int e = pos / c.page;
          off = pos - e * c.page;
          pg = c.table[cur.r * c.table_stride + e];
        }
      } else {
        off = cur.a.t0 + pos;
      }
    };
    find();
    for (; u < n_units; u++) {
      const int st = u % STAGES;
      if (!__all_sync(0xffffffffu, wait(&sh.empty[st], ((u / STAGES) & 1) ^ 1))) break;
      const int count = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_arrive_expect_tx(&sh.full[st], (uint32_t)count * bytes);
      __syncwarp();
      if (mine) {
        if (PAGED && (pg < 0 || pg >= c.n_pages)) { pg = c.n_pages; bad = QTB_PS_PAGE; }   // past the last page: zeros
        tma_load_5d(dst0 + st * 2 * KEYS_B, map, 0, off, 0, cur.h, PAGED ? pg : 0, &sh.full[st]);
      }
      cur.next(c);
      if (u + 1 < n_units) find();
    }
    // copies in flight land before the block leaves
    for (int f = max(u - STAGES, 0); f < u; f++) mbar_wait(&sh.full[f % STAGES], (f / STAGES) & 1, ROWS_WAIT);
    raise_status(c.status, bad);
    return;
  }

  // ----------------------------------------------------------------- math ---
  const float scale = fabsf(c.scale_log2);
  const uint32_t flip = c.scale_log2 < 0.f ? 0x80008000u : 0u;   // a negative scale turns the queries' signs
  const uint32_t keep = c.scale_log2 == 0.f ? 0u : 0xffffffffu;  // a scale of zero makes them zeros ...
  const float mul = c.scale_log2 == 0.f ? 1.f : scale;           // ... so that -inf stays -inf
  // this warp's 16 keys within a stage: [box][half][row][128 bytes]
  const int half_b = box * 128;
  const int k_at = (warp * 16 / box) * half_b * (HD / 64) + (warp * 16 % box) * 128;
  const int k_row = (lane & 7) + ((lane & 16) >> 1), k_half = (lane >> 3) & 1, v_row = lane & 15, v_half = lane >> 4;

  uint32_t q[KS][4];
  float o[NT][4], m[2], l[2];
  int last_key[2], first_key[2], tok[2];   // per row: the keys it sees, its token (-1: no row)
  int all_first = 0, all_last = 0;         // keys that every row sees
  bool starts = cur.ch == 0;               // this block holds the current item from its first chunk
  bool fresh = true;

  for (int u = 0; u < n_units; u++) {
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int row = cur.rg * ROWS_M + gid + 8 * i, t = row / c.group, g = row - t * c.group;
        const bool live = t < cur.a.n;
        tok[i] = live ? t : -1;
        last_key[i] = !live ? -1 : min(c.causal ? cur.a.first + t : cur.a.hi - 1, cur.a.hi - 1);
        first_key[i] = c.window > 0 ? max(cur.a.first + t - c.window + 1, 0) : 0;
        const uint16_t *qp = c.q + (long long)(cur.a.t0 + t) * c.q_st + (long long)(cur.h * c.group + g) * c.q_sh + 2 * tig;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          q[k][i] = live ? (__ldg(reinterpret_cast<const uint32_t *>(qp + 16 * k)) ^ flip) & keep : 0u;
          q[k][2 + i] = live ? (__ldg(reinterpret_cast<const uint32_t *>(qp + 16 * k + 8)) ^ flip) & keep : 0u;
        }
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      const int t_a = cur.rg * ROWS_M / c.group, t_b = min((cur.rg * ROWS_M + ROWS_M - 1) / c.group, cur.a.n - 1);
      all_last = min(c.causal ? cur.a.first + t_a : cur.a.hi - 1, cur.a.hi - 1);
      all_first = c.window > 0 ? max(cur.a.first + t_b - c.window + 1, 0) : 0;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[n][i] = 0.f;
    }
    const int st = u % STAGES;
    wait(&sh.full[st], (u / STAGES) & 1);
    __syncwarp();

    // --- this warp's 16 keys of the chunk
    const unsigned char *ks = smem + st * 2 * KEYS_B + k_at, *vs = ks + KEYS_B;
    const int key0 = (cur.c0 + cur.ch) * ROWS_CHUNK + warp * 16;
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < KS; k++) {
      uint32_t b[4];
      ldsm_x4(b, ks + (k >> 2) * half_b + k_row * 128 + ((((2 * k) & 7) + k_half) ^ (k_row & 7)) * 16);
      mma16<F16>(s[0], q[k], b[0], b[1]);
      mma16<F16>(s[1], q[k], b[2], b[3]);
    }
    uint32_t vmask[2] = {0xffffffffu, 0xffffffffu};   // of keys 2 tig, 2 tig + 1 and those 8 on
    if (key0 < all_first || key0 + 15 > all_last) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const int key = key0 + 8 * t + 2 * tig;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (key + (i & 1) > last_key[i >> 1] || key + (i & 1) < first_key[i >> 1]) s[t][i] = -INFINITY;
        vmask[t] = (key >= cur.a.lo && key < cur.a.hi ? 0xffffu : 0u) | (key + 1 >= cur.a.lo && key + 1 < cur.a.hi ? 0xffff0000u : 0u);
      }
    }
    float mx[2];
#pragma unroll
    for (int w = 0; w < 2; w++)
      mx[w] = fmaxf(fmaxf(s[0][2 * w], s[0][2 * w + 1]), fmaxf(s[1][2 * w], s[1][2 * w + 1])) * mul;
    if (__any_sync(0xffffffffu, mx[0] > m[0] + 8.f || mx[1] > m[1] + 8.f)) {
#pragma unroll
      for (int w = 0; w < 2; w++) {
        mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
        mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
        const float m2 = fmaxf(m[w], mx[w]), f = m2 == -INFINITY ? 1.f : exp2_approx(m[w] - m2);
        m[w] = m2;
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
        s[t][i] = exp2_approx(fmaf(s[t][i], mul, -base[i >> 1]));
        l[i >> 1] += s[t][i];
      }
    // probabilities are rounded to the cache's type for the product with V, as
    // large as the result's own rounding; their sum l is of the unrounded ones
    const uint32_t pa[4] = {pack2<F16>(s[0][0], s[0][1]), pack2<F16>(s[0][2], s[0][3]),
                            pack2<F16>(s[1][0], s[1][1]), pack2<F16>(s[1][2], s[1][3])};
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t b[4];
      ldsm_x4_trans(b, vs + (n >> 3) * half_b + v_row * 128 + (((n & 7) + v_half) ^ (v_row & 7)) * 16);
      mma16<F16>(o[n], pa, b[0] & vmask[0], b[1] & vmask[1]);
      mma16<F16>(o[n + 1], pa, b[2] & vmask[0], b[3] & vmask[1]);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[st]);

    const bool ends = cur.ch == cur.chunks - 1;
    if (ends || u + 1 == n_units) {
      // --- join the four warps' states
#pragma unroll
      for (int w = 0; w < 2; w++) {
        l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
        l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
        if (tig == 0) sh.ml[warp][gid + 8 * w] = make_float2(m[w], l[w]);
      }
      bar_sync_n(1, 32 * ROWS_WARPS);
      float mt[2], lt[2];
#pragma unroll
      for (int w = 0; w < 2; w++) {
        mt[w] = -INFINITY;
        lt[w] = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS_WARPS; i++) mt[w] = fmaxf(mt[w], sh.ml[i][gid + 8 * w].x);
        const float b = mt[w] == -INFINITY ? 0.f : mt[w];
#pragma unroll
        for (int i = 0; i < ROWS_WARPS; i++) {
          const float2 x = sh.ml[i][gid + 8 * w];
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
        bar_sync_n(1, 32 * ROWS_WARPS);
        if (warp < half) {
          const float *d = s_red + warp * 32 * (HD / 2);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[n][i] += d[(n * 4 + i) * 32 + lane];
        }
        bar_sync_n(1, 32 * ROWS_WARPS);
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
            if (tok[w] < 0) continue;
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
            cuts[blockIdx.x] = AttnCut{b, cur.a.t0, cur.a.n, cur.h * c.group, cur.rg * ROWS_M, ROWS_M, {0, 0}};
          }
        }
      }
      fresh = true;
      starts = true;
    }
    cur.next(c);
  }
}

// ------------------------------------------------------------------ host ---
static inline size_t rows_workspace(int hd, int sms) {
  const size_t grid = (size_t)sms * ROWS_PER_SM;
  return grid * sizeof(AttnCut) + grid * 2 * (size_t)(hd == 128 ? rows_part_floats<128>() : rows_part_floats<64>()) * 4;
}

// Keys in boxes of a run of a page's positions, all dims: [dim / 64][position][64].
static inline int rows_box(bool paged, int page) {
  int b = ROWS_CHUNK;
  while (paged && page % b) b >>= 1;
  return b;
}
static inline bool rows_maps(const AttnCall &c, bool paged, bool f16, int hd, TensorMapFn fn, RowsMaps &m) {
  const long long pos = paged ? c.page : c.n_tokens, pages = paged ? c.n_pages : 1;
  auto one = [&](CUtensorMap *out, const uint16_t *base, const long long *st) {
    const long long ext[5] = {64, pos, hd / 64, c.n_kv, pages};
    const long long str[5] = {1, paged ? st[2] : st[0], 64, st[1], paged ? st[0] : 0};
    const int box[5] = {64, rows_box(paged, c.page), hd / 64, 1, 1};
    return tensor_map(fn, out, base, f16, 5, ext, str, box);
  };
  return one(&m.k, c.k, c.k_st) && one(&m.v, c.v, c.v_st);
}

template <int HD, bool F16, bool PAGED>
static cudaError_t rows_run(bool prepare, const AttnCall *c, const RowsMaps *m, int sms, int max_rows, void *ws,
                            cudaStream_t st) {
  if (prepare)
    return cudaFuncSetAttribute(rows_kernel<HD, F16, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, rows_smem<HD>());
  const int grid = sms * ROWS_PER_SM;
  AttnCut *cuts = static_cast<AttnCut *>(ws);
  float *parts = reinterpret_cast<float *>(cuts + grid);
  rows_kernel<HD, F16, PAGED><<<grid, ROWS_THREADS, rows_smem<HD>(), st>>>(*c, *m, rows_box(PAGED, c->page), parts, cuts);
  if (cudaError_t e = cudaGetLastError()) return e;
  return launch_early(join_kernel<HD, F16, ROWS_M, 1, JOIN_WARPS, 1>, dim3(grid, max_rows), 32 * JOIN_WARPS, 0, st, *c, (const float *)parts,
                      (const AttnCut *)cuts);
}
// max_rows: how many rows (of 16) an item has, as far as known.
static inline cudaError_t rows_any(bool prepare, int which, const AttnCall *c, const RowsMaps *m, int sms, int max_rows,
                                   void *ws, cudaStream_t st) {
  switch (which) {
    case 0: return rows_run<64, false, false>(prepare, c, m, sms, max_rows, ws, st);
    case 1: return rows_run<64, false, true>(prepare, c, m, sms, max_rows, ws, st);
    case 2: return rows_run<64, true, false>(prepare, c, m, sms, max_rows, ws, st);
    case 3: return rows_run<64, true, true>(prepare, c, m, sms, max_rows, ws, st);
    case 4: return rows_run<128, false, false>(prepare, c, m, sms, max_rows, ws, st);
    case 5: return rows_run<128, false, true>(prepare, c, m, sms, max_rows, ws, st);
    case 6: return rows_run<128, true, false>(prepare, c, m, sms, max_rows, ws, st);
    default: return rows_run<128, true, true>(prepare, c, m, sms, max_rows, ws, st);
  }
}
static inline cudaError_t rows_prepare() {
  for (int i = 0; i < 8; i++)
    if (cudaError_t e = rows_any(true, i, nullptr, nullptr, 0, 0, nullptr, nullptr)) return e;
  return cudaSuccess;
}
static inline cudaError_t rows_launch(const AttnCall &c, bool paged, bool f16, int hd, const RowsMaps &m, int sms, int max_rows,
                                       void *ws, cudaStream_t st) {
  return rows_any(false, (hd == 128 ? 4 : 0) + (f16 ? 2 : 0) + (paged ? 1 : 0), &c, &m, sms, max_rows, ws, st);
}

}  // namespace qtb
