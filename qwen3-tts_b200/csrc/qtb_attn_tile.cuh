// qtb_attn_tile.cuh -- attention of many query rows on the 5th-generation
// tensor cores.
//
// A query row is one (token, query head).  The rows of a request that share a
// key head, token-major with the group's heads inside, fill tiles of 128 (as
// many whole tokens as fit); a block works on two such tiles at a time, against
// key tiles of 128, in two waves that hide each other:
//
//   load warp      Q tiles, and K_0 V_0 K_1 V_1 ... by TMA into a ring (128-byte
//                  swizzle; a paged key tile is one box per run of a page's
//                  positions)
//   MMA warp       S = Q K^T into tensor memory, and O += P V with P from there;
//                  tile 0's products run while tile 1's softmax does, and back
//   warps 0-3, 4-7 softmax of tile 0, of tile 1: a thread has a row
//   (warps 8 and 9 load and issue; 10 and 11 fill their warpgroup)
//
// Tensor memory (512 columns): S of both tiles (128 each; P, in the tensors'
// type, takes S's place), O of both (head_dim each).
//
// The running maximum is renewed lazily: with scores in units of log2 (scale *
// log2 e folded in), p = 2^(s - m) where m is a maximum seen so far, at most
// 8 below the true one, so p <= 2^8 and the sum stays exact to f32 rounding;
// only when a row outgrows that are its O and l scaled.  The final O / l does
// not depend on m.
// The probabilities of a tile start from the old maximum at once, beside the new
// maximum's search, and are thrown away in the rare tile that outgrows it.
//
// A pair whose second tile has no token (a decoding request, a short chunk, the
// end of a prompt) would leave half of the pipeline idle: there both tiles' warps
// take the same rows, tile 0 every other key tile and tile 1 those between, and
// their two states are joined in tensor memory at the end ("twin": 64 requests of 8
// tokens over 4000 keys 199 -> 186 us, a mixed call of 16 requests, cut, 152 -> 135).
//
// An item of work is a tile pair and a key head.  Where whole items fill the
// blocks evenly enough, they are dealt out whole, longest first.  Where not, the
// key tiles of all are dealt out in equal runs, whatever the requests' lengths; an
// item that is cut between blocks leaves its parts in the workspace, and
// join_kernel adds them.  Cutting costs the parts, the join and the key tiles'
// reuse in L2, since blocks then walk the keys at as many places as there are
// blocks.  Evenly enough: the fullest block has at most 5/4 of the mean and 5 steps
// (us, whole / cut, at fullest and mean: 16 mixed requests 123 / 134 at 69 and 59;
// 33 of 1 to 74 tokens 22 / 29 at 10 and 9; 37 of 1 to 3 tokens 15 / 19 at 6 and 2;
// 16 prompts of 1973 to 7895 147 / 107 at 94 and 54; 8 x 64 tokens over 8192 keys
// 129 / 73 at 50 and 22; 64 tokens over 2112 keys 37 / 21 at 15 and 1).
//
// What bounds it.  A step (two query tiles, one key tile) needs 2048 cycles of the
// tensor pipe at 128 dims and 2048 of the MUFU's exponentials, and takes about
// 3400: both pipes 60 % busy (8192-token prompt, 16 / 8 heads), with the chain
// scores - softmax - P V - next scores of one tile under the other's.  Tried and
// not kept (8192 tokens): a quarter of the exponentials by a polynomial on the FMA
// pipe (-2 to -4 %), two threads to a row (-18 %), P handed over in one piece
// (-1 %), in three (-11 %).  Measured: a 16384-token prompt, 16 / 8 heads, 128 dims
// 835 to 960 us by the clock that the power limit leaves (1150 to 1320 TFLOP/s);
// 8192 tokens 215 to 225 us, of 64 dims, where the exponentials weigh twice, 188
// us (730 TFLOP/s).  A short call is its start: 64 tokens take 9 us, of which a
// launch is 2 and most of the rest code fetched for the first time.
//
// Products are issued in order, so the commit that completes S of tile j also
// says that P V of tile j - 1 is in O: the softmax warps may scale O then.
// Every wait is bounded; one that runs out raises QTB_PS_TIMEOUT, and the roles
// run on to their end without waiting (what they then read and write lies within
// the block's own buffers and outputs).
#pragma once
#include <climits>

#include "qtb_paged.cuh"

namespace qtb {

constexpr int TILE_THREADS = 384, TILE_M = 128, TILE_N = 128;
// Registers of a thread: the block starts with 168 for each of its 384 threads
// (64512 in all); the softmax warps, a row of S each, take what the loading and
// issuing warpgroup gives up: 256 * 208 + 128 * 80 = 256 * 200 + 128 * 96 = 63488.
// (16384-token prompt of 128 dims 845 us with 208, 859 with 200; 8192 tokens of 64
// dims 192 and 185.)
template <int HD>
constexpr int tile_regs_softmax() { return HD == 128 ? 208 : 200; }
template <int HD>
constexpr int tile_regs_other() { return HD == 128 ? 80 : 96; }
constexpr int TILE_START = 2;              // what starting an item costs, in its steps over a key tile
constexpr int TILE_CUT = 1;                // steps that a block has of an item at least, where it has not all
constexpr int TILE_PAIRS = 256;            // pairs whose costs are looked at: as many as shared memory has room for
constexpr int TILE_SEGS = 64;              // runs of requests that the in-block search tells apart
constexpr int TILE_RUN = (1 << 25) - 1;    // pairs in a run: more than all of a call can be
constexpr long long TILE_WAIT = 4000000000ll;   // cycles: about two seconds

template <int HD>
constexpr int tile_stages() { return HD == 128 ? 5 : 8; }
template <int HD>
constexpr int tile_kv_bytes() { return TILE_N * HD * 2; }
template <int HD>
constexpr int tile_operands() { return 2 * TILE_M * HD * 2 + tile_stages<HD>() * tile_kv_bytes<HD>(); }

template <int HD>
constexpr int tile_part_floats() { return TILE_M * (HD + 2); }   // O rows, then (m, l) pairs

struct TileMaps {
  CUtensorMap q, k, v;
};

struct TileSync {
  uint64_t q_full, q_empty, drain;
  uint64_t s_full[2], p_full[2][2], o_full[2], o_empty[2];
  uint64_t kv_full[8], kv_empty[8];
  uint32_t tmem;
  int abort;
};

// Whether a single request's `items` fill `sms` blocks evenly enough to be dealt out
// whole, as its launch sees it; a kernel with a workspace looks at their lengths.
inline bool tile_whole(long long items, int sms) {
  return 2 * items >= 5 * sms || (items <= sms && 4 * items >= 3 * sms);
}

// What lies in shared memory behind the operands (which start it, on 1024 bytes).
struct TileShared {
  TileSync sy;
  int pre[TILE_SEGS + 1];                  // query tile pairs before each run of requests
  // the requests themselves, where a run is one: in order of their keys, so that
  // items taken from the last to the first begin with the longest
  int t0[TILE_SEGS], n[TILE_SEGS], hi[TILE_SEGS], first[TILE_SEGS];
  unsigned char r[TILE_SEGS];
  long long scan[TILE_THREADS / 32];
  int most[TILE_THREADS / 32];
  int item[2], off[2];                     // the block's first item and place in it, and where the next block's are
  union {
    int cost[TILE_PAIRS];                  // of each pair, while the work is shared out
    float2 ml[TILE_M];                     // (m, l) of a twin item's second state
  };
  unsigned char order[TILE_PAIRS];         // the pairs by cost, where they are dealt out so
  long long base;                          // units of work before item[1]
};
template <int HD>
constexpr int tile_smem() { return tile_operands<HD>() + (int)sizeof(TileShared); }
static_assert(tile_smem<128>() <= 232448 && tile_smem<64>() <= 232448, "shared memory of a block");

// D (+)= A B with A in tensor memory.
QTB_DEV void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of an operand whose N (or M) axis is contiguous: 64 elements of it
// per 128-byte swizzled row, rows along K, 8-row groups 1024 bytes apart, the
// next 64 elements `chunk` bytes further on.
QTB_DEV uint64_t umma_desc_mn128(uint32_t saddr, uint32_t chunk) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)((chunk >> 4) & 0x3fffu) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
QTB_DEV void tmem_ld32_async(uint32_t taddr, float *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
QTB_DEV void tmem_ld8_async(uint32_t taddr, float *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
      : "r"(taddr));
}
QTB_DEV void tmem_ld16_async(uint32_t taddr, float *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr));
}
QTB_DEV void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
QTB_DEV void tmem_st16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
QTB_DEV void tmem_st8(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
      : "memory");
}
QTB_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
QTB_DEV void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
QTB_DEV void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Waits for a phase, for a bounded number of the hardware's suspensions; 0 where it
// has not completed.  (The loop is written out: the MMA warp's reaction to a
// barrier is on the path between two tiles.)
QTB_DEV uint32_t mbar_tries(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 1024;\n\t"
      "MBAR_TRY:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra MBAR_DONE;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, n, 0;\n\t"
      "@q bra MBAR_TRY;\n\t"
      "MBAR_DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done;
}
QTB_DEV bool tile_wait_long(uint32_t bar, uint32_t parity, volatile int *abort, int *status) {
  const long long t0 = clock64();
  while (!*abort) {
    if (mbar_tries(bar, parity)) return true;
    if (clock64() - t0 > TILE_WAIT) {
      *abort = 1;
      raise_status(status, QTB_PS_TIMEOUT);
    }
  }
  return false;
}
// True in one lane of the (converged) warp, always the same one.
QTB_DEV bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
QTB_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two f32 values in a register pair, and their sum / product-sum in one instruction.
QTB_DEV uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
QTB_DEV void f2_get(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
QTB_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
QTB_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// One unit of work: 2 tpt tokens (a tile pair) of a request, one key head.
struct TileItem {
  int r, h, t0, tok;    // request, key head, the request's first packed token, first token of the pair
  int first, end, n;    // position of the request's token 0, its keys, its tokens
  int low;              // keys before this are seen by no row of the pair
  int k0;               // first key of key tile 0 (a multiple of 128)
  int tok0, tok1;       // tokens in each tile
  int from, n0, n1;     // key tiles [from, n0) are this block's for query tile 0, [from, n1) for tile 1
  bool whole;           // those are all
  bool twin;            // no tile 1: of [from, n0) = [from, n1) tile 0's warps take every other one, tile 1's the rest
  int high;             // keys at and past this are seen by no row
};

template <int HD, bool F16, bool PAGED>
__global__ void __launch_bounds__(TILE_THREADS, 1)
tile_kernel(const AttnCall c, const __grid_constant__ TileMaps maps, int tpt, int box,
            float *__restrict__ parts, AttnCut *__restrict__ cuts) {
  constexpr int STAGES = tile_stages<HD>(), KV_B = tile_kv_bytes<HD>(), Q_B = TILE_M * HD * 2, HALF_B = TILE_M * 128;
  constexpr uint32_t S_COL = 0, O_COL = 256;
  extern __shared__ __align__(1024) unsigned char tile_smem_base[];
  unsigned char *smem = tile_smem_base;
  TileShared &sh = *reinterpret_cast<TileShared *>(smem + tile_operands<HD>());
  TileSync &sy = sh.sy;
  unsigned char *s_q = smem, *s_kv = smem + 2 * Q_B;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // known to be the same in the whole warp
  if (parts) pdl_release();                // the join kernel's blocks may come up; they wait for this grid's end
  if (warp == 8) {
    if (lane < 3) {
      const CUtensorMap *m = lane == 0 ? &maps.q : lane == 1 ? &maps.k : &maps.v;
      asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
  } else if (warp == 9) {
    tmem_alloc(&sy.tmem, 512);
  } else if (tid == 10 * 32) {
    mbar_init(&sy.q_full, 1); mbar_init(&sy.q_empty, 1); mbar_init(&sy.drain, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sy.s_full[i], 1); mbar_init(&sy.p_full[i][0], 4); mbar_init(&sy.p_full[i][1], 4);
      mbar_init(&sy.o_full[i], 1); mbar_init(&sy.o_empty[i], 4);
    }
    for (int i = 0; i < STAGES; i++) { mbar_init(&sy.kv_full[i], 1); mbar_init(&sy.kv_empty[i], 1); }
    sy.abort = 0;
    fence_mbar_init();
  }
  // --- pairs of every request, summed over runs of requests: one of the first TILE_SEGS threads has a run
  const int seg = (c.n_req + TILE_SEGS - 1) / TILE_SEGS;
  auto pairs_of = [&](int n) { return (n + 2 * tpt - 1) / (2 * tpt); };
  int sum = 0, pre = 0, wrong = 0;
  if (seg > 1) {
    if (tid < TILE_SEGS)
      for (int r = tid * seg; r < min((tid + 1) * seg, c.n_req); r++) {
        sum = min(sum + pairs_of(attn_request<PAGED>(c, r).n), TILE_RUN);
        if (blockIdx.x == 0) wrong |= attn_wrong<PAGED>(c, r);
      }
  } else {
    AttnReq a = {};
    int place = tid;
    if (tid < c.n_req) {
      a = attn_request<PAGED>(c, tid);
      if (blockIdx.x == 0) wrong = attn_wrong<PAGED>(c, tid);
    }
    if (c.n_req > 1) {
      if (tid < TILE_SEGS) sh.pre[tid] = a.hi;
      __syncthreads();
      if (tid < c.n_req) {
        place = 0;
        for (int r = 0; r < c.n_req; r++) place += sh.pre[r] < a.hi || (sh.pre[r] == a.hi && r < tid);
      }
    }
    if (tid < c.n_req) {
      sh.t0[place] = a.t0; sh.n[place] = a.n; sh.hi[place] = a.hi; sh.first[place] = a.first; sh.r[place] = (unsigned char)tid;
    }
    __syncthreads();
    if (tid < c.n_req) sum = pairs_of(sh.n[tid]);
  }
  raise_status(c.status, wrong);
  if (tid < TILE_SEGS) {
    pre = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += x;
    }
    if (lane == 31) sh.pre[warp] = pre;
  }
  __syncthreads();
  int before = 0, pairs = 0;
#pragma unroll
  for (int w = 0; w < TILE_SEGS / 32; w++) {
    const int x = sh.pre[w];
    if (w < warp) before += x;
    pairs += x;
  }
  // more than requests of tokens of their own can have, as offsets that fall let them: no work
  if (pairs > c.n_tokens / (2 * tpt) + c.n_req) pairs = 0;
  __syncthreads();
  if (tid < TILE_SEGS) sh.pre[tid] = before + pre - sum;
  if (tid == 0) sh.pre[TILE_SEGS] = pairs;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sy.tmem;

  // A query tile pair of a request and its keys; the items of the call are
  // (pair, key head), numbered pair by pair.
  auto get_pair = [&](int p, TileItem &it) {
    int lo = 0;                            // the last run that starts at or before p
#pragma unroll 1
    for (int step = TILE_SEGS / 2; step; step >>= 1)
      if (sh.pre[lo + step] <= p) lo += step;
    p -= sh.pre[lo];
    it.r = sh.r[lo];
    int n_tok = sh.n[lo];
    it.t0 = sh.t0[lo];
    it.end = sh.hi[lo];
    it.first = sh.first[lo];
    if (seg > 1) {
      it.r = lo * seg;
      AttnReq a = attn_request<PAGED>(c, it.r);
      for (int q; p >= (q = pairs_of(a.n)); a = attn_request<PAGED>(c, ++it.r)) p -= q;
      n_tok = a.n; it.t0 = a.t0; it.end = a.hi; it.first = a.first;
    }
    it.n = n_tok;
    it.tok = p * 2 * tpt;
    it.tok0 = min(n_tok - it.tok, tpt);
    it.tok1 = max(min(n_tok - it.tok - tpt, tpt), 0);
    it.low = c.window > 0 ? max(it.first + it.tok - c.window + 1, 0) : 0;
    it.k0 = it.low / TILE_N * TILE_N;
    const int mid = it.first + it.tok + it.tok0;          // position past the tile's last token
    const int hi0 = c.causal ? min(mid, it.end) : it.end, hi1 = c.causal ? min(mid + it.tok1, it.end) : it.end;
    it.n0 = hi0 > it.low ? (hi0 - it.k0 + TILE_N - 1) / TILE_N : 0;
    it.n1 = it.tok1 > 0 && hi1 > it.low ? (hi1 - it.k0 + TILE_N - 1) / TILE_N : 0;
    it.high = max(hi0, hi1);
    it.twin = it.tok1 == 0 && it.n0 > 1;
    if (it.twin) it.n1 = it.n0;
  };
  // What an item costs, in steps of the two query tiles over a key tile.  A key
  // tile of a twin item is three quarters of one (it is half of a step, but of one
  // that loads twice as much): with 1/2, 5/8, 3/4, 7/8, 1 of one a mixed call of 16
  // requests took 162, 139, 142, 150, 154 us, 8 requests of 64 rows and 8000 keys
  // 56.0, 56.6, 54.9, 56.5, 54.5; and with TILE_START 1, 2, 3 at 3/4 142, 137, 135
  // and 54.9, 55.2, 56.4.
  auto cost_of = [&](const TileItem &it) {
    const int n = max(it.n0, it.n1);
    return TILE_START + (it.twin ? (3 * n + 3) >> 2 : n);
  };
  auto tiles_at = [&](const TileItem &it, int off) {       // key tiles that cost off past the start
    return it.twin ? (off - TILE_START) * 4 / 3 : off - TILE_START;
  };
  const int items = pairs * c.n_kv;        // the host has bounded it
  const int grid = (int)gridDim.x;
  // Whole items go from the costliest pair to the cheapest, key heads inside, and to
  // and fro over the blocks, so that the sums come out alike (us, by the requests'
  // lengths / by cost: 3 prompts of 743 to 2974 tokens 67 / 57, 32 of 297 to 1188
  // 66 / 60; the sort costs up to 0.8).  Pairs whose costs are not looked at go from
  // the last to the first, a request's longest causal ones first.
  auto dealt = [&](int n, int block) { return n * grid + (n & 1 ? grid - 1 - block : block); };
  // --- whether they are dealt out whole: a thread adds up a block's.
  const bool known = parts && pairs <= TILE_PAIRS;
  long long total = 0;                     // the cost of all
  bool deal = true;
  if (known) {
    int cost = 0;
    if (tid < pairs) {
      TileItem it;
      get_pair(tid, it);
      sh.cost[tid] = cost = cost_of(it);
    }
    __syncthreads();
    if (tid < pairs) {
      int rank = 0;
#pragma unroll 4
      for (int p = 0; p < pairs; p++) rank += sh.cost[p] > cost || (sh.cost[p] == cost && p > tid);
      sh.order[rank] = (unsigned char)tid;
    }
    __syncthreads();
    int most = 0;
#pragma unroll 1
    for (int b = tid; b < grid; b += TILE_THREADS) {
      long long load = 0;
#pragma unroll 1
      for (int n = 0, i; (i = dealt(n, b)) < items; n++) load += sh.cost[sh.order[(unsigned)i / (unsigned)c.n_kv]];
      total += load;
      most = max(most, (int)min(load, (long long)INT_MAX));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) { sh.scan[warp] = total; sh.most[warp] = most; }
    __syncthreads();
    total = 0;
#pragma unroll 1
    for (int w = 0; w < TILE_THREADS / 32; w++) { total += sh.scan[w]; most = max(most, sh.most[w]); }
    deal = 4ll * grid * most <= 5 * total + 20 * grid;
  }
  // --- this block's run of work; boundaries between blocks move to an item's start
  // or end where less than TILE_CUT steps would be left on that side.
  if (deal) {
    if (tid == 0 && parts) cuts[blockIdx.x].last = -1;
  } else {
    // the costs of the pairs up to this thread's
    const int cost = tid < pairs ? sh.cost[tid] : 0;
    long long upto = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 31) sh.scan[warp] = upto;
    const long long blocks = max(min((long long)grid, total / (2 * TILE_CUT)), 1ll);
    if (tid < 2) {                         // where no boundary is found: past the end
      sh.item[tid] = items;
      sh.off[tid] = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < warp; w++) upto += sh.scan[w];
    const long long first = (upto - cost) * c.n_kv;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (blockIdx.x + e >= blocks) continue;
      const long long x = total * (blockIdx.x + e) / blocks;
      if (x < first || x >= first + (long long)cost * c.n_kv) continue;
      int h = (int)((unsigned)(x - first) / (unsigned)cost), off = (int)(x - first) - h * cost;
      if (off < TILE_START + TILE_CUT) off = 0;
      else if (cost - off < TILE_CUT) { off = 0; h++; }
      sh.item[e] = tid * c.n_kv + h;       // h may be n_kv: the next pair's first
      sh.off[e] = off;
      if (e) sh.base = first + (long long)h * cost;
    }
    __syncthreads();
    if (tid == 10 * 32) {                  // an item that this block begins and does not finish
      int last = -1;
      TileItem it;
      if (blockIdx.x < blocks && sh.off[1] > 0 && !(sh.item[0] == sh.item[1] && sh.off[0] > 0)) {
        get_pair(sh.item[1] / c.n_kv, it);
        const int cost = cost_of(it);
        last = blockIdx.x + 1;
        for (long long x; last + 1 < blocks && (x = total * (last + 1) / blocks - sh.base) < cost && cost - x >= TILE_CUT;) last++;
      }
      cuts[blockIdx.x] = last < 0 ? AttnCut{-1, 0, 0, 0, 0, 0, {0, 0}}
                                  : AttnCut{last, it.t0, it.n, (sh.item[1] % c.n_kv) * c.group, it.tok * c.group, tpt * c.group, {0, 0}};
    }
  }

  // The block's n-th item and its share of the key tiles: [from, n0) for query
  // tile 0, [from, n1) for tile 1.  False past the end.
  auto get_item = [&](int n, TileItem &it) {
    int i, from = 0, off1 = 0;
    if (deal) {
      i = dealt(n, blockIdx.x);
      if (i >= items) return false;
    } else {
      i = sh.item[0] + n;
      if (n == 0) from = sh.off[0];
      if (i >= sh.item[1]) off1 = sh.off[1];
      if (i > sh.item[1] || (i == sh.item[1] && off1 == 0)) return false;
    }
    const int p = (int)((unsigned)i / (unsigned)c.n_kv);
    get_pair(!deal ? p : known ? sh.order[p] : pairs - 1 - p, it);
    it.h = i - p * c.n_kv;
    const int all = max(it.n0, it.n1), to = off1 > 0 ? tiles_at(it, off1) : all;
    if (from > 0) from = tiles_at(it, from);
    it.from = from;
    it.whole = from == 0 && to == all;
    it.n0 = max(min(to, it.n0), from);
    it.n1 = max(min(to, it.n1), from);
    return true;
  };
  // Bounded wait of a whole warp; false: it, or another role's, ran out.
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    const uint32_t at = smem_u32(bar);
    bool ok = true;
    if (!mbar_tries(at, parity)) ok = tile_wait_long(at, parity, &sy.abort, c.status);
    __syncwarp();
    return ok;
  };

  if (warp >= 8) {
    regs_give<tile_regs_other<HD>()>();
    if (warp == 8) {
    // ------------------------------------------------------------- loads ---
    int bad = 0;
    uint32_t fill = 0, n_items = 0;        // ring fills issued; items begun
    bool ok = true;
#pragma unroll 1
    for (int i = 0; ok; i++) {
      TileItem it;
      if (!get_item(i, it)) break;
      const int to = max(it.n0, it.n1);
      if (to == it.from) continue;
      auto load_q = [&]() {
        if (!__all_sync(0xffffffffu, wait(&sy.q_empty, (n_items & 1) ^ 1))) return false;
        if (lane == 0) {
          const int rows = tpt * c.group, two = it.tok1 > 0;
          mbar_arrive_expect_tx(&sy.q_full, (uint32_t)(rows * 128 * (HD / 64) * (1 + two)));
          for (int t = 0; t <= two; t++)
            for (int x = 0; x < HD / 64; x++)
              tma_load_4d(s_q + t * Q_B + x * HALF_B, &maps.q, x * 64, it.h * c.group, it.t0 + it.tok + t * tpt, 0, &sy.q_full);
        }
        n_items++;
        return true;
      };
      // K (kv = 0) or V of key tile j into the ring's next place
      auto load = [&](int kv, int j) {
        const int kb = it.k0 + j * TILE_N;
        // this lane's box of the key tile: positions [pos, pos + box), 64 dims
        const int boxes = PAGED ? TILE_N / box : 1, bi = lane / (HD / 64), x = lane % (HD / 64);
        const int pos = kb + bi * box;
        const bool mine = bi < boxes && pos < it.high && pos + box > it.low;
        int pg = 0, off = 0;
        if (PAGED && mine) {
          const int e = pos / c.page;
          off = pos - e * c.page;
          pg = c.table[it.r * c.table_stride + e];
          if (pg < 0 || pg >= c.n_pages) { pg = c.n_pages; bad |= QTB_PS_PAGE; }   // past the last page: reads zeros
        }
        const int count = __popc(__ballot_sync(0xffffffffu, mine));
        const int st = (int)(fill % STAGES);
        if (!__all_sync(0xffffffffu, wait(&sy.kv_empty[st], ((fill / STAGES) & 1) ^ 1))) return false;
        if (lane == 0) mbar_arrive_expect_tx(&sy.kv_full[st], (uint32_t)(count * box * 128));
        __syncwarp();
        if (mine) {
          unsigned char *dst = s_kv + st * KV_B + x * HALF_B + bi * box * 128;
          const CUtensorMap *map = kv ? &maps.v : &maps.k;
          if (PAGED) tma_load_4d(dst, map, x * 64, off, it.h, pg, &sy.kv_full[st]);
          else tma_load_4d(dst, map, x * 64, it.t0 + pos, it.h, 0, &sy.kv_full[st]);
        }
        fill++;
        return true;
      };
      // in the order in which the MMA warp needs them: K of the first step(s), then V
      // of a step and K of the next of the same tile.  The queries' buffer may still
      // serve the item before: its keys go first.
      const int ahead = it.twin ? 2 : 1;
      ok = load(0, it.from) && load_q();
      if (ok && it.twin && it.from + 1 < to) ok = load(0, it.from + 1);
#pragma unroll 1
      for (int j = it.from; j < to && ok; j++) {
        ok = load(1, j);
        if (ok && j + ahead < to) ok = load(0, j + ahead);
      }
    }
    // copies in flight land before the block leaves
    for (uint32_t f = fill > STAGES ? fill - STAGES : 0; f < fill; f++)
      mbar_wait(&sy.kv_full[f % STAGES], (f / STAGES) & 1, TILE_WAIT);
    if (n_items) mbar_wait(&sy.q_full, (n_items - 1) & 1, TILE_WAIT);
    raise_status(c.status, bad);
    } else if (warp == 9) {
    // --------------------------------------------------------------- MMA ---
    const uint32_t ab = F16 ? 0u : 1u;
    const uint32_t idesc_s = umma_idesc(1u, ab, TILE_N), idesc_o = umma_idesc(1u, ab, HD) | (1u << 16);   // B as [K][N]
    uint32_t fill = 0, n_items = 0;
    uint32_t p_n = 0, o_n = 0;             // bit t: parity of the P hand-overs, of the finished outputs of tile t
    bool issued = false;
    // descriptors of the first tile and stage: others are an address (in 16 bytes) further on
    const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), k_desc = umma_desc_sw128(smem_u32(s_kv));
    const uint64_t v_desc = umma_desc_mn128(smem_u32(s_kv), HALF_B);
#pragma unroll 1
    for (int i = 0;; i++) {
      TileItem it;
      if (!get_item(i, it)) break;
      const int to = max(it.n0, it.n1);
      if (to == it.from) continue;
      wait(&sy.q_full, n_items & 1);
      n_items++;
      auto scores = [&](int t, int st) {
        const uint64_t q = q_desc + (uint32_t)(it.twin ? 0 : t * (Q_B >> 4)), k = k_desc + (uint32_t)(st * (KV_B >> 4));
        const uint32_t d = tmem + S_COL + t * 128;
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ks++) {
            const uint32_t o = ((ks >> 2) * HALF_B + (ks & 3) * 32) >> 4;
            umma_bf16(d, q + o, k + o, idesc_s, ks != 0);
          }
          umma_commit(&sy.s_full[t]);
        }
        __syncwarp();
      };
      // O += P V of key tile in stage sv for tile t, P's second half when it is there;
      // its K follows in stage sk where there is one
      auto product = [&](int t, int sv, bool first, bool last) {
        const uint64_t v = v_desc + (uint32_t)(sv * (KV_B >> 4));
        const uint32_t d = tmem + O_COL + t * HD, p = tmem + S_COL + t * 128;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < TILE_N / 32; ks++) umma_ts(d, p + ks * 8, v + ks * (2048 >> 4), idesc_o, !first || ks > 0);
        }
        __syncwarp();
        wait(&sy.p_full[t][1], (p_n >> t) & 1);
        p_n ^= 1u << t;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int ks = TILE_N / 32; ks < TILE_N / 16; ks++) umma_ts(d, p + ks * 8, v + ks * (2048 >> 4), idesc_o, 1);
          if (last) umma_commit(&sy.o_full[t]);
        }
        __syncwarp();
        if (last) o_n ^= 1u << t;
      };
      // The first half of P of tile t, and with it V and the next K, the fills f and
      // f + 1 (lanes wait for one each: the waits' latencies would add up).
      auto inputs = [&](int t, uint32_t f, bool more, bool first) {
        uint64_t *bar = &sy.p_full[t][0];
        uint32_t par = (p_n >> t) & 1;
        if (lane == 1) { bar = &sy.kv_full[f % STAGES]; par = (f / STAGES) & 1; }
        if (lane == 2 && more) { bar = &sy.kv_full[(f + 1) % STAGES]; par = ((f + 1) / STAGES) & 1; }
        if (lane == 3 && first) { bar = &sy.o_empty[t]; par = ((o_n >> t) & 1) ^ 1; }
        wait(bar, par);
      };
      issued = true;
      if (it.twin) {
#pragma unroll 1
        for (int t = 0; t < min(2, to - it.from); t++) {
          const int st = (int)(fill % STAGES);
          wait(&sy.kv_full[st], (fill / STAGES) & 1);
          scores(t, st);
          if (elect_one()) {
            umma_commit(&sy.kv_empty[st]);
            if (t == to - it.from - 1) umma_commit(&sy.q_empty);
          }
          __syncwarp();
          fill++;
        }
#pragma unroll 1
        for (int j = it.from; j < to; j++) {
          const int t = (j - it.from) & 1, sv = (int)(fill % STAGES), sk = (int)((fill + 1) % STAGES);
          const bool more = j + 2 < to, first = j < it.from + 2;
          inputs(t, fill, more, first);
          product(t, sv, first, !more);
          if (more) scores(t, sk);
          if (elect_one()) {
            umma_commit(&sy.kv_empty[sv]);
            if (more) umma_commit(&sy.kv_empty[sk]);
            if (j + 3 == to) umma_commit(&sy.q_empty);
          }
          __syncwarp();
          fill += more ? 2 : 1;
        }
        continue;
      }
      int st = (int)(fill % STAGES);
      wait(&sy.kv_full[st], (fill / STAGES) & 1);
      if (it.n0 > it.from) scores(0, st);
      if (it.n1 > it.from) scores(1, st);
      if (elect_one()) {
        umma_commit(&sy.kv_empty[st]);
        if (to == it.from + 1) umma_commit(&sy.q_empty);
      }
      __syncwarp();
      fill++;
#pragma unroll 1
      for (int j = it.from; j < to; j++) {
        const int sv = (int)(fill % STAGES), sk = (int)((fill + 1) % STAGES);
        const bool more = j + 1 < to;
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const int n = t ? it.n1 : it.n0;
          if (j >= n) continue;
          inputs(t, fill, more, j == it.from);
          product(t, sv, j == it.from, j == n - 1);
          if (j + 1 < n) scores(t, sk);
        }
        if (elect_one()) {
          umma_commit(&sy.kv_empty[sv]);
          if (more) umma_commit(&sy.kv_empty[sk]);
          if (j + 2 == to) umma_commit(&sy.q_empty);
        }
        __syncwarp();
        fill += more ? 2 : 1;
      }
    }
    if (issued) {                          // nothing reads shared or tensor memory any more
      if (elect_one()) umma_commit(&sy.drain);
      __syncwarp();
      mbar_wait(&sy.drain, 0, TILE_WAIT);
    }
    }
  } else {
    regs_take<tile_regs_softmax<HD>()>();
    // ----------------------------------------------------------- softmax ---
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + S_COL + t * 128 + lanes, o_at = tmem + O_COL + t * HD + lanes;
    uint32_t fill = 0, s_n = 0, o_n = 0;
#pragma unroll 1
    for (int i = 0;; i++) {
      TileItem it;
      if (!get_item(i, it)) break;
      const int to = max(it.n0, it.n1), n = t ? it.n1 : it.n0, n_tok = t && !it.twin ? it.tok1 : it.tok0;
      const int tok = it.tok + (it.twin ? 0 : t * tpt), step = it.twin ? 2 : 1, begin = it.from + (it.twin ? t : 0);
      const int tt = row / c.group;
      const int pos = it.first + tok + tt;                        // this row's position
      const int tk = tt < n_tok ? it.t0 + tok + tt : -1;          // its packed token (-1: no row)
      const int head = it.h * c.group + row - tt * c.group;
      // key tiles [clear_a, clear_b) are seen whole by every row of the tile
      const int pos_a = pos - tt, pos_b = pos_a + n_tok - 1;
      const int all_last = min(c.causal ? pos_a : it.end - 1, it.end - 1);
      const int clear_a = c.window > 0 ? (max(pos_b - c.window + 1, 0) - it.k0 + TILE_N - 1) / TILE_N : 0;
      const int clear_b = all_last < it.k0 ? 0 : (all_last + 1 - it.k0) / TILE_N;
      // A row of no token (the next request's queries, or old ones) starts from a
      // maximum that no score passes: the warp renews m for its own rows alone, so
      // that a request's results do not depend on what is beside it.
      float m = tk >= 0 ? -INFINITY : INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = begin; j < n; j += step) {
        wait(&sy.s_full[t], s_n & 1);
        s_n++;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int x = 0; x < 4; x++) tmem_ld32_async(s_at + 32 * x, s + 32 * x);
        tmem_ld_wait();
        const bool masked = j < clear_a || j >= clear_b;
        if (masked) {
          const int kb = it.k0 + j * TILE_N;
          // this row sees keys a .. b of the tile
          const int a = max((c.window > 0 ? max(pos - c.window + 1, 0) : 0) - kb, 0);
          const int b = min(c.causal ? pos : it.end - 1, it.end - 1) - kb;
#pragma unroll
          for (int y = 0; y < 4; y++) {
            const int u = min(max(a - 32 * y, 0), 32), w = min(max(b + 1 - 32 * y, 0), 32);   // keys u .. w - 1 of 32
            const uint32_t seen = (uint32_t)((1ull << w) - 1) & ~(uint32_t)((1ull << u) - 1);
#pragma unroll
            for (int x = 0; x < 32; x++) s[32 * y + x] = seen & (1u << x) ? s[32 * y + x] : -INFINITY;
          }
          if (kb < it.low || kb + TILE_N > it.high) {
            // keys that no row sees: their V may be anything, and 0 * NaN is NaN
            const int v_j = j - it.from;   // V's place among the item's fills
            const uint32_t f = fill + (it.twin ? 2 + v_j + min(v_j, to - it.from - 2) : 2 * v_j + 1);
            unsigned char *v = s_kv + (f % STAGES) * KV_B;
            wait(&sy.kv_full[f % STAGES], (f / STAGES) & 1);
            if (kb + row < it.low || kb + row >= it.high) {
#pragma unroll 1
              for (int y = 0; y < 8 * (HD / 64); y++)
                *reinterpret_cast<uint4 *>(v + (y >> 3) * HALF_B + row * 128 + (y & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        auto maximum = [&]() {
          float mx[4];
#pragma unroll
          for (int x = 0; x < 4; x++) mx[x] = max3(s[x], s[x + 4], s[x + 8]);
#pragma unroll
          for (int x = 12; x + 8 <= 128; x += 8)
#pragma unroll
            for (int y = 0; y < 4; y++) mx[y] = max3(mx[y], s[x + y], s[x + 4 + y]);
#pragma unroll
          for (int y = 0; y < 4; y++) mx[y] = fmaxf(mx[y], s[124 + y]);
          return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c.scale_log2;
        };
        const uint64_t scale2 = f2(c.scale_log2, c.scale_log2);
        uint64_t sum[2];
        // Probabilities of keys 32 part .. 32 part + 31 to tensor memory, rounded to
        // the tensors' type for the product with V, as large as the result's own
        // rounding; the sum is of the unrounded ones.
        auto probabilities = [&](int part) {
          const float base = m == -INFINITY ? 0.f : m;
          const uint64_t base2 = f2(-base, -base);
          uint32_t p[16];
#pragma unroll
          for (int x = 0; x < 16; x++) {
            float a, b;
            f2_get(fma2(f2(s[32 * part + 2 * x], s[32 * part + 2 * x + 1]), scale2, base2), a, b);
            a = exp2_approx(a);
            b = exp2_approx(b);
            sum[x & 1] = add2(sum[x & 1], f2(a, b));
            p[x] = pack2<F16>(a, b);
          }
          tmem_st16(s_at + 16 * part, p);
        };
        auto hand_over = [&](int part) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sy.p_full[t][part]);
        };
        // Past the first tile m rarely moves: the probabilities start from the old
        // one while the maximum is taken beside them, and are made anew where a row
        // has outgrown it.
        bool anew = j == begin;
        if (!anew) {
          sum[0] = sum[1] = 0;
#pragma unroll
          for (int part = 0; part < 2; part++) probabilities(part);
          anew = __any_sync(0xffffffffu, maximum() > m + 8.f);
        }
        if (anew) {
          const float top = maximum();
          if (__any_sync(0xffffffffu, top > m + 8.f)) {
            const float m2 = fmaxf(m, top), f = m2 == -INFINITY ? 1.f : exp2_approx(m - m2);
            m = m2;
            l *= f;
            if (j > begin) {
#pragma unroll 1
              for (int x = 0; x < HD / 8; x++) {
                float o[8];
                uint32_t w[8];
                tmem_ld8_async(o_at + 8 * x, o);
                tmem_ld_wait();
#pragma unroll
                for (int y = 0; y < 8; y++) w[y] = __float_as_uint(o[y] * f);
                tmem_st8(o_at + 8 * x, w);
              }
            }
          }
          sum[0] = sum[1] = 0;
#pragma unroll
          for (int part = 0; part < 2; part++) probabilities(part);
        }
        hand_over(0);
#pragma unroll
        for (int part = 2; part < 4; part++) probabilities(part);
        hand_over(1);
        float la, lb;
        f2_get(add2(sum[0], sum[1]), la, lb);
        l += la + lb;
      }
      fill += 2 * (to - it.from);
      const bool some = n > begin;
      if (some) {
        wait(&sy.o_full[t], o_n & 1);
        o_n++;
        tc_fence_after();
      }
      // A thread has a row, so that its 16-byte stores would each touch a line of
      // their own: four neighbours turn their 4 x 4 units first, and a store
      // instruction writes 64 bytes of each of 8 rows.
      auto turn = [&](uint32_t (&w)[4][4]) {
#pragma unroll
        for (int bit = 1; bit <= 2; bit <<= 1)
#pragma unroll
          for (int y = 0; y < 4; y++) {
            if (y & bit) continue;
#pragma unroll
            for (int z = 0; z < 4; z++) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & bit ? w[y][z] : w[y | bit][z], bit);
              if (lane & bit) w[y][z] = got;
              else w[y | bit][z] = got;
            }
          }
      };
      // A twin item's second state reaches the first one's threads: they are in the
      // same lanes of tensor memory.
      float f0 = 1.f, f1 = 0.f;
      if (it.twin) {
        if (t == 1) {
          sh.ml[row] = make_float2(m, l);
          tc_fence_before();
        }
        bar_sync_n(1, 256);
        if (t == 0) {
          tc_fence_after();
          const float2 z = sh.ml[row];
          const float m2 = fmaxf(m, z.x), base = m2 == -INFINITY ? 0.f : m2;
          f0 = exp2_approx(m - base);
          f1 = exp2_approx(z.x - base);
          m = m2;
          l = l * f0 + z.y * f1;
        }
      }
      const bool both = it.twin && it.from + 1 < n;
      if (it.twin && t == 1) {
        // nothing to write: tile 0's warps have both states
        if (!it.whole) {
          float *part = parts + ((long long)(2 * blockIdx.x + (it.from == 0 ? 1 : 0)) * 2 + 1) * tile_part_floats<HD>();
          *reinterpret_cast<float2 *>(part + TILE_M * HD + 2 * row) = make_float2(-INFINITY, 0.f);
        }
      } else if (it.whole) {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;   // no visible key: zeros
        const long long at = tk >= 0 ? (long long)tk * c.o_st + head * c.o_sh : -1;
        long long rows[4];
#pragma unroll
        for (int y = 0; y < 4; y++) rows[y] = __shfl_sync(0xffffffffu, at, (lane & ~3) + y);
#pragma unroll 1
        for (int x = 0; x < HD / 32; x++) {
          float o[32];
          if (some) {
            tmem_ld32_async(o_at + 32 * x, o);
            tmem_ld_wait();
          }
          if (both) {
            float z[32];
            tmem_ld32_async(o_at + HD + 32 * x, z);
            tmem_ld_wait();
#pragma unroll
            for (int y = 0; y < 32; y++) o[y] = o[y] * f0 + z[y] * f1;
          }
          uint32_t w[4][4];
#pragma unroll
          for (int y = 0; y < 4; y++)
#pragma unroll
            for (int z = 0; z < 4; z++)
              w[y][z] = some ? pack2<F16>(o[8 * y + 2 * z] * inv, o[8 * y + 2 * z + 1] * inv) : 0u;
          turn(w);
#pragma unroll
          for (int y = 0; y < 4; y++)
            if (rows[y] >= 0)
              *reinterpret_cast<uint4 *>(c.out + rows[y] + 32 * x + 8 * (lane & 3)) = make_uint4(w[y][0], w[y][1], w[y][2], w[y][3]);
          __syncwarp();
        }
        if (tk >= 0 && c.lse) c.lse[(long long)tk * c.n_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        float *part = parts + ((long long)(2 * blockIdx.x + (it.from == 0 ? 1 : 0)) * 2 + t) * tile_part_floats<HD>();
        if (some) {
#pragma unroll 1
          for (int x = 0; x < HD / 16; x++) {
            uint32_t w[4][4];
            tmem_ld16_async(o_at + 16 * x, reinterpret_cast<float *>(w));
            tmem_ld_wait();
            if (both) {
              float z[16];
              tmem_ld16_async(o_at + HD + 16 * x, z);
              tmem_ld_wait();
#pragma unroll
              for (int y = 0; y < 16; y++) w[y >> 2][y & 3] = __float_as_uint(__uint_as_float(w[y >> 2][y & 3]) * f0 + z[y] * f1);
            }
            turn(w);
#pragma unroll
            for (int y = 0; y < 4; y++)
              *reinterpret_cast<uint4 *>(part + ((row & ~3) + y) * HD + 16 * x + 4 * (lane & 3)) = make_uint4(w[y][0], w[y][1], w[y][2], w[y][3]);
            __syncwarp();
          }
        }
        *reinterpret_cast<float2 *>(part + TILE_M * HD + 2 * row) = make_float2(m, l);
      }
      tc_fence_before();
      if (it.twin) bar_sync_n(2, 256);     // both states have been read
      if (some) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sy.o_empty[t]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ host ---
// Whether the tile kernel can have the call: it takes the maximum of the scores
// before they are scaled.
static inline bool tile_form(const AttnCall &c) { return c.scale_log2 > 0.f; }

// The key box: as many of a page's positions as divide both page and tile.
static inline int tile_box(bool paged, int page) {
  int b = TILE_N;
  while (paged && page % b) b >>= 1;
  return b;
}

static inline bool tile_maps(const AttnCall &c, bool paged, bool f16, int hd, TensorMapFn fn, TileMaps &m) {
  const long long qe[4] = {hd, c.n_heads, c.n_tokens, 1}, qs[4] = {1, c.q_sh, c.q_st, 0};
  const int qb[4] = {64, c.group, TILE_M / c.group, 1}, kb[4] = {64, tile_box(paged, c.page), 1, 1};
  const long long ke[4] = {hd, paged ? c.page : c.n_tokens, c.n_kv, paged ? c.n_pages : 1};
  auto keys = [&](CUtensorMap *out, const uint16_t *base, const long long *st) {
    const long long str[4] = {1, paged ? st[2] : st[0], st[1], paged ? st[0] : 0};
    return tensor_map(fn, out, base, f16, 4, ke, str, kb);
  };
  return tensor_map(fn, &m.q, c.q, f16, 4, qe, qs, qb) && keys(&m.k, c.k, c.k_st) && keys(&m.v, c.v, c.v_st);
}

static inline size_t tile_workspace(int hd, int sms) {
  return (size_t)sms * (sizeof(AttnCut) + 2 * 2 * (size_t)(hd == 128 ? tile_part_floats<128>() : tile_part_floats<64>()) * 4);
}

template <int HD, bool F16, bool PAGED>
static cudaError_t tile_run(bool prepare, const AttnCall *c, const TileMaps *m, int sms, void *ws, cudaStream_t st) {
  if (prepare)
    return cudaFuncSetAttribute(tile_kernel<HD, F16, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, tile_smem<HD>());
  const int tpt = TILE_M / c->group, box = tile_box(PAGED, c->page);
  if (!ws) {                               // whole items only
    const long long items = ((c->n_tokens + 2 * tpt - 1) / (2 * tpt) + (c->n_req > 1 ? c->n_req : 0)) * (long long)c->n_kv;   // at most
    tile_kernel<HD, F16, PAGED><<<(int)(items < sms ? items : sms), TILE_THREADS, tile_smem<HD>(), st>>>(*c, *m, tpt, box, nullptr, nullptr);
    return cudaGetLastError();
  }
  AttnCut *cuts = static_cast<AttnCut *>(ws);
  float *parts = reinterpret_cast<float *>(cuts + sms);
  tile_kernel<HD, F16, PAGED><<<sms, TILE_THREADS, tile_smem<HD>(), st>>>(*c, *m, tpt, box, parts, cuts);
  if (cudaError_t e = cudaGetLastError()) return e;
  return launch_early(join_kernel<HD, F16, TILE_M, 2, 1, 2>, dim3(sms, 2 * TILE_M / (2 * JOIN_WARPS)), 32 * JOIN_WARPS, 0, st, *c,
                      (const float *)parts, (const AttnCut *)cuts);
}
static inline cudaError_t tile_any(bool prepare, int which, const AttnCall *c, const TileMaps *m, int sms, void *ws,
                                   cudaStream_t st) {
  switch (which) {
    case 0: return tile_run<64, false, false>(prepare, c, m, sms, ws, st);
    case 1: return tile_run<64, false, true>(prepare, c, m, sms, ws, st);
    case 2: return tile_run<64, true, false>(prepare, c, m, sms, ws, st);
    case 3: return tile_run<64, true, true>(prepare, c, m, sms, ws, st);
    case 4: return tile_run<128, false, false>(prepare, c, m, sms, ws, st);
    case 5: return tile_run<128, false, true>(prepare, c, m, sms, ws, st);
    case 6: return tile_run<128, true, false>(prepare, c, m, sms, ws, st);
    default: return tile_run<128, true, true>(prepare, c, m, sms, ws, st);
  }
}
static inline cudaError_t tile_prepare() {
  for (int i = 0; i < 8; i++)
    if (cudaError_t e = tile_any(true, i, nullptr, nullptr, 0, nullptr, nullptr)) return e;
  return cudaSuccess;
}
// Without a workspace no item is cut.
static inline cudaError_t tile_launch(const AttnCall &c, bool paged, bool f16, int hd, const TileMaps &m, int sms, void *ws,
                                       cudaStream_t st) {
  return tile_any(false, (hd == 128 ? 4 : 0) + (f16 ? 2 : 0) + (paged ? 1 : 0), &c, &m, sms, ws, st);
}

}  // namespace qtb
