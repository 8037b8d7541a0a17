// Causal attention of new tokens over the paged KV cache (sm_100a).
//
// Per request b with n new tokens (its rows of q) and L keys, token i and
// q-head hq:  o = softmax_j(q . k_j * sm_scale | j <= L - n + i) . v_j.
//
// A unit is (request, kv-head, query tile).  The G q-heads of a kv-head share
// its keys, so a tile's rows are tokens x G heads (row = token * G + head) and
// one tcgen05 MMA serves them all; a single token's G rows go through the same
// tile, whose spare rows cost no memory traffic.  D <= 128: a CTA and 128 rows.
// D = 256: two CTAs (cta_group::2) and 256 rows, each CTA holding half of every
// K / V tile: a CTA alone has room for Q (64 KB) and one 128 KB tile of 128 keys
// in its shared memory, not for the next one, and with 64 keys its S MMAs run at
// half rate (72 cycles for 128 x 64 x 16, bound by reading A).  Per tile of 128
// keys, one pass with a running maximum and sum:
//   K, V  by slot, 16 keys at a time, into separate rings of stages by one
//         producer warp each: where the 16 slots are consecutive (pages of 16 and
//         more) TMA boxes of 8 (K) or 16 (V) cache rows by 64-dim chunks, else
//         16-byte cp.async row by row (a gather of four rows per TMA copy took
//         39 ns a copy, 5 us per 64 KB)
//   S     = Q K^T    kind::f16, fp32 in TMEM; Q from shared memory, where one TMA
//         box of tokens x G heads per 64 dims puts it while the unit before ends
//   P     = 2^(S sm_scale log2e - m), two threads per row; the reference m moves
//         (and O is rescaled in TMEM) only when the maximum grows by more than
//         8, so P <= 2^8; rounded to the 16-bit type over its own S (the second
//         product's operand has V's type), summed unrounded
//   O    += P V      P from TMEM, V as an MN-major operand
// S / P are double-buffered and the S MMA runs a tile ahead of the P V MMA.  S of
// tile t+2 waits for P V of tile t, so a tile's softmax latency counts twice: a
// warpgroup per tile, in turn, took 3000 cycles a tile, both on one tile 1600.
//
// Work is split by keys, not by unit: unit costs (keys + a fixed part) are laid
// out on one line, and worker c (a CTA, a pair) takes the c-th share of it,
// whatever units that crosses.  One long prompt, many ragged requests and one
// long decode all fill the GPU evenly, from lengths that only the device knows.
// A unit cut by a share's border leaves partials (O, m, l) that a second kernel
// merges.
//
// Tiles past a row's last key hold the masked keys' values: their P is 0, but 0
// times NaN or infinity is not.  In those tiles alone the softmax threads zero
// V's rows past the request's end and its non-finite elements before the P V
// product reads them; the epilogue adds such an element back to the rows that
// do see its key.
//
// Measured (bf16, 16 q-heads, 4 kv-heads of 256), in captured graphs of a few ms and,
// in brackets, call by call on changing inputs: a prompt of 8192 tokens 398 to 450 us,
// 1.2 to 1.4 PFLOP/s (468 us, 1.2), bound by the tensor cores under the power cap; 64
// single tokens on up to 4097 keys 122 us, 5.4 TB/s (145 us, 4.6), bound by the stages'
// turnover (two of K and two of V, held by MMAs of 256 rows); 512 tokens on 33280 keys in
// single-token pages 260 us, 1.1 PFLOP/s (307 us, 0.90), bound by the row copies' issue
// and latency (L2 18 % busy; in pages of 16 a shorter such chunk takes 0.8 of the time);
// one token on 701 keys 13.5 us (15.1).
//
// Every wait is bounded (~1 s); on timeout the CTA raises DFT_DEV_TIMEOUT (its
// pair gives up with it), waits (bounded) for its MMAs and for every copy that was
// issued, frees TMEM and exits.
#include "dft_common.cuh"
#include "dft_gdn_tile.cuh"
#include "dft_tc.cuh"

#include <cstring>
#include <type_traits>

using namespace dft;
using namespace dft::tc;

namespace {

constexpr int kMaxB = 1024;
constexpr int kMaxKeys = 1 << 25; // of a request: 2^18 tiles of up to 4000 cycles, half of what a wait is given
constexpr int kRows = 128;        // query rows of a CTA
constexpr int kSoftmax = 256;     // two threads per query row, in warps w and w + 4
constexpr int kCtlWarp = 8, kProdWarp0 = 9, kPlanWarp = 11;  // a producer warp for K, one for V
constexpr int kThreads = 384;     // twelve warps leave 168 registers a thread; a row of 64 scores takes most of them
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxStages = 4, kRing = 4;
// A unit's fixed cost in keys (query load, first tile's latency, output).  D = 256:
// with 256 / 384 / 512 / 768 a prompt of 8192 tokens took 429 / 414 / 415 / 422 us and
// 8 ragged single tokens on 1000 keys 17.7 / 18.5 / 18.5 / 19.8; D <= 128, whose tiles
// are as long and whose output is half: 12 ragged prompts of D = 128 61 / 65 / 65 / 69
// us, 16 single tokens of D = 64 on 2000 keys 23.6 / 23.7 / 24.9 / 26.0.
constexpr int unit_keys(int D) { return D == 256 ? 512 : 256; }
// The least share of a worker, under which a cut costs more than it spreads:
// with 128 / 256 / 384 / 512 a single token on 701 keys took 12.9 / 13.3 / 14.7 / 15.5
// us and 64 tokens on 1000 keys, whose partials are 64 KB each, 32 with 128, 28 with 256.
constexpr int kMinShare = 256;

constexpr int KT = 128;           // keys per tile
constexpr int NB = 2;             // S / P buffers
constexpr float kLog2e = 1.4426950408889634f;
template <int N>
using Int = std::integral_constant<int, N>;

template <int D>
struct Cfg {
  static constexpr bool kPair = D == 256;
  static constexpr int CG = kPair ? 2 : 1;                    // CTAs of a worker
  static constexpr int KS = kPair ? 2 : D == 128 ? 3 : 4, VS = D == 64 ? 4 : 2;  // stages of K and of V
  static constexpr int KR = KT / CG, KC = D / 64;             // K rows and 64-dim chunks in this CTA
  static constexpr int VC = D / 64 / CG;                      // V chunks in this CTA (all KT rows)
  static constexpr uint32_t kKBytes = KR * KC * 128, kVBytes = KT * VC * 128;
  static constexpr uint32_t kQBytes = kRows * D * 2;
  static constexpr int kSlotRows = kRows * CG;                // of a partial
  static constexpr uint32_t OFF_V = KS * kKBytes, OFF_Q = OFF_V + VS * kVBytes;
  static constexpr uint32_t OFF_SMALL = OFF_Q + kQBytes;
  static constexpr uint32_t COL_O = 0, COL_S = D;  // S / P buffer b at COL_S + KT b
  static_assert(COL_S + NB * KT <= kTmemCols, "TMEM");
};

// A worker's part of one unit: key tiles [t0, t1) of nt.  b < 0: there are no more.
struct Piece {
  int b, h, tok0, ntok;  // first token row of q, tokens
  int k0;                // its request's first entry in kv_indices
  int vis0, L;           // keys that the first token sees (may be negative), keys of the request
  int t0, t1;
  int slot;              // -1: the whole unit; 0 / 1: partial that continues / begins it
  bool last, once;       // the unit's last tiles; its keys are read by this tile alone
};

struct Small {
  uint64_t q_ready, q_empty;
  uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
  uint64_t k_copied[kMaxStages], v_copied[kMaxStages];  // rank 1 of a pair: its cp.async rows of the stage
  uint64_t s_full[NB], p_full[NB], pv_done[NB];
  uint64_t v_here[NB];      // rank 1 of a pair: [S buffer] the tile's V is in (its boxes complete on rank 0)
  uint64_t o_full, o_free, mma_done;
  uint64_t ring_full[kRing], ring_empty[kRing];
  uint32_t tmem_base;
  int abort;                // of both CTAs of a pair
  int sent[3], relayed[2];  // after the roles' end: tiles of K, of V and pieces' Q issued; tiles of K, V relayed
  int odd[8];               // [piece & 7] = piece + 1 when one of its masked tiles held a non-finite value
  float xmax[2][2][kRows];  // [tile parity][half][row] tile max exchange between a row's two threads
  float lsum[2][kRows];     // [half][row] final row sums
  int okx[2][2][4];         // [tile parity][half][row warp] wait outcomes, shared by a row's two warps
  int okr[2][2][4];         // the same for the rescale's wait
  int okt[2][2][4];         // [unit parity][half][row warp] whether the warp goes on to the next unit
  uint32_t pre[kMaxB + 1];  // cost of the requests before b
  int shift;                // costs on the line are in 2^shift keys
  int qo[kMaxB + 1], kv[kMaxB + 1];
  Piece ring[kRing];           // the worker's pieces as they come, from the plan warp
  int4 slots[2][32];
  int k_mixed[kMaxStages], v_mixed[kMaxStages];  // [stage]: the CTA's part holds rows copied by cp.async
};

struct Params {
  dft_chunk_attn_args a;
  int unit_keys;            // fixed cost of a unit
  int G, TC, TQ;            // q-heads per kv-head, tokens of a query tile per CTA and in all
  uint32_t inv_G;           // ceil(2^16 / G): row / G = row * inv_G >> 16 for rows below 256 and G up to 128
  // Partials: slot 2c continues a unit, 2c + 1 begins one.  O by 8 dims of all
  // rows, so that a warp, a row to a lane, stores 1 KB in one piece (by rows its
  // 32 pieces of 16 bytes took 16000 cycles for 128 rows of 256).
  float* ws_o;              // [2 workers][D / 8][rows][8]
  float* ws_ml;             // [2 workers][rows][2] partial (m, l)
  int4* ws_meta;            // [2 workers] (flags, first token row, tokens, kv-head); flags 1: used, 2: the unit's last
};

template <int D>
constexpr uint32_t smem_bytes() {
  static_assert(Cfg<D>::OFF_SMALL + sizeof(Small) + 1024 <= 232448, "shared memory");
  return Cfg<D>::OFF_SMALL + (uint32_t)sizeof(Small) + 1024;  // + alignment slack
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF>
__device__ __forceinline__ float unpack(uint16_t v) {
  return BF ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

template <bool PAIR>
__device__ __forceinline__ void set_abort(Small& sm, int rank, int32_t* status) {
  *reinterpret_cast<volatile int*>(&sm.abort) = 1;
  if (PAIR) st_cluster(map_rank(smem_u32(&sm.abort), rank ^ 1), 1);
  raise_status(status, DFT_DEV_TIMEOUT);
}

// Bounded wait that also gives up once another role has; the clock is read
// only when the first try fails.
__device__ __forceinline__ bool wait(uint64_t& bar, uint32_t parity, const volatile int* abort) {
  return mbar_try(smem_u32(&bar), parity) || mbar_wait_or_abort(smem_u32(&bar), parity, abort);
}
// Arrive, once per warp and after all of its lanes, on the barrier of the CTA
// that issues the MMAs.
template <bool PAIR>
__device__ __forceinline__ void warp_arrive(uint64_t& bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if (PAIR) mbar_arrive_cluster(map_rank(smem_u32(&bar), 0));
    else mbar_arrive(smem_u32(&bar));
  }
}

// -------------------------------------------------------------- schedule --
// Request b: n tokens in nt query tiles, L keys.  Tile i ends at token e =
// min((i + 1) TQ, n) and reads the keys its last token sees, clamp(L - n + e,
// 0, L); its cost is that + unit_keys, and the sum over the tiles before i is
// an arithmetic series.  Costs on the line are those sums over 2^shift, rounded
// down (a tile's own is the difference of two), so that the line fits 31 bits:
// with 64-bit divisions finding a first piece took 8000 cycles of fetching code.
struct Req {
  int n, L, nt;
};
__device__ __forceinline__ Req request(const Small& sm, int b, int TQ) {
  Req r;
  r.n = sm.qo[b + 1] - sm.qo[b];
  r.L = sm.kv[b + 1] - sm.kv[b];
  r.nt = (int)(((uint32_t)r.n + (uint32_t)TQ - 1) / (uint32_t)TQ);  // n + TQ may pass 2^31
  return r;
}
__device__ __forceinline__ uint64_t cost_before(const Req& r, int i, const Params& P, int shift) {
  uint64_t last = 0;
  if (i == r.nt && i > 0) {  // the last tile is the one that may be short
    last = (uint32_t)r.L + P.unit_keys;
    --i;
  }
  const int a = r.L - r.n;
  const uint32_t z = a < 0 ? min((uint32_t)i, (uint32_t)-a / (uint32_t)P.TQ) : 0u;  // tiles that see no key
  const uint64_t pairs = (uint64_t)(uint32_t)i * (uint32_t)(i + 1) - (uint64_t)z * (z + 1);
  const int64_t keys = (int64_t)(i - (int)z) * a + (int64_t)(pairs >> 1) * P.TQ;
  return (last + (uint64_t)(uint32_t)i * P.unit_keys + (uint64_t)keys) >> shift;
}

// The line: offsets to shared memory, and the cost of the requests before each
// (by one warp; lane i sums a run of requests).  Returns the line's length.
// Up to 2^8 every tile keeps a cost of its own; 2^39 keys are half a minute of
// work, and a longer line is refused.
constexpr int kMaxShift = 8;
static_assert(unit_keys(64) >> kMaxShift >= 1 && unit_keys(256) >> kMaxShift >= 1 && kMinShare >> kMaxShift >= 1, "costs");
__device__ __forceinline__ uint32_t plan_costs(Small& sm, const Params& P, int32_t* status) {
  const dft_chunk_attn_args& a = P.a;
  const int lane = threadIdx.x & 31, per = (a.B + 31) >> 5;
#pragma unroll 1
  for (int i = lane; i <= a.B; i += 32) {
    sm.qo[i] = a.qo_indptr[i];
    sm.kv[i] = a.kv_indptr[i];
  }
  __syncwarp();
  const int b0 = lane * per, b1 = min(a.B, b0 + per);
  bool bad = false;
  int shift = 0;
  uint64_t inc, sum, total;
#pragma unroll 1
  while (true) {
    sum = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      const int q0 = sm.qo[b], q1 = sm.qo[b + 1], k0 = sm.kv[b], k1 = sm.kv[b + 1];
      const bool ok = q0 >= 0 && q0 <= q1 && q1 <= a.T && k0 >= 0 && k0 <= k1 && k1 <= a.n_kv && k1 - k0 <= kMaxKeys;
      bad |= !ok;
      sm.pre[b] = (uint32_t)sum;  // so far from the lane's first
      if (ok && q1 > q0) {
        const Req r = request(sm, b, P.TQ);
        sum += a.Hkv * cost_before(r, r.nt, P, shift);
      }
    }
    inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint64_t o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    total = __shfl_sync(0xffffffffu, inc, 31);
    if (total >> 31 == 0) break;
    if (shift == kMaxShift) {
      bad = true;
      total = 0;
      break;
    }
    shift = min(kMaxShift, shift + 33 - __clzll((long long)total));
  }
  if (bad && blockIdx.x == 0) raise_status(status, DFT_DEV_BAD_INDEX);
#pragma unroll 1
  for (int b = b0; b < b1; ++b) sm.pre[b] += (uint32_t)(inc - sum);
  if (lane == 0) {
    sm.pre[a.B] = (uint32_t)total;
    sm.shift = shift;
  }
  __syncwarp();
  return (uint32_t)total;
}

// The next piece of the line from w, w < w1, that has something to do.
__device__ __forceinline__ bool next_piece(const Small& sm, const Params& P, uint32_t& w, uint32_t w1, Piece& p) {
#pragma unroll 1
  while (w < w1) {
    int lo = 0, hi = P.a.B;  // pre[lo] <= w < pre[hi]
#pragma unroll 1
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sm.pre[mid] <= w) lo = mid;
      else hi = mid;
    }
    const Req r = request(sm, lo, P.TQ);
    const uint32_t at = w - sm.pre[lo], per_head = (sm.pre[lo + 1] - sm.pre[lo]) / (uint32_t)P.a.Hkv;
    const uint32_t h = at / per_head, rest = at - h * per_head;
    // the tile: cost_before(i) <= rest < cost_before(i + 1)
    int i = 0;
    uint32_t c0 = 0, c1 = per_head;
#pragma unroll 1
    for (int top = r.nt; top - i > 1;) {
      const int mid = (i + top) >> 1;
      const uint32_t c = (uint32_t)cost_before(r, mid, P, sm.shift);
      if (c <= rest) {
        i = mid;
        c0 = c;
      } else {
        top = mid;
        c1 = c;
      }
    }
    const uint32_t x0 = rest - c0, x1 = min(c1 - c0, x0 + (w1 - w));
    const bool whole = x1 == c1 - c0;
    w += x1 - x0;
    const int keys = max(0, r.L - r.n + (int)min((int64_t)(i + 1) * P.TQ, (int64_t)r.n));
    const int nt = (keys + KT - 1) / KT;
    const auto tile = [&](uint32_t x) { return (int)min((uint64_t)nt, (((uint64_t)x << sm.shift) + KT / 2) / KT); };
    p.t0 = x0 == 0 ? 0 : tile(x0);
    p.t1 = whole ? nt : tile(x1);
    if (p.t0 == p.t1 && !(nt == 0 && x0 == 0)) continue;
    p.b = lo;
    p.h = (int)h;
    p.tok0 = sm.qo[lo] + i * P.TQ;
    p.ntok = min(P.TQ, r.n - i * P.TQ);
    p.k0 = sm.kv[lo];
    p.vis0 = r.L - r.n + i * P.TQ + 1;
    p.L = r.L;
    p.last = p.t1 == nt;
    p.slot = p.t0 == 0 ? (p.last ? -1 : 1) : 0;
    p.once = r.nt == 1;
    return true;
  }
  return false;
}

template <bool BF, int D>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap q1_map,
                      const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const __grid_constant__ Params P, int32_t* status) {
  using F = Cfg<D>;
  constexpr bool PAIR = F::kPair;
  constexpr int CG = F::CG;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Small& sm = *reinterpret_cast<Small*>(smem + F::OFF_SMALL);
  const volatile int* abort_flag = &sm.abort;
  const dft_chunk_attn_args& a = P.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t k_base = smem_u32(smem), v_base = k_base + F::OFF_V;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

  // the merge kernel's blocks may come up now; they wait for this grid to end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == kCtlWarp) {
    if (lane == 0) {
      mbar_init(smem_u32(&sm.q_ready), CG);
      mbar_init(smem_u32(&sm.q_empty), 1);
      for (int i = 0; i < kMaxStages; ++i) {
        // a warp's cp.async and an expect_tx; from rank 1 an expect_tx and, once its cp.async are in, an arrival
        mbar_init(smem_u32(&sm.k_copied[i]), 32);
        mbar_init(smem_u32(&sm.v_copied[i]), 32);
        mbar_init(smem_u32(&sm.k_full[i]), 32 + 1 + 2 * (CG - 1));
        mbar_init(smem_u32(&sm.k_empty[i]), 1);
        mbar_init(smem_u32(&sm.v_full[i]), 32 + 1 + 2 * (CG - 1));
        mbar_init(smem_u32(&sm.v_empty[i]), 1);
      }
      for (int i = 0; i < NB; ++i) {
        mbar_init(smem_u32(&sm.s_full[i]), 1);
        mbar_init(smem_u32(&sm.p_full[i]), kSoftmax / 32 * CG);
        mbar_init(smem_u32(&sm.pv_done[i]), 1);
        mbar_init(smem_u32(&sm.v_here[i]), 1);
      }
      mbar_init(smem_u32(&sm.o_full), 1);
      mbar_init(smem_u32(&sm.o_free), kSoftmax / 32 * CG);
      mbar_init(smem_u32(&sm.mma_done), 1);
      for (int i = 0; i < kRing; ++i) {
        mbar_init(smem_u32(&sm.ring_full[i]), 1);
        mbar_init(smem_u32(&sm.ring_empty[i]), kSoftmax / 32 + 3);  // the warps that take pieces
      }
      sm.abort = 0;
      for (int i = 0; i < 8; ++i) sm.odd[i] = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (PAIR) tmem_alloc_2(smem_u32(&sm.tmem_base), kTmemCols);
    else tmem_alloc(smem_u32(&sm.tmem_base), kTmemCols);
  }
  for (uint32_t i = tid * 16; i < F::kQBytes; i += kThreads * 16)
    *reinterpret_cast<uint4*>(smem + F::OFF_Q + i) = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_arrive();  // this CTA's barriers are up
  pdl_wait();  // inputs and workspace are the launches before's until here
  const uint32_t total = warp == kPlanWarp ? plan_costs(sm, P, status) : 0u;
  if (PAIR) cluster_wait();    // the other CTA's are too, before anything arrives on them
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  Piece p;

  // The pieces are worked out by one warp for all: at each role the search and
  // its 64-bit arithmetic were 144 KB of kernel, and every unit's change waited
  // 8 us for instructions.
  int taken = 0;
  const auto take = [&](Piece& x) {
    const int i = taken % kRing;
    if (!__all_sync(0xffffffffu, wait(sm.ring_full[i], (taken / kRing) & 1, abort_flag))) {
      x.b = -2;  // a wait gave up
      return false;
    }
    x = sm.ring[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sm.ring_empty[i]));
    ++taken;
    return x.b >= 0;
  };
  if (warp == kCtlWarp) {
    if (rank == 0) {
      // ---------------------------------------------------- control: MMAs
      const uint32_t lead = elect_lane();
      const auto commit = [&](uint64_t& bar) { mma_commit_lead<CG>(lead, smem_u32(&bar)); };
      // waits of the whole warp: one outcome for all lanes
      const auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
      constexpr uint32_t id_s = BF ? idesc_bf16(128 * CG, KT, false) : idesc_f16(128 * CG, KT, false);
      constexpr uint32_t id_o = BF ? idesc_bf16(128 * CG, D, true) : idesc_f16(128 * CG, D, true);
      const uint32_t q_base = k_base + F::OFF_Q;
      int g = 0, ui = 0;
      bool ok = true;
      while (ok && take(p)) {
        const int T = p.t1 - p.t0;
        if (T == 0) continue;
        ok = all(wait(sm.q_ready, ui & 1, abort_flag));
        for (int t = 0; ok && t <= T; ++t) {
          if (t < T) {
            const int gt = g + t, st = gt % F::KS, sb = gt % NB;
            bool got = wait(sm.k_full[st], (gt / F::KS) & 1, abort_flag);
            if (got && gt >= NB) got = wait(sm.pv_done[sb], (gt / NB - 1) & 1, abort_flag);  // P of tile gt - NB is read
            ok = all(got);
            if (!ok) break;
            tc_fence_after();
            if (sm.k_mixed[st]) fence_async_smem();  // cp.async (generic proxy) writes -> tensor-core reads
            const uint32_t kb = __shfl_sync(0xffffffffu, k_base + st * F::kKBytes, 0);
            const uint32_t ds = __shfl_sync(0xffffffffu, tmem + F::COL_S + KT * sb, 0);
            // K: 8-key groups KC KB apart, a group's 64-dim chunks 1 KB apart
            const uint64_t ad = sw128_desc(q_base), bd = sw128_desc(kb, 16, F::KC * 1024);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_ss<CG>(lead, ds, ad + ((k >> 2) * (kRows * 128) + (k & 3) * 32) / 16,
                         bd + ((k >> 2) * 1024 + (k & 3) * 32) / 16, id_s, k > 0);
            commit(sm.k_empty[st]);
            commit(sm.s_full[sb]);
            if (t == T - 1) commit(sm.q_empty);
          }
          if (t > 0) {
            const int gu = g + t - 1, st = gu % F::VS, pb = gu % NB;
            bool got = wait(sm.v_full[st], (gu / F::VS) & 1, abort_flag);
            if (PAIR && got && lead) mbar_arrive_cluster(map_rank(smem_u32(&sm.v_here[pb]), 1));
            // the first P V of a unit overwrites O: the previous unit's epilogue has read it
            if (got && t == 1 && ui > 0) got = wait(sm.o_free, (ui - 1) & 1, abort_flag);
            ok = all(got && wait(sm.p_full[pb], (gu / NB) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            if (sm.v_mixed[st]) fence_async_smem();
            const uint32_t vb = __shfl_sync(0xffffffffu, v_base + st * F::kVBytes, 0);
            const uint32_t ps = __shfl_sync(0xffffffffu, tmem + F::COL_S + KT * pb, 0);
            const uint32_t keep = __shfl_sync(0xffffffffu, t > 1 ? 1u : 0u, 0);
            // P: 64 keys in columns 0 to 31 of its buffer, 64 in 64 to 95.
            // V [keys x dims] is MN-major: of 16 keys, 64-dim chunks 2 KB apart, 8-key groups 1 KB apart
            const uint64_t bd = sw128_desc(vb, 2048, 1024);
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
              mma_ts<CG>(lead, tmem + F::COL_O, ps + 8 * k + (k < 4 ? 0 : 32), bd + k * F::VC * 2048 / 16, id_o, k > 0 ? 1u : keep);
            commit(sm.v_empty[st]);
            commit(sm.pv_done[pb]);
            if (t == T) commit(sm.o_full);
          }
        }
        g += T;
        ++ui;
      }
      ok = ok && p.b != -2;
      if (!ok && lane == 0 && !*abort_flag) set_abort<PAIR>(sm, rank, status);
      // every MMA issued above has retired before TMEM is freed
      commit(sm.mma_done);
    } else {
      // Rank 1 of a pair: its boxes complete on rank 0's barriers by themselves.
      // For the cp.async rows of each stage (none, maybe) this warp arrives there
      // once they are in.  K and V run apart, so it waits for neither alone; it
      // arrives for every tile, so a stage is not reused before and its parity
      // keeps its meaning.
      // It takes a piece only when it owes no arrival: piece n + 1 comes once the S
      // of piece n - 1 are done, and those need every K and V up to there.  What it
      // owes for pieces up to n needs nothing of n + 1 (producers, Q and MMAs of a
      // piece wait for earlier tiles alone), so the waits form no cycle; and no time
      // goes, since the last V of n is read before the first K of n + 1.
      int end = 0, next[2] = {0, 0};  // tiles known of, and the next of K and of V
      bool ok = true, more = true;
      long long t0 = clock64();
      while (ok && (more || next[0] < end || next[1] < end)) {
        if (more && next[0] == end && next[1] == end) {
          more = take(p);
          ok = p.b != -2;
          if (more) end += p.t1 - p.t0;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int n = v ? F::VS : F::KS, st = next[v] % n;
          if (next[v] >= end || !__all_sync(0xffffffffu, mbar_test(smem_u32(v ? &sm.v_copied[st] : &sm.k_copied[st]),
                                                                  (next[v] / n) & 1)))
            continue;
          if ((v ? sm.v_mixed : sm.k_mixed)[st]) fence_async_smem();
          if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(v ? &sm.v_full[st] : &sm.k_full[st]), 0));
          ++next[v];
          t0 = clock64();
        }
        ok = ok && __all_sync(0xffffffffu, !*abort_flag && clock64() - t0 < 2000000000ll);
      }
      if (lane == 0) {
        sm.relayed[0] = next[0];
        sm.relayed[1] = next[1];
      }
      if (!ok && lane == 0 && !*abort_flag) set_abort<PAIR>(sm, rank, status);
    }
    if (lane == 0 && !mbar_wait(smem_u32(&sm.mma_done), 0)) raise_status(status, DFT_DEV_TIMEOUT);
    __syncwarp();
  } else if (warp == kPlanWarp) {
    // ------------------------------------------ plan: the pieces, and their Q
    const uint32_t share = max((uint32_t)kMinShare >> sm.shift, (total + workers - 1) / workers);
    uint32_t w = (uint32_t)min((uint64_t)total, (uint64_t)share * worker);
    const uint32_t w1 = (uint32_t)min((uint64_t)total, (uint64_t)w + share);
    const uint64_t pol = l2_evict_first();
    const uint32_t lead = elect_lane();
    bool ok = true;
    int ui = 0;  // pieces whose Q is on its way
#pragma unroll 1
    for (int n = 0;; ++n) {
      const int i = n % kRing;
      if (n >= kRing) ok = __all_sync(0xffffffffu, wait(sm.ring_empty[i], (n / kRing - 1) & 1, abort_flag));
      if (!ok) break;
      const bool more = next_piece(sm, P, w, w1, p);
      if (!more) p.b = -1;
      if (lane == 0) {
        sm.ring[i] = p;
        mbar_arrive(smem_u32(&sm.ring_full[i]));
      }
      if (!more) break;
      if (p.t1 == p.t0) continue;
      // Its Q, a box of tokens x G heads per 64 dims, once the piece before has no S
      // MMA left; rows past the piece's tokens hold what follows and are nobody's.  A
      // single token's box is its own: 64 KB of rows that are nobody's are not read,
      // and zeros in them (from the start, while units are single tokens) leave the
      // tensor core little to switch.
      if (ui > 0) ok = __all_sync(0xffffffffu, wait(sm.q_empty, (ui - 1) & 1, abort_flag));
      if (!ok) break;
      const uint32_t bar = PAIR ? map_rank(smem_u32(&sm.q_ready), 0) : smem_u32(&sm.q_ready);
      const bool one = p.ntok == 1;
      const int rows = one ? (rank ? 0 : P.G) : P.TC * P.G;
      if (lane == 0) mbar_expect_tx_cluster<PAIR>(bar, rows * D * 2);
      __syncwarp();
      if (rows > 0) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d<CG>(lead, smem_u32(smem) + F::OFF_Q + c * (kRows * 128), one ? &q1_map : &q_map, 0, p.h * P.G,
                          p.tok0 + rank * P.TC, c, bar, pol);
      }
      ++ui;
    }
    if (lane == 0) sm.sent[2] = ui;
    if (!ok && lane == 0 && !*abort_flag) set_abort<PAIR>(sm, rank, status);
  } else if (warp >= kProdWarp0) {
    // ------------------------------------------- producers: paged K/V tiles
    // A dependent instruction costs a lone warp 4 to 6 cycles, so what a tile
    // takes is counted in instructions: K and V have code and a warp each (one
    // body for both, three warps sharing its rows, took 2700 cycles a tile).
    auto produce = [&](auto v_) {
      constexpr bool V = decltype(v_)::value;
      // K: this CTA's rows, all chunks; V: all rows, this CTA's chunks
      constexpr int NG = V ? KT / 16 : F::KR / 16, NC = V ? F::VC : F::KC, kStages = V ? F::VS : F::KS;
      const int g0 = V ? 0 : rank * NG, c0 = V ? rank * NC : 0;
      uint64_t* full = V ? sm.v_full : sm.k_full;
      uint64_t* empty = V ? sm.v_empty : sm.k_empty;
      int* mixed = V ? sm.v_mixed : sm.k_mixed;
      const uint32_t ring = V ? v_base : k_base;
      constexpr uint32_t kStageBytes = V ? F::kVBytes : F::kKBytes;
      const uint64_t pol_first = l2_evict_first(), pol_keep = l2_evict_normal();
      const uint64_t pitch = (uint32_t)a.kv_st * 2u;  // bytes, below 2^32
      const uint32_t lead = elect_lane();
      int4* slots = sm.slots[V];
      int g = 0;
      bool ok = true;
      while (ok && take(p)) {
        const int T = p.t1 - p.t0;
        if (T == 0) continue;
        const int32_t* idx = a.kv_indices + p.k0;
        const uint64_t pol = p.once ? pol_first : pol_keep;
        int s[4];  // slots of keys 4 lane + q of a tile; past the request's end, of its last
        auto fetch = [&](int tile) {
#pragma unroll
          for (int q = 0; q < 4; ++q) s[q] = __ldg(idx + min(tile * KT + 4 * lane + q, p.L - 1));
        };
        fetch(p.t0);
#pragma unroll 1
        for (int t = 0; t < T; ++t) {
          const int gt = g + t, st = gt % kStages, j0 = (p.t0 + t) * KT;
          int4 c = make_int4(s[0], s[1], s[2], s[3]);
          if (t + 1 < T) fetch(p.t0 + t + 1);
          const uint32_t n_slots = (uint32_t)a.n_slots;
          if ((uint32_t)c.x >= n_slots || (uint32_t)c.y >= n_slots || (uint32_t)c.z >= n_slots ||
              (uint32_t)c.w >= n_slots) {
            raise_status(status, DFT_DEV_BAD_INDEX);
            c = make_int4((uint32_t)c.x < n_slots ? c.x : 0, (uint32_t)c.y < n_slots ? c.y : 0,
                          (uint32_t)c.z < n_slots ? c.z : 0, (uint32_t)c.w < n_slots ? c.w : 0);
          }
          // boxes: bit 4 i set where the 16 slots of group i are consecutive; keys past the end go along
          const int first = __shfl_sync(0xffffffffu, c.x, lane & 28), at0 = first + 4 * (lane & 3);
          const int left = p.L - j0 - 4 * lane;
          uint32_t boxes = __ballot_sync(
              0xffffffffu, (uint32_t)first + 16 <= n_slots && (left <= 0 || c.x == at0) && (left <= 1 || c.y == at0 + 1) &&
                               (left <= 2 || c.z == at0 + 2) && (left <= 3 || c.w == at0 + 3));
          boxes &= boxes >> 1;
          boxes = boxes & boxes >> 2 & 0x11111111u;
          // groups with a key; the others' rows stay as they are
          const int n = min(NG, (p.L - j0 + 15) / 16 - g0);
          const uint32_t mine = n > 0 ? boxes >> 4 * g0 & (0xFFFFFFFFu >> (32 - 4 * n)) : 0u;
          if (gt >= kStages) {
            ok = __all_sync(0xffffffffu, wait(empty[st], (gt / kStages - 1) & 1, abort_flag));
            if (!ok) {
              g += t;
              break;
            }
          }
          // rank 0's barrier takes both CTAs' boxes, a rank 1's own its cp.async
          const uint32_t bar = PAIR ? map_rank(smem_u32(&full[st]), 0) : smem_u32(&full[st]);
          const uint32_t dst = ring + st * kStageBytes;
          const bool copies = __popc(mine) < n;  // their readers need a proxy fence
          if (lane == 0) {
            mixed[st] = copies;
            mbar_expect_tx_cluster<PAIR>(bar, __popc(mine) * 16 * NC * 128);
          }
          slots[lane] = c;
          __syncwarp();
          auto send = [&](uint32_t go, int i, int row) {
            const uint32_t at = dst + i * NC * 2048;
            if (V) {
              tma_load_4d<CG>(go, at, &v_map, 0, row, c0, p.h, bar, pol);
            } else {
              tma_load_4d<CG>(go, at, &k_map, 0, row, 0, p.h, bar, pol);
              tma_load_4d<CG>(go, at + NC * 1024, &k_map, 0, row + 8, 0, p.h, bar, pol);
            }
          };
          if (lead) {
#pragma unroll 1
            for (int i = 0; i < n; ++i)
              if (mine >> 4 * i & 1) send(1, i, reinterpret_cast<const int*>(slots)[16 * (g0 + i)]);
          }
          __syncwarp();
          if (copies) {
            // a group's 16 rows of 8 NC pieces of 16 bytes, 32 pieces a turn
            constexpr int kRow = 32 / (8 * NC);  // rows a turn
            const int lr = lane / (8 * NC), col = lane % (8 * NC);
            const unsigned char* src = static_cast<const unsigned char*>(V ? a.v_cache : a.k_cache) +
                                       ((int64_t)p.h * a.kv_sh + 64 * c0) * 2 + col * 16;
            const uint32_t to = dst + (col >> 3) * (V ? 2048 : 1024) + lr * 128, swz = ((col ^ lr) & 7) << 4;
            const int* slot = reinterpret_cast<const int*>(slots) + 16 * g0 + lr;
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
              if (mine >> 4 * i & 1) continue;
              constexpr int kTurns = 4 * NC;
#pragma unroll
              for (int q0 = 0; q0 < kTurns; q0 += 4) {
                int sl[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) sl[q] = slot[16 * i + (q0 + q) * kRow];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const int row = (q0 + q) * kRow;  // and lr
                  cp_async16(to + i * (NC * 2048) + (V ? row * 128 : (row >> 3) * (NC * 1024) + (row & 7) * 128) +
                                 (swz ^ ((row & 7) << 4)),
                             src + (uint64_t)(uint32_t)sl[q] * pitch, 16u, pol);
                }
              }
            }
            __syncwarp();
          }
          cp_async_arrive_noinc(smem_u32(rank ? (V ? &sm.v_copied[st] : &sm.k_copied[st]) : &full[st]));
        }
        if (ok) g += T;
      }
      ok = ok && p.b != -2;
      if (!ok && lane == 0 && !*abort_flag) set_abort<PAIR>(sm, rank, status);
      if (lane == 0) sm.sent[V] = g;
      cp_async_wait_all();
    };
    if (warp == kProdWarp0) produce(Int<0>());
    else produce(Int<1>());
  } else {
    // ------------- softmax and output, two threads per row, one half of the columns each
    constexpr float kBias = BF ? 0.f : 6.f; // float16 P: up to 2^14, so that small weights stay clear of its smallest step
    const int r = (warp & 3) * 32 + lane;   // TMEM lane
    const int wg = warp >> 2;               // half of S's, O's and Q's columns
    const int pair_bar = 1 + (warp & 3);    // named barrier of warps w and w + 4 (same rows)
    const int wq = warp & 3;
    const int rt = (int)(r * P.inv_G >> 16), g_ = r - rt * P.G;  // the row's token in the CTA, and its head
    const int tok = rt < P.TC ? rank * P.TC + rt : 1 << 20;      // in the piece; rows past the last token are spare
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const float sc = a.sm_scale * kLog2e;
    // a partial slot that no piece of this CTA fills is marked so
    int slots_used = 0;
    // A row's two warps meet at the same named barriers in the same order; every
    // early exit is decided from outcomes that both have exchanged there.
    bool held = true;  // false: a wait gave up since the last exchange
    bool ok = true;
    int g = 0, ui = 0, calls = 0;
    // the next piece with keys; those without give zero rows
    auto next_live = [&](Piece& u) {
      while (take(u) && u.t1 == u.t0) {
        if (tok < u.ntok) {
          uint4* orow = reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.o) +
                                                 ((int64_t)(u.tok0 + tok) * a.o_st + (int64_t)(u.h * P.G + g_) * a.o_sh) * 2 +
                                                 wg * D);
#pragma unroll 1
          for (int q = 0; q < D / 16; ++q) orow[q] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      const int par = calls++ & 1;
      held = held && u.b != -2;
      if (lane == 0) sm.okt[par][wg][wq] = held;
      named_bar(pair_bar, 64);
      ok = held && sm.okt[par][wg ^ 1][wq];
      return u.b >= 0;
    };
    // this thread's share of a masked tile's V: rows past the end and non-finite values -> 0
    auto clean_v = [&](const Piece& u, int t, int gt) -> bool {
      constexpr uint32_t kExp = BF ? 0x7F807F80u : 0x7C007C00u, kOne = BF ? 0x00800080u : 0x04000400u;
      const int j0 = (u.t0 + t) * KT, st = gt % F::VS;
      if (!__all_sync(0xffffffffu, rank ? wait(sm.v_here[gt % NB], (gt / NB) & 1, abort_flag)
                                        : wait(sm.v_full[st], (gt / F::VS) & 1, abort_flag)))
        return false;
      const int live = min(KT, u.L - j0);          // rows of real keys
      // rows from 32 first on are not seen by every token
      const int first = max(0, min(live, u.vis0 - j0)) >> 5;
      unsigned char* vb = smem + F::OFF_V + st * F::kVBytes;
      bool any = false, wrote = false;
      // A thread: 16 bytes of each chunk of rows (tid >> 3) + 32 i.  Kept short: this runs
      // once a unit, and most of its 700 to 1000 cycles are fetching code (1250 unrolled).
#pragma unroll 1
      for (int i = first; i < KT / 32; ++i) {
        uint4* at = reinterpret_cast<uint4*>(vb + (i * 2 + (tid >> 7)) * (F::VC * 2048)) + (tid & 127);
        if (32 * i + (tid >> 3) >= live) {
#pragma unroll
          for (int c = 0; c < F::VC; ++c) at[c * 128] = make_uint4(0u, 0u, 0u, 0u);
          wrote = true;
          continue;
        }
        uint4 x[F::VC];
#pragma unroll
        for (int c = 0; c < F::VC; ++c) x[c] = at[c * 128];
        // a half's exponent is all ones iff adding one to it carries out
        uint32_t hit = 0;
#pragma unroll
        for (int c = 0; c < F::VC; ++c)
          hit |= ((x[c].x & kExp) + kOne) | ((x[c].y & kExp) + kOne) | ((x[c].z & kExp) + kOne) | ((x[c].w & kExp) + kOne);
        if (hit & 0x80008000u) {
          any = true;
          uint32_t* y = reinterpret_cast<uint32_t*>(at);
#pragma unroll 1
          for (int j = 0; j < F::VC * 4; ++j) {
            uint32_t& z = y[(j >> 2) * 512 + (j & 3)];
            z &= ~(((((z & kExp) + kOne) & 0x80008000u) >> 15) * 0xFFFFu);
          }
        }
      }
      if (any) {  // every row's epilogue, the other CTA's too
        *reinterpret_cast<volatile int*>(&sm.odd[ui & 7]) = ui + 1;
        if (PAIR) st_cluster(map_rank(smem_u32(&sm.odd[ui & 7]), rank ^ 1), ui + 1);
      }
      if (any || wrote) fence_async_smem();  // these writes before the tensor core's reads
      return true;
    };
    // Unit after unit; the next one's Q, K and S come in while the last one's output goes out.
    bool pending = false;
    float m_used = -INFINITY, l = 0.f;
    Piece u;
    while (ok) {
      const bool more = next_live(p);
      if (!ok) break;
      if (pending) {
        // ---- epilogue of unit u: wait for its last P V, then O (or its partial) out
        const bool row_ok = tok < u.ntok, busy = wq * 32 < min(P.TC, u.ntok - rank * P.TC) * P.G;
        const int vis = max(0, min(u.L, u.vis0 + (row_ok ? tok : 0)));
        sm.lsum[wg][r] = l;
        named_bar(pair_bar, 64);
        l = sm.lsum[0][r] + sm.lsum[1][r];
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t prow = (int64_t)(2 * worker + max(u.slot, 0)) * F::kSlotRows;
        // the rows of this lane's two; its 16 bytes of each 32
        unsigned char* to[2];
        bool there[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int rr = (r & ~1) + q, t = (int)(rr * P.inv_G >> 16);
          there[q] = t < min(P.TC, u.ntok - rank * P.TC);
          to[q] = static_cast<unsigned char*>(a.o) + wg * D + (lane & 1) * 16 +
                  ((int64_t)(u.tok0 + rank * P.TC + t) * a.o_st + (int64_t)(u.h * P.G + rr - t * P.G) * a.o_sh) * 2;
        }
        held = held && __all_sync(0xffffffffu, wait(sm.o_full, ui & 1, abort_flag));
        tc_fence_after();
        if (held && busy) {
          const bool odd = sm.odd[ui & 7] == ui + 1;
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 16) {
            float v[16];
            tmem_ld16(tmem + lane_base + F::COL_O + (D / 2) * wg + c, v);
            if (odd) {
              // the masked tiles' non-finite values, for the rows that see their keys
#pragma unroll 1
              for (int j = max(u.t0 * KT, max(u.vis0, 0) / KT * KT); j < min(u.t1 * KT, vis); ++j) {
                const int64_t s = a.kv_indices[u.k0 + j];
                if (s < 0 || s >= a.n_slots) continue;
                const uint16_t* vr = static_cast<const uint16_t*>(a.v_cache) + s * a.kv_st + u.h * a.kv_sh + (D / 2) * wg + c;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float y = unpack<BF>(vr[i]);
                  v[i] += fabsf(y) < INFINITY ? 0.f : y;
                }
              }
            }
            if (u.slot < 0) {
              // two lanes swap 16-byte pieces, so that a store writes 32 bytes of 16
              // rows and not 16 of 32
              uint32_t y[2][4];
#pragma unroll
              for (int q = 0; q < 8; ++q) y[q >> 2][q & 3] = pack2<BF>(v[2 * q] * inv, v[2 * q + 1] * inv);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t get = __shfl_xor_sync(0xffffffffu, lane & 1 ? y[0][e] : y[1][e], 1);
                if (lane & 1) y[0][e] = get;
                else y[1][e] = get;
              }
#pragma unroll
              for (int q = 0; q < 2; ++q)  // y[q]: piece lane & 1 of the q-th of the two rows
                if (there[q])
                  *reinterpret_cast<uint4*>(to[q] + c * 2) = make_uint4(y[q][0], y[q][1], y[q][2], y[q][3]);
            } else if (row_ok) {
              float* dst = P.ws_o + prow * D + ((D / 16 * wg + (c >> 3)) * F::kSlotRows + rank * kRows + r) * 8;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(dst + (q >> 1) * (F::kSlotRows * 8) + (q & 1) * 4) =
                    make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            }
          }
          if (u.slot >= 0 && wg == 0 && row_ok) {
            *reinterpret_cast<float2*>(P.ws_ml + 2 * (prow + rank * kRows + r)) = make_float2(m_used, l);
          }
        }
        if (held) {
          if (u.slot >= 0) {
            slots_used |= 1 << u.slot;
            if (tid == 0 && rank == 0)
              P.ws_meta[2 * worker + u.slot] = make_int4(1 | (u.last ? 2 : 0), u.tok0, u.ntok, u.h);
          }
          // O may now be overwritten by the next unit's first P V
          tc_fence_before();
          warp_arrive<PAIR>(sm.o_free);
        }
        ++ui;
      }
      if (!more) break;
      u = p;
      pending = true;
      const bool row_ok = tok < u.ntok;
      const int T = u.t1 - u.t0;
      const int vis = max(0, min(u.L, u.vis0 + (row_ok ? tok : 0)));  // keys this row sees: j < vis
      const bool busy = wq * 32 < min(P.TC, u.ntok - rank * P.TC) * P.G;  // the warp holds rows
      m_used = -INFINITY;
      l = 0.f;
#pragma unroll 1
      for (int t = 0; t < T; ++t) {
        const int gt = g + t, sb = gt % NB, par = gt & 1;
        const bool got = __all_sync(0xffffffffu, held && wait(sm.s_full[sb], (gt / NB) & 1, abort_flag));
        // keys that every token of the tile sees need no mask (uniform)
        const int j0 = (u.t0 + t) * KT;
        const bool plain = j0 + KT <= u.vis0 && j0 + KT <= u.L;
        if (busy) {  // else spare rows: whatever P holds stays in them
          const uint32_t ts = tmem + lane_base + F::COL_S + KT * sb + 64 * wg;  // this thread's 64 columns of S
          float x[64];
          tc_fence_after();
          tmem_ld32_async(ts, &x[0]);
          tmem_ld32_async(ts + 32, &x[32]);
          tmem_ld_wait(x);
          if (!plain) {
            const int seen = max(0, min(64, vis - j0 - 64 * wg));  // columns that the row sees
            const uint32_t off[2] = {seen >= 32 ? 0u : 0xFFFFFFFFu << seen, seen >= 64 ? 0u : 0xFFFFFFFFu << max(0, seen - 32)};
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (off[i >> 5] >> (i & 31) & 1) x[i] = -INFINITY;
          }
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            mx[0] = fmaxf(fmaxf(mx[0], x[i]), x[i + 1]);
            mx[1] = fmaxf(fmaxf(mx[1], x[i + 2]), x[i + 3]);
          }
          float tmax = fmaxf(mx[0], mx[1]);
          // S stays raw: P = 2^(S sc - m)
          tmax *= sc;
          sm.xmax[par][wg][r] = tmax;
          if (lane == 0) sm.okx[par][wg][wq] = got;
          named_bar(pair_bar, 64);
          tmax = fmaxf(tmax, sm.xmax[par][wg ^ 1][r]);
          ok = got && sm.okx[par][wg ^ 1][wq];
          if (!ok) break;
          // a row moves its reference only when the tile's maximum exceeds it by
          // more than 8 (P <= 2^8 otherwise); O then scales by 2^(old - new)
          const bool grow = tmax > m_used + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            const float m_new = grow ? tmax : m_used;
            if (t > 0) {
              // O holds P V of this unit's earlier tiles: wait for the last, then rescale this half row
              const bool done = __all_sync(0xffffffffu, wait(sm.pv_done[(gt - 1) % NB], ((gt - 1) / NB) & 1, abort_flag));
              if (lane == 0) sm.okr[par][wg][wq] = done;
              named_bar(pair_bar, 64);
              ok = done && sm.okr[par][wg ^ 1][wq];
              if (!ok) break;
              tc_fence_after();
              const float alpha = grow ? ex2_approx(m_used - m_new) : 1.f;
#pragma unroll 1
              for (int c = 0; c < D / 2; c += 32) {
                float v[32];
                tmem_ld32(tmem + lane_base + F::COL_O + (D / 2) * wg + c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= alpha;
                tmem_st32(tmem + lane_base + F::COL_O + (D / 2) * wg + c, v);
              }
              l *= alpha;
            }
            m_used = m_new;
          }
          // a row whose scores so far are all -inf has no reference yet: its P is 0
          const float nm = m_used == -INFINITY ? 0.f : kBias - m_used;
          const f32x2 sc2 = pk2(sc, sc), nm2 = pk2(nm, nm);
          f32x2 sum2[2] = {pk2(0.f, 0.f), pk2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float e0, e1;
              upk2(fma2(pk2(x[c + 2 * i], x[c + 2 * i + 1]), sc2, nm2), e0, e1);
              const float p0 = ex2_approx(e0), p1 = ex2_approx(e1);
              sum2[i & 1] = add2(sum2[i & 1], pk2(p0, p1));
              pk[i] = pack2<BF>(p0, p1);
            }
            tmem_st16_async(ts + c / 2, pk);  // over this thread's own columns, which are read
          }
          float s0, s1;
          upk2(add2(sum2[0], sum2[1]), s0, s1);
          l += s0 + s1;
          tmem_st_wait();
        }
        held = got && (plain || clean_v(u, t, gt));
        tc_fence_before();
        if (held) warp_arrive<PAIR>(sm.p_full[sb]);
        else if (!busy) break;
      }
      if (!ok) break;
      g += T;
    }
    ok = ok && held && p.b != -2;
    if (tid == 0 && rank == 0)
      for (int s = 0; s < 2; ++s)
        if (!(slots_used >> s & 1)) P.ws_meta[2 * worker + s] = make_int4(0, 0, 0, 0);
    if (!ok && !*abort_flag) set_abort<PAIR>(sm, rank, status);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // nothing of the other CTA's arrives here any more
  if (*abort_flag) {
    // A wait gave up (in both CTAs of a pair, or neither): MMAs may not have taken
    // all copies, and those must land before their shared memory goes.  No role runs
    // any more, so a phase that lacks arrivals gets them here and is waited for; its
    // transactions, rank 1's among them, are all on rank 0's barriers.  Every phase
    // before the ones below is complete: their stages were handed out again.
    if (rank == 0 && tid == 0) {
      const auto other = [&](int& x) { return PAIR ? (int)ld_cluster(map_rank(smem_u32(&x), 1)) : x; };
      const auto settle = [&](uint64_t& bar, int missing, int phase) {
        for (int i = 0; i < missing; ++i) mbar_arrive(smem_u32(&bar));
        mbar_wait(smem_u32(&bar), phase & 1);
      };
      const int q0 = sm.sent[2], q1 = other(sm.sent[2]), nq = max(q0, q1);
      if (nq > 0) settle(sm.q_ready, (q0 < nq) + (q1 < nq), nq - 1);
#pragma unroll 1
      for (int v = 0; v < 2; ++v) {
        const int n = v ? F::VS : F::KS, g0 = sm.sent[v], g1 = other(sm.sent[v]);
        const int relayed = PAIR ? other(sm.relayed[v]) : 0, g = max(g0, g1);
#pragma unroll 1
        for (int gt = max(0, g - n); gt < g; ++gt)
          settle((v ? sm.v_full : sm.k_full)[gt % n], (gt < g0 ? 0 : 32 + 1) + (PAIR ? (gt >= g1) + (gt >= relayed) : 0),
                 gt / n);
      }
    }
    __syncwarp();
    if (PAIR) cluster_sync();  // rank 1's shared memory stays until then
  }
  if (warp == kCtlWarp) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_2(tmem, kTmemCols);
    else tmem_dealloc(tmem, kTmemCols);
  }
}

// Merge the partials of the unit that worker c begins and leaves unfinished: its
// own, then the continuing slots of the workers after it up to the unit's last.
//   o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s
constexpr int kMergeThreads = 256, kMergeY = 8, kMaxWorkers = 160;
template <bool BF, int D>
__global__ void __launch_bounds__(kMergeThreads) chunk_attn_merge(const __grid_constant__ Params P) {
  pdl_wait();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // a warp: 8 rows, 32 dims; a pass of the block: kPass rows
  constexpr int kWide = D / 32, kPass = kMergeThreads / 32 / kWide * 8, kSlotRows = Cfg<D>::kSlotRows;
  __shared__ int list[kMaxWorkers + 1];
  __shared__ uint32_t used[kMergeThreads / 32], ends[kMergeThreads / 32];
  __shared__ float2 mls[kMaxWorkers * kPass];
  static_assert(kMaxWorkers <= kMergeThreads, "a thread per worker");
  const int c = blockIdx.x, grid = gridDim.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 meta = P.ws_meta[2 * c + 1];
  const int flags = (int)threadIdx.x > c && (int)threadIdx.x < grid ? P.ws_meta[2 * threadIdx.x].x : 0;
  if (!(meta.x & 1)) return;
  const dft_chunk_attn_args& a = P.a;
  const int rows = meta.z * P.G, e = warp % kWide * 4 + (lane & 3);  // rows of the unit; this thread's 8 dims
  if (blockIdx.y * kPass >= rows) return;
  // the unit's partials: slot 2c + 1, then the used even slots after it to the unit's last
  const uint32_t u = __ballot_sync(0xffffffffu, flags & 1), l = __ballot_sync(0xffffffffu, flags & 2);
  if (lane == 0) {
    used[warp] = u;
    ends[warp] = l;
  }
  __syncthreads();
  int n = 1;         // partials of the unit
  bool open = true;  // no last one so far
#pragma unroll
  for (int w = 0; w < kMergeThreads / 32; ++w) {
    const uint32_t to = ends[w] ? ends[w] ^ (ends[w] - 1) : 0xFFFFFFFFu;  // up to the first last one
    const uint32_t mine = open ? used[w] & to : 0u;
    if (w == warp) {
      if (mine >> lane & 1) list[n + __popc(mine & ((1u << lane) - 1))] = 2 * threadIdx.x;
    }
    n += __popc(mine);
    open = open && !ends[w];
  }
  if (threadIdx.x == 0) list[0] = 2 * c + 1;
  const int low = P.TC * P.G;  // a unit's first rows are one CTA's, further ones the other's
  for (int i0 = blockIdx.y * kPass; i0 < rows; i0 += kMergeY * kPass) {
    // all partials' (m, l) of the pass's rows at once
    __syncthreads();
    for (int x = threadIdx.x; x < n * kPass; x += kMergeThreads) {
      const int i = i0 + x % kPass;
      if (i < rows)
        mls[x] = *reinterpret_cast<const float2*>(P.ws_ml + 2 * (list[x / kPass] * kSlotRows + (i < low ? i : kRows + i - low)));
    }
    __syncthreads();
    const int rr = warp / kWide * 8 + (lane >> 2), i = i0 + rr;
    if (i >= rows) continue;
    const int tok = (int)(i * P.inv_G >> 16), r = i < low ? i : kRows + i - low;  // its token, its row in a slot
    float M = -INFINITY;
#pragma unroll 1
    for (int k = 0; k < n; ++k) M = fmaxf(M, mls[k * kPass + rr].x);
    const float* part = P.ws_o + (e * kSlotRows + r) * 8;
    float acc[8] = {};
    float L = 0.f;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float4* v = reinterpret_cast<const float4*>(part + (int64_t)list[k] * (kSlotRows * D));
      const float4 v0 = v[0], v1 = v[1];
      const float2 ml = mls[k * kPass + rr];
      // a sum of 0: the row sees none of these keys (a NaN sum goes on)
      const float wgt = ml.y == 0.f ? 0.f : ex2_approx(ml.x - M);
      acc[0] += wgt * v0.x;
      acc[1] += wgt * v0.y;
      acc[2] += wgt * v0.z;
      acc[3] += wgt * v0.w;
      acc[4] += wgt * v1.x;
      acc[5] += wgt * v1.y;
      acc[6] += wgt * v1.z;
      acc[7] += wgt * v1.w;
      L += wgt * ml.y;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    unsigned char* orow = static_cast<unsigned char*>(a.o) +
                          ((int64_t)(meta.y + tok) * a.o_st + (int64_t)(meta.w * P.G + (i - tok * P.G)) * a.o_sh) * 2;
    reinterpret_cast<uint4*>(orow)[e] =
        make_uint4(pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv),
                   pack2<BF>(acc[4] * inv, acc[5] * inv), pack2<BF>(acc[6] * inv, acc[7] * inv));
  }
}

// ------------------------------------------------------------------ host --
using gtile::al16;

int check_args(const dft_chunk_attn_args* a) {
  if (!a || a->B < 0 || a->T < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->n_slots < 0 || a->n_kv < 0)
    return DFT_ERR_INVALID;
  if (a->dtype != DFT_BF16 && a->dtype != DFT_F16) return DFT_ERR_INVALID;
  if (!(a->sm_scale > 0.f) || !(a->sm_scale * kLog2e < INFINITY)) return DFT_ERR_INVALID;  // the kernel scales by both
  if ((a->D != 64 && a->D != 128 && a->D != 256) || a->Hq / a->Hkv > 128 || a->B > kMaxB) return DFT_ERR_UNSUPPORTED;
  if (a->B == 0 || a->T == 0) return DFT_OK;
  if (!a->q || !a->o || !a->qo_indptr || !a->kv_indptr || !a->k_cache || !a->v_cache || a->n_slots < 1 ||
      (a->n_kv > 0 && !a->kv_indices))
    return DFT_ERR_INVALID;
  if (!al16(a->q) || !al16(a->o) || !al16(a->k_cache) || !al16(a->v_cache)) return DFT_ERR_UNSUPPORTED;
  if (a->q_st % 8 || a->q_sh % 8 || a->o_st % 8 || a->o_sh % 8 || a->kv_st % 8 || a->kv_sh % 8)
    return DFT_ERR_UNSUPPORTED;
  if ((a->T > 1 && a->q_st <= 0) || (a->Hq > 1 && a->q_sh <= 0) || a->kv_st < a->D || (a->Hkv > 1 && a->kv_sh < a->D) ||
      !rows_apart(a->D, {a->T, a->Hq}, {a->o_st, a->o_sh}))
    return DFT_ERR_INVALID;
  if (a->kv_st >= ((int64_t)1 << 31) || a->kv_sh >= ((int64_t)1 << 38) || a->q_st >= ((int64_t)1 << 38) ||
      a->q_sh >= ((int64_t)1 << 38) || a->n_slots > 0x7FFFFFFF)
    return DFT_ERR_UNSUPPORTED;
  return DFT_OK;
}

// one CTA per SM; the merge has room for so many partials of a unit
int worker_count(int D) {
  const int n = gtile::sm_count() / (D == 256 ? Cfg<256>::CG : 1);
  return n < kMaxWorkers ? n : kMaxWorkers;
}

struct Workspace {
  int64_t o, ml, meta, total;
};
Workspace workspace(const dft_chunk_attn_args* a, int workers) {
  const int64_t slots = 2 * (int64_t)workers, rows = slots * kRows * (a->D == 256 ? Cfg<256>::CG : 1);
  Workspace w;
  w.meta = 0;
  w.ml = up256(slots * sizeof(int4));
  w.o = w.ml + up256(rows * 2 * sizeof(float));
  w.total = w.o + rows * a->D * sizeof(float);
  return w;
}

// three-level strides in elements under 64 contiguous dims
bool encode(CUtensorMap* m, const dft_chunk_attn_args* a, const void* base, const int64_t (&size)[3],
            const int64_t (&stride)[3], const int (&box_)[3]) {
  const cuuint64_t dims[4] = {64, (cuuint64_t)size[0], (cuuint64_t)size[1], (cuuint64_t)size[2]};
  const cuuint64_t strides[3] = {(cuuint64_t)stride[0] * 2, (cuuint64_t)stride[1] * 2, (cuuint64_t)stride[2] * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_[0], (cuuint32_t)box_[1], (cuuint32_t)box_[2]}, estr[4] = {1, 1, 1, 1};
  return gtile::encode_fn() &&
         gtile::encode_fn()(m, a->dtype == DFT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF, int D>
int launch(const Params& P, int workers, const CUtensorMap& q_map, const CUtensorMap& q1_map, const CUtensorMap& k_map,
           const CUtensorMap& v_map, int32_t* status, cudaStream_t st) {
  DFT_CUDA_CHECK(cudaFuncSetAttribute(chunk_attn_kernel<BF, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)smem_bytes<D>()));
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(workers * Cfg<D>::CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes<D>();
  cfg.stream = st;
  cfg.attrs = attr;
  // like the merge, it comes up under the launch before it and waits for its end
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = Cfg<D>::kPair ? 2 : 1;
  DFT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, chunk_attn_kernel<BF, D>, q_map, q1_map, k_map, v_map, P, status));
  return launch_pdl(chunk_attn_merge<BF, D>, dim3((unsigned)workers, kMergeY), dim3(kMergeThreads), 0, st, P);
}

}  // namespace

extern "C" int64_t dft_chunk_attn_workspace_bytes(const dft_chunk_attn_args* a) {
  if (check_args(a)) return -1;
  if (a->B == 0 || a->T == 0) return 0;
  return workspace(a, worker_count(a->D)).total;
}

extern "C" int dft_chunk_attn(const dft_chunk_attn_args* a, void* ws, int32_t* dev_status, void* stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  if (a->B == 0 || a->T == 0) return DFT_OK;
  if (!ws || !al16(ws)) return DFT_ERR_INVALID;
  const int workers = worker_count(a->D);
  const Workspace w = workspace(a, workers);
  Params P;
  memset(&P, 0, sizeof(P));
  P.a = *a;
  P.unit_keys = unit_keys(a->D);
  P.G = a->Hq / a->Hkv;
  P.inv_G = (65535u + P.G) / P.G;
  P.TC = kRows / P.G;
  P.TQ = P.TC * (a->D == 256 ? Cfg<256>::CG : 1);
  P.ws_meta = reinterpret_cast<int4*>(static_cast<char*>(ws) + w.meta);
  P.ws_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + w.ml);
  P.ws_o = reinterpret_cast<float*>(static_cast<char*>(ws) + w.o);
  // K, V: (slots, 64-dim chunks, heads); Q: (heads, tokens, chunks); the stride of a
  // dimension of one may be anything and is not looked at
  const int64_t chunks = a->D / 64, kv_sh = a->Hkv > 1 ? a->kv_sh : a->D;
  const int64_t q_st = a->T > 1 ? a->q_st : a->D, q_sh = a->Hq > 1 ? a->q_sh : a->D;
  const int vc = a->D == 256 ? Cfg<256>::VC : (int)chunks;
  CUtensorMap q_map, q1_map, k_map, v_map;
  if (!encode(&q_map, a, a->q, {a->Hq, a->T, chunks}, {q_sh, q_st, 64}, {P.G, P.TC, 1}) ||
      !encode(&q1_map, a, a->q, {a->Hq, a->T, chunks}, {q_sh, q_st, 64}, {P.G, 1, 1}) ||
      !encode(&k_map, a, a->k_cache, {a->n_slots, chunks, a->Hkv}, {a->kv_st, 64, kv_sh}, {8, (int)chunks, 1}) ||
      !encode(&v_map, a, a->v_cache, {a->n_slots, chunks, a->Hkv}, {a->kv_st, 64, kv_sh}, {16, vc, 1}))
    return DFT_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a->dtype == DFT_BF16;
#define DFT_GO(D_)                                                                       \
  return bf ? launch<true, D_>(P, workers, q_map, q1_map, k_map, v_map, dev_status, st) \
            : launch<false, D_>(P, workers, q_map, q1_map, k_map, v_map, dev_status, st)
  if (a->D == 64) DFT_GO(64);
  if (a->D == 128) DFT_GO(128);
  DFT_GO(256);
#undef DFT_GO
}
