// Causal attention of new tokens over the paged KV cache (sm_100a).
//
// Per request b with n new tokens (its rows of q) and L keys, token i and
// q-head hq:  o = softmax_j(q . k_j * sm_scale | j <= L - n + i) . v_j.
//
// A unit is (request, kv-head, query tile).  The G q-heads of a kv-head share
// its keys, so a tile's 128 rows are 128 / G tokens x G heads (row = token * G
// + head) and one tcgen05 MMA of M = 128 serves them all; a single token's G
// rows go through the same tile, whose spare rows cost no memory traffic.  Per
// tile of KT keys, one pass with a running maximum and sum:
//   K, V  by slot, 16 keys at a time, into separate rings of stages by three
//         producer warps: where the 16 slots are consecutive (pages of 16 and
//         more) one TMA box of 16 cache rows x 64 dims per copy, else 16-byte
//         cp.async row by row (a gather of four rows per TMA copy took 39 ns a
//         copy, 5 us per 64 KB tile)
//   S     = Q K^T    kind::f16, A = Q from TMEM, M=128 N=KT K=D, fp32 in TMEM
//   P     = 2^(S sm_scale log2e - m), two threads per row; the reference m
//         moves (and O is rescaled in TMEM) only when the maximum grows by
//         more than 8, so P <= 2^8; rounded to the 16-bit type over its own S
//         (the second product's operand has V's type), summed unrounded
//   O    += P V      A = P from TMEM, V as an MN-major operand, N = D
// S / P are double-buffered, so the S MMA of tile t+1 runs under the softmax
// of tile t.
//
// Work is split by keys, not by unit: unit costs (keys + a fixed part) are laid
// out on one line, and CTA c takes the c-th share of it, whatever units that
// crosses.  One long prompt, many ragged requests and one long decode all fill
// the GPU evenly, from lengths that only the device knows.  A unit cut by a
// share's border leaves partials (O, m, l) that a second kernel merges.
//
// Tiles past a row's last key hold the masked keys' values: their P is 0, but 0
// times NaN or infinity is not.  In those tiles alone the softmax threads zero
// V's rows past the request's end and its non-finite elements before the P V
// product reads them; the epilogue adds such an element back to the rows that
// do see its key.
//
// Every wait is bounded (~1 s); on timeout the CTA raises DFT_DEV_TIMEOUT,
// drains its copies and MMAs (bounded), frees TMEM and exits.
#include "dft_common.cuh"
#include "dft_gdn_tile.cuh"
#include "dft_tc.cuh"

#include <cstring>

using namespace dft;
using namespace dft::tc;

namespace {

constexpr int kMaxB = 1024;
constexpr int kRows = 128;
constexpr int kSoftmax = 256;     // two threads per query row
constexpr int kCtlWarp = 8, kProdWarp0 = 9, kProdWarps = 3, kProducers = 32 * kProdWarps;
constexpr int kThreads = 384;     // twelve warps leave 168 registers a thread
constexpr uint32_t kTmemCols = 512;
// A unit's fixed cost in keys (query load, first tile's latency, output), and
// the least share of a CTA: under it a cut costs more than it spreads.
constexpr int kUnitKeys = 128;
constexpr int kMinShare = 256;

template <int D>
struct Cfg {
  static constexpr int KT = D == 256 ? 64 : 128;              // keys per tile: O, Q and two S fit TMEM's 512 columns
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kChunks = D / 64;                      // 128-byte columns of a tile
  static constexpr uint32_t kChunkBytes = KT * 128;
  static constexpr uint32_t kTileBytes = kChunks * kChunkBytes;
  static constexpr uint32_t COL_O = 0, COL_Q = D, COL_S = D + D / 2;  // S / P buffer b at COL_S + KT b
  static_assert(COL_S + 2 * KT <= kTmemCols, "TMEM");
};

struct Small {
  uint64_t q_ready;
  uint64_t k_full[6], k_empty[6], v_full[6], v_empty[6];
  uint64_t s_full[2], p_full[2];
  uint64_t o_done, o_full, o_free, mma_done;
  uint32_t tmem_base;
  int abort;
  int odd[8];               // [piece & 7] = piece + 1 when one of its masked tiles held a non-finite value
  float xmax[2][2][kRows];  // [tile parity][half][row] tile max exchange between a row's two threads
  float lsum[2][kRows];     // [half][row] final row sums
  int okx[2][2][4];         // [tile parity][half][row warp] wait outcomes, shared by a row's two warps
  int okr[2][2][4];         // the same for the rescale's wait
  int oke[2][4];            // [half][row warp] the epilogue's wait
  int64_t warp_sum[kThreads / 32];
  int64_t pre[kMaxB + 1];   // cost of the requests before b
  int qo[kMaxB + 1], kv[kMaxB + 1];
};

struct Params {
  dft_chunk_attn_args a;
  int G, TQ;                // q-heads per kv-head, tokens per query tile
  int x_head, row_head;     // kv-head h starts at column h * x_head, row h * row_head of the tensor map
  float* ws_o;              // [2 grid][128][D] partial O: slot 2c continues a unit, 2c + 1 begins one
  float* ws_ml;             // [2 grid][128][2] partial (m, l)
  int4* ws_meta;            // [2 grid] (flags, first token row, tokens, kv-head); flags 1: used, 2: the unit's last
};

template <int D>
constexpr uint32_t smem_bytes() {
  static_assert(2 * Cfg<D>::kStages * Cfg<D>::kTileBytes + sizeof(Small) + 1024 <= 232448, "shared memory");
  return 2 * Cfg<D>::kStages * Cfg<D>::kTileBytes + (uint32_t)sizeof(Small) + 1024;  // + alignment slack
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

__device__ __forceinline__ void set_abort(Small& sm, int32_t* status) {
  *reinterpret_cast<volatile int*>(&sm.abort) = 1;
  raise_status(status, DFT_DEV_TIMEOUT);
}

// -------------------------------------------------------------- schedule --
// Request b: n tokens in nt query tiles, L keys.  Tile i ends at token e =
// min((i + 1) TQ, n) and reads the keys its last token sees, clamp(L - n + e,
// 0, L); its cost is that + kUnitKeys, and the sum over the tiles before i is
// an arithmetic series.
struct Req {
  int n, L, nt;
};
__device__ __forceinline__ Req request(const Small& sm, int b, int TQ) {
  Req r;
  r.n = sm.qo[b + 1] - sm.qo[b];
  r.L = sm.kv[b + 1] - sm.kv[b];
  r.nt = (r.n + TQ - 1) / TQ;
  return r;
}
__device__ __forceinline__ int tile_keys(const Req& r, int i, int TQ) {
  const int64_t e = min((int64_t)(i + 1) * TQ, (int64_t)r.n);
  return (int)max((int64_t)0, r.L - r.n + e);
}
__device__ __forceinline__ int64_t cost_before(const Req& r, int i, int TQ) {
  int64_t last = 0;
  if (i == r.nt && i > 0) {  // the last tile is the one that may be short
    last = r.L + kUnitKeys;
    --i;
  }
  const int64_t a = r.L - (int64_t)r.n;
  const int64_t z = a < 0 ? min((int64_t)i, -a / TQ) : 0;  // tiles that see no key
  return last + (int64_t)i * kUnitKeys + (i - z) * a + TQ * (((int64_t)i * (i + 1) - z * (z + 1)) / 2);
}

// A CTA's part of one unit: key tiles [t0, t1) of nt.
struct Piece {
  int b, h, tok0, ntok;  // first token row of q, tokens
  int vis0, L;           // keys that the first token sees (may be negative), keys of the request
  int t0, t1;
  int slot;              // -1: the whole unit; 0 / 1: partial that continues / begins it
  bool last, once;       // the unit's last tiles; its keys are read by this tile alone
};

// The next piece of the line from w, w < w1, that has something to do.
template <int KT>
__device__ __forceinline__ bool next_piece(const Small& sm, const Params& P, int64_t& w, int64_t w1, Piece& p) {
  while (w < w1) {
    int lo = 0, hi = P.a.B;  // pre[lo] <= w < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sm.pre[mid] <= w) lo = mid;
      else hi = mid;
    }
    const Req r = request(sm, lo, P.TQ);
    const int64_t per_head = cost_before(r, r.nt, P.TQ);
    int64_t rest = w - sm.pre[lo];
    const int h = (int)(rest / per_head);
    rest -= h * per_head;
    int i = 0;
    for (int top = r.nt; top - i > 1;) {
      const int mid = (i + top) >> 1;
      if (cost_before(r, mid, P.TQ) <= rest) i = mid;
      else top = mid;
    }
    const int64_t x0 = rest - cost_before(r, i, P.TQ);
    const int keys = tile_keys(r, i, P.TQ);
    const int64_t cost = keys + kUnitKeys, x1 = min(cost, x0 + (w1 - w));
    w += x1 - x0;
    const int nt = (keys + KT - 1) / KT;
    p.t0 = x0 == 0 ? 0 : (int)min((int64_t)nt, (x0 + KT / 2) / KT);
    p.t1 = x1 == cost ? nt : (int)min((int64_t)nt, (x1 + KT / 2) / KT);
    if (p.t0 == p.t1 && !(nt == 0 && x0 == 0)) continue;
    p.b = lo;
    p.h = h;
    p.tok0 = sm.qo[lo] + i * P.TQ;
    p.ntok = min(P.TQ, r.n - i * P.TQ);
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
    chunk_attn_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const __grid_constant__ Params P, int32_t* status) {
  using F = Cfg<D>;
  constexpr int KT = F::KT, kStages = F::kStages;
  constexpr uint32_t kTile = F::kTileBytes, kChunk = F::kChunkBytes;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Small& sm = *reinterpret_cast<Small*>(smem + 2 * kStages * kTile);
  const volatile int* abort_flag = &sm.abort;
  const dft_chunk_attn_args& a = P.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t k_base = smem_u32(smem), v_base = k_base + kStages * kTile;

  // the merge kernel's blocks may come up now; they wait for this grid to end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == kCtlWarp) {
    if (lane == 0) {
      mbar_init(smem_u32(&sm.q_ready), kSoftmax);
      for (int i = 0; i < kStages; ++i) {
        mbar_init(smem_u32(&sm.k_full[i]), kProducers + 1);
        mbar_init(smem_u32(&sm.k_empty[i]), 1);
        mbar_init(smem_u32(&sm.v_full[i]), kProducers + 1);
        mbar_init(smem_u32(&sm.v_empty[i]), 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&sm.s_full[i]), 1);
        mbar_init(smem_u32(&sm.p_full[i]), kSoftmax);
      }
      mbar_init(smem_u32(&sm.o_done), 1);
      mbar_init(smem_u32(&sm.o_full), 1);
      mbar_init(smem_u32(&sm.o_free), kSoftmax);
      mbar_init(smem_u32(&sm.mma_done), 1);
      sm.abort = 0;
      for (int i = 0; i < 8; ++i) sm.odd[i] = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    tmem_alloc(smem_u32(&sm.tmem_base), kTmemCols);
  }
  // offsets and the requests' costs: thread t sums requests [t per, ...)
  {
    constexpr int kPer = (kMaxB + kThreads - 1) / kThreads;
    for (int i = tid; i <= a.B; i += kThreads) {
      sm.qo[i] = a.qo_indptr[i];
      sm.kv[i] = a.kv_indptr[i];
    }
    __syncthreads();
    int64_t c[kPer], sum = 0;
    bool bad = false;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int b = tid * kPer + q;
      c[q] = 0;
      if (b < a.B) {
        const int q0 = sm.qo[b], q1 = sm.qo[b + 1], k0 = sm.kv[b], k1 = sm.kv[b + 1];
        const bool ok = q0 >= 0 && q0 <= q1 && q1 <= a.T && k0 >= 0 && k0 <= k1 && k1 <= a.n_kv &&
                        k1 - k0 <= 0x7FFFFF00;
        bad |= !ok;
        if (ok && q1 > q0) {
          const Req r = request(sm, b, P.TQ);
          c[q] = a.Hkv * cost_before(r, r.nt, P.TQ);
        }
      }
      sum += c[q];
    }
    if (bad && blockIdx.x == 0) raise_status(status, DFT_DEV_BAD_INDEX);
    int64_t inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) sm.warp_sum[warp] = inc;
    __syncthreads();
    int64_t at = inc - sum;
    for (int i = 0; i < warp; ++i) at += sm.warp_sum[i];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int b = tid * kPer + q;
      if (b <= a.B) sm.pre[b] = at;
      at += c[q];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int64_t total = sm.pre[a.B];
  const int64_t share = max((int64_t)kMinShare, (total + gridDim.x - 1) / gridDim.x);
  const int64_t w0 = min(total, share * blockIdx.x), w1 = min(total, w0 + share);
  int64_t w = w0;
  Piece p;

  if (warp == kCtlWarp) {
    // ------------------------------------------------------ control: MMAs
    if (lane == 0) {
      constexpr uint32_t id_s = BF ? idesc_bf16(128, KT, false) : idesc_f16(128, KT, false);
      constexpr uint32_t id_o = BF ? idesc_bf16(128, D, true) : idesc_f16(128, D, true);
      int g = 0, ui = 0;
      bool ok = true;
      while (ok && next_piece<KT>(sm, P, w, w1, p)) {
        const int T = p.t1 - p.t0;
        if (T == 0) continue;
        ok = mbar_wait_or_abort(smem_u32(&sm.q_ready), ui & 1, abort_flag);
        for (int t = 0; ok && t <= T; ++t) {
          if (t < T) {
            const int gt = g + t, st = gt % kStages, sb = gt & 1;
            ok = mbar_wait_or_abort(smem_u32(&sm.k_full[st]), (gt / kStages) & 1, abort_flag);
            // S/P buffer sb is free once P V of tile gt-2 has retired.  For a
            // unit's first tile that wait happened before the previous unit's
            // last P V was issued: o_done's parity tells phases apart only
            // while P V gt-1 is not yet issued.
            if (ok && t >= 1 && gt >= 2) ok = mbar_wait_or_abort(smem_u32(&sm.o_done), (gt - 2) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            fence_async_smem();  // cp.async (generic proxy) writes -> tensor-core reads
            const uint32_t kb = k_base + st * kTile;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint64_t bd = sw128_desc(kb + (k >> 2) * kChunk + (k & 3) * 32);
              mma_bf16_ts(tmem + F::COL_S + KT * sb, tmem + F::COL_Q + 8 * k, bd, id_s, k > 0);
            }
            mma_commit(smem_u32(&sm.k_empty[st]));
            mma_commit(smem_u32(&sm.s_full[sb]));
          }
          if (t >= 1) {
            const int gu = g + t - 1, st = gu % kStages, pb = gu & 1;
            ok = mbar_wait_or_abort(smem_u32(&sm.v_full[st]), (gu / kStages) & 1, abort_flag);
            ok = ok && mbar_wait_or_abort(smem_u32(&sm.p_full[pb]), (gu >> 1) & 1, abort_flag);
            // the first P V of a unit overwrites O: the previous unit's epilogue has read it
            if (ok && t == 1 && ui > 0) ok = mbar_wait_or_abort(smem_u32(&sm.o_free), (ui - 1) & 1, abort_flag);
            // before a unit's last P V, P V gu-1 has retired (frees the next unit's first S/P buffer)
            if (ok && t == T && gu >= 1) ok = mbar_wait_or_abort(smem_u32(&sm.o_done), (gu - 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            fence_async_smem();
            const uint32_t vb = v_base + st * kTile;
#pragma unroll
            for (int k = 0; k < KT / 16; ++k) {
              // V [keys x dims] is MN-major: 64-dim chunks kChunk apart, 8-key groups 1 KB apart
              const uint64_t bd = sw128_desc(vb + k * 16 * 128, kChunk, 1024);
              mma_bf16_ts(tmem + F::COL_O, tmem + F::COL_S + KT * pb + 8 * k, bd, id_o, (t > 1 || k > 0) ? 1u : 0u);
            }
            mma_commit(smem_u32(&sm.v_empty[st]));
            mma_commit(smem_u32(&sm.o_done));
            if (t == T) mma_commit(smem_u32(&sm.o_full));
          }
        }
        g += T;
        ++ui;
      }
      if (!ok && !*abort_flag) set_abort(sm, status);
      // every MMA issued above has retired before TMEM is freed
      mma_commit(smem_u32(&sm.mma_done));
      if (!mbar_wait(smem_u32(&sm.mma_done), 0)) raise_status(status, DFT_DEV_TIMEOUT);
    }
    __syncwarp();
  } else if (warp >= kProdWarp0) {
    // ------------------------------------------- producers: paged K/V tiles
    constexpr int kPer = KT / 32, kGroups = KT / 16;
    const int pt = tid - kProdWarp0 * 32, pw = warp - kProdWarp0;
    const uint64_t pol_first = l2_evict_first(), pol_keep = l2_evict_normal();
    int g = 0;
    bool ok = true;
    while (ok && next_piece<KT>(sm, P, w, w1, p)) {
      const int T = p.t1 - p.t0;
      if (T == 0) continue;
      const int32_t* idx = a.kv_indices + sm.kv[p.b];
      const uint64_t pol = p.once ? pol_first : pol_keep;
      const int64_t head = (int64_t)p.h * a.kv_sh;
      int s[kPer];  // slots of keys lane + 32 q of a tile; -1 past the request's end
      auto fetch = [&](int tile) {
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int j = tile * KT + 32 * q + lane;
          s[q] = j < p.L ? __ldg(idx + j) : -1;
        }
      };
      fetch(p.t0);
      for (int t = 0; t < T; ++t) {
        const int gt = g + t, st = gt % kStages, j0 = (p.t0 + t) * KT;
        int cur[kPer];
        uint32_t boxes = 0;  // bit i: the 16 slots of group i are consecutive
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int j = j0 + 32 * q + lane;
          cur[q] = s[q];
          if (j < p.L && (cur[q] < 0 || (int64_t)cur[q] >= a.n_slots)) {
            raise_status(status, DFT_DEV_BAD_INDEX);
            cur[q] = 0;
          }
          // keys past the end go along with their group's box
          const int first = __shfl_sync(0xffffffffu, cur[q], lane & 16);
          const uint32_t with = __ballot_sync(
              0xffffffffu, first >= 0 && (int64_t)first + 16 <= a.n_slots && (j >= p.L || cur[q] == first + (lane & 15)));
          boxes |= (with & 0xFFFFu) == 0xFFFFu ? 1u << (2 * q) : 0u;
          boxes |= (with >> 16) == 0xFFFFu ? 2u << (2 * q) : 0u;
        }
        if (t + 1 < T) fetch(p.t0 + t + 1);
        const int live = min(kGroups, (p.L - j0 + 15) / 16);  // groups with a key; the rest stay as they are
        auto load = [&](uint64_t& full, uint64_t& empty, const CUtensorMap& map, const void* cache, uint32_t base) {
          if (gt >= kStages) {
            ok = __all_sync(0xffffffffu,
                            mbar_wait_or_abort(smem_u32(&empty), (gt / kStages - 1) & 1, abort_flag));
            if (!ok) return;
          }
          const uint32_t bar = smem_u32(&full), dst = base + st * kTile;
          if (pt == 0) mbar_expect_tx(bar, __popc(boxes) * 16 * D * 2);
#pragma unroll
          for (int i = 0; i < kGroups; ++i) {
            if (i >= live) break;
            if (boxes >> i & 1) {
              const int row = __shfl_sync(0xffffffffu, cur[i >> 1], (i & 1) * 16);
              if (i % kProdWarps == pw && lane < F::kChunks)
                tma_load_2d(dst + lane * kChunk + i * 2048, &map, p.h * P.x_head + 64 * lane, row + p.h * P.row_head, bar,
                            pol);
              continue;
            }
            constexpr int kUnits = D / 8;  // 16-byte pieces of a row
#pragma unroll
            for (int w0 = 0; w0 < kUnits / 2; w0 += kProdWarps) {  // 32 pieces a warp
              if (w0 + pw >= kUnits / 2) break;
              const int u = (w0 + pw) * 32 + lane, row = u / kUnits, col = u % kUnits, r = 16 * i + row;
              const int slot = __shfl_sync(0xffffffffu, cur[i >> 1], (i & 1) * 16 + row);
              if (j0 + r < p.L)
                cp_async16(dst + (col >> 3) * kChunk + r * 128 + (((uint32_t)(col ^ r) & 7) << 4),
                           static_cast<const unsigned char*>(cache) + (slot * a.kv_st + head) * 2 + col * 16, 16u, pol);
            }
          }
          cp_async_arrive_noinc(bar);
        };
        // a group without a key has first = -1: no box
        load(sm.k_full[st], sm.k_empty[st], k_map, a.k_cache, k_base);
        if (ok) load(sm.v_full[st], sm.v_empty[st], v_map, a.v_cache, v_base);
        if (!ok) {
          g += t;
          break;
        }
      }
      if (ok) g += T;
    }
    if (!ok && lane == 0 && !*abort_flag) set_abort(sm, status);
    // The last copies land before the block's shared memory goes, whatever
    // became of their readers; after an abort tile g may have its K on the way.
    cp_async_wait_all();
    for (int gt = max(0, g - kStages); gt < g; ++gt) {
      mbar_wait(smem_u32(&sm.k_full[gt % kStages]), (gt / kStages) & 1);
      mbar_wait(smem_u32(&sm.v_full[gt % kStages]), (gt / kStages) & 1);
    }
    if (!ok) mbar_wait(smem_u32(&sm.k_full[g % kStages]), (g / kStages) & 1);
  } else {
    // ---------------------- softmax / epilogue: two threads per row, one half each
    constexpr int kCols = KT / 2;           // S columns of a thread
    constexpr int kPk = KT / 4;             // its packed P columns
    constexpr float kBias = BF ? 0.f : 6.f; // float16 P: up to 2^14, so that small weights stay clear of its smallest step
    const int r = (warp & 3) * 32 + lane;   // TMEM lane (query row)
    const int hf = warp >> 2;               // S columns [kCols hf, ..), O / Q columns by halves
    const int pair_bar = 1 + (warp & 3);    // named barrier of warps w and w + 4 (same rows)
    const int wq = warp & 3;
    const int tok = r / P.G, g_ = r - tok * P.G;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const float sc = a.sm_scale * 1.4426950408889634f;
    // a partial slot that no piece of this CTA fills is marked so
    int slots_used = 0;
    // Q row half of a piece -> TMEM (packed, D / 4 columns; spare rows are zero)
    auto load_q = [&](const Piece& u) {
      const bool row_ok = tok < u.ntok;
      const uint4* qrow = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.q) +
                                                         ((int64_t)(u.tok0 + (row_ok ? tok : 0)) * a.q_st +
                                                          (int64_t)(u.h * P.G + (row_ok ? g_ : 0)) * a.q_sh) * 2 +
                                                         hf * D);
#pragma unroll 1
      for (int c = 0; c < D / 4; c += 16) {
        uint32_t v[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4 x = row_ok ? __ldg(qrow + c / 4 + q) : make_uint4(0u, 0u, 0u, 0u);
          v[4 * q] = x.x;
          v[4 * q + 1] = x.y;
          v[4 * q + 2] = x.z;
          v[4 * q + 3] = x.w;
        }
        tmem_st16(tmem + lane_base + F::COL_Q + (D / 4) * hf + c, v);
      }
      tc_fence_before();
      mbar_arrive(smem_u32(&sm.q_ready));
    };
    // pieces without keys give zero rows; true when u then holds a piece with some
    auto next_live = [&](Piece& u) {
      while (next_piece<KT>(sm, P, w, w1, u)) {
        if (u.t1 > u.t0) return true;
        if (tok < u.ntok) {
          uint4* orow = reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.o) +
                                                 ((int64_t)(u.tok0 + tok) * a.o_st + (int64_t)(u.h * P.G + g_) * a.o_sh) * 2 +
                                                 hf * D);
#pragma unroll 4
          for (int q = 0; q < D / 16; ++q) orow[q] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      return false;
    };
    int g = 0, ui = 0;
    // this thread's share of a masked tile's V: rows past the end and non-finite values -> 0
    auto clean_v = [&](const Piece& u, int t, int gt) -> bool {
      constexpr uint32_t kExp = BF ? 0x7F807F80u : 0x7C007C00u, kOne = BF ? 0x00800080u : 0x04000400u;
      const int j0 = (u.t0 + t) * KT, st = gt % kStages;
      const bool got =
          __all_sync(0xffffffffu, mbar_wait_or_abort(smem_u32(&sm.v_full[st]), (gt / kStages) & 1, abort_flag));
      if (!got) {
        if (lane == 0 && !*abort_flag) set_abort(sm, status);
        return false;
      }
      const int live = min(KT, u.L - j0);          // rows of real keys
      const bool scan = u.vis0 < j0 + live;        // some token does not see them all
      unsigned char* vb = smem + (kStages + st) * kTile;
      bool any = false;
#pragma unroll
      for (int c = 0; c < F::kChunks; ++c) {
#pragma unroll
        for (int i = 0; i < KT * 8; i += kSoftmax) {
          uint4* q = reinterpret_cast<uint4*>(vb + c * kChunk) + i + tid;
          if (i + tid >= live * 8) {
            *q = make_uint4(0u, 0u, 0u, 0u);
          } else if (scan) {
            uint4 x = *q;
            // a half's exponent is all ones iff adding one to it carries out
            const uint32_t hit = (((x.x & kExp) + kOne) | ((x.y & kExp) + kOne) | ((x.z & kExp) + kOne) |
                                  ((x.w & kExp) + kOne)) & 0x80008000u;
            if (hit) {
              any = true;
              auto clean = [&](uint32_t& y) { y &= ~(((((y & kExp) + kOne) & 0x80008000u) >> 15) * 0xFFFFu); };
              clean(x.x);
              clean(x.y);
              clean(x.z);
              clean(x.w);
              *q = x;
            }
          }
        }
      }
      if (any) *reinterpret_cast<volatile int*>(&sm.odd[ui & 7]) = ui + 1;
      fence_async_smem();  // these writes before the tensor core's reads
      return true;
    };
    bool more = next_live(p);
    if (more) load_q(p);
    bool ok = true;
    while (ok && more) {
      const Piece u = p;
      const bool row_ok = tok < u.ntok;
      const int T = u.t1 - u.t0;
      const int vis = max(0, min(u.L, u.vis0 + (row_ok ? tok : 0)));  // keys this row sees: j < vis
      const bool busy = wq * 32 < u.ntok * P.G;                       // the warp holds rows
      // A row's two warps meet at the same named barriers in the same order;
      // every early exit is decided from outcomes both have exchanged there.
      float m_used = -INFINITY, l = 0.f;
      bool held = true;  // false: the last tile's V never came; told to the other warp at the next barrier
      for (int t = 0; t < T; ++t) {
        const int gt = g + t, sb = gt & 1;
        const bool got = __all_sync(0xffffffffu, held && mbar_wait_or_abort(smem_u32(&sm.s_full[sb]), (gt >> 1) & 1,
                                                                           abort_flag));
        // keys that every token of the tile sees need no mask (block-uniform)
        const bool plain = (u.t0 + t + 1) * KT <= u.vis0 && (u.t0 + t + 1) * KT <= u.L;
        if (!busy) {  // spare rows: whatever P holds stays in them
          ok = got && (plain || clean_v(u, t, gt));
          if (!ok) break;
          mbar_arrive(smem_u32(&sm.p_full[sb]));
          continue;
        }
        float x[kCols];
        if (got) {
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c) {
            float(&xc)[32] = *reinterpret_cast<float(*)[32]>(&x[32 * c]);
            tmem_ld32(tmem + lane_base + F::COL_S + KT * sb + kCols * hf + 32 * c, xc);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kCols; ++i) x[i] = 0.f;
        }
        const int j0 = (u.t0 + t) * KT + kCols * hf;
        // x stays raw: P = 2^(x sc - m)
        float tmax = -INFINITY;
        if (!plain) {
#pragma unroll
          for (int i = 0; i < kCols; ++i)
            if (j0 + i >= vis) x[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kCols; ++i) tmax = fmaxf(tmax, x[i]);
        tmax *= sc;
        sm.xmax[sb][hf][r] = tmax;
        if (lane == 0) sm.okx[sb][hf][wq] = got;
        // the barrier also orders this half's S reads before the other half's P
        // stores (half 1 writes P over S columns that half 0 reads)
        tc_fence_before();
        named_bar(pair_bar, 64);
        tc_fence_after();
        tmax = fmaxf(tmax, sm.xmax[sb][hf ^ 1][r]);
        ok = got && sm.okx[sb][hf ^ 1][wq];
        if (!ok) break;
        // a row moves its reference max only when the tile max exceeds it by
        // more than 8 (P <= 2^8 otherwise); O then scales by 2^(old - new)
        const bool grow = tmax > m_used + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? tmax : m_used;
          if (t > 0) {
            // O holds P V of this unit's earlier tiles: wait for the last, then rescale this half row
            const bool done = __all_sync(0xffffffffu,
                                         mbar_wait_or_abort(smem_u32(&sm.o_done), (gt - 1) & 1, abort_flag));
            if (lane == 0) sm.okr[sb][hf][wq] = done;
            named_bar(pair_bar, 64);
            ok = done && sm.okr[sb][hf ^ 1][wq];
            if (!ok) break;
            tc_fence_after();
            const float alpha = grow ? ex2(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < D / 64; ++c) {
              float v[32];
              tmem_ld32(tmem + lane_base + F::COL_O + (D / 2) * hf + 32 * c, v);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= alpha;
              tmem_st32(tmem + lane_base + F::COL_O + (D / 2) * hf + 32 * c, v);
            }
            l *= alpha;
          }
          m_used = m_new;
        }
        uint32_t pk[kPk];
        f32x2 sum2 = pk2(0.f, 0.f);
        // a row whose scores so far are all -inf has no reference yet: its P is 0
        const float nm = (m_used == -INFINITY && !plain) ? 0.f : kBias - m_used;
        const f32x2 sc2 = pk2(sc, sc), nm2 = pk2(nm, nm);
#pragma unroll
        for (int i = 0; i < kPk; ++i) {
          float e0, e1;
          upk2(fma2(pk2(x[2 * i], x[2 * i + 1]), sc2, nm2), e0, e1);
          const float p0 = ex2(e0), p1 = ex2(e1);
          sum2 = add2(sum2, pk2(p0, p1));
          pk[i] = pack2<BF>(p0, p1);
        }
        float s0, s1;
        upk2(sum2, s0, s1);
        l += s0 + s1;
        // P (pairs) over columns [kPk hf, kPk hf + kPk) of its own S buffer
#pragma unroll
        for (int c = 0; c < kPk / 16; ++c) {
          const uint32_t(&pc)[16] = *reinterpret_cast<const uint32_t(*)[16]>(&pk[16 * c]);
          tmem_st16(tmem + lane_base + F::COL_S + KT * sb + kPk * hf + 16 * c, pc);
        }
        held = plain || clean_v(u, t, gt);
        tc_fence_before();
        if (held) mbar_arrive(smem_u32(&sm.p_full[sb]));
      }
      if (!ok) break;
      g += T;
      // every S MMA of this unit has been consumed: the next unit's Q may go in
      more = next_live(p);
      if (more) load_q(p);
      // ---- epilogue: wait for this unit's last P V, then O (or its partial) out
      const bool got =
          __all_sync(0xffffffffu, held && mbar_wait_or_abort(smem_u32(&sm.o_full), ui & 1, abort_flag));
      tc_fence_after();
      if (busy) {
        sm.lsum[hf][r] = l;
        if (lane == 0) sm.oke[hf][wq] = got;
        named_bar(pair_bar, 64);
        l = sm.lsum[0][r] + sm.lsum[1][r];
        ok = got && sm.oke[hf ^ 1][wq];
      } else {
        ok = got;
      }
      if (ok && busy) {
        const int64_t prow = ((int64_t)(2 * blockIdx.x + (u.slot < 0 ? 0 : u.slot))) * kRows + r;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        unsigned char* orow = static_cast<unsigned char*>(a.o) +
                              ((int64_t)(u.tok0 + tok) * a.o_st + (int64_t)(u.h * P.G + g_) * a.o_sh) * 2 + hf * D;
        const bool odd = sm.odd[ui & 7] == ui + 1;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          float v[32];
          tmem_ld32(tmem + lane_base + F::COL_O + (D / 2) * hf + 32 * c, v);
          if (odd) {
            // the masked tiles' non-finite values, for the rows that see their keys
            for (int j = max(0, min(u.vis0, u.t1 * KT) / KT * KT); j < min(u.t1 * KT, vis); ++j) {
              if (j < u.t0 * KT) continue;
              const int64_t s = a.kv_indices[sm.kv[u.b] + j];
              if (s < 0 || s >= a.n_slots) continue;
              const uint16_t* vr = static_cast<const uint16_t*>(a.v_cache) + s * a.kv_st + u.h * a.kv_sh + (D / 2) * hf + 32 * c;
              for (int i = 0; i < 32; ++i) {
                const float y = unpack<BF>(vr[i]);
                if (!(fabsf(y) < INFINITY)) {
#pragma unroll
                  for (int e = 0; e < 32; ++e)
                    if (e == i) v[e] += y;
                }
              }
            }
          }
          if (!row_ok) continue;
          if (u.slot < 0) {
            uint4* dst = reinterpret_cast<uint4*>(orow + c * 64);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              dst[q] = make_uint4(pack2<BF>(v[8 * q] * inv, v[8 * q + 1] * inv),
                                  pack2<BF>(v[8 * q + 2] * inv, v[8 * q + 3] * inv),
                                  pack2<BF>(v[8 * q + 4] * inv, v[8 * q + 5] * inv),
                                  pack2<BF>(v[8 * q + 6] * inv, v[8 * q + 7] * inv));
          } else {
            float4* dst = reinterpret_cast<float4*>(P.ws_o + prow * D + (D / 2) * hf + 32 * c);
#pragma unroll
            for (int q = 0; q < 8; ++q) dst[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          }
        }
        if (u.slot >= 0 && hf == 0 && row_ok) {
          P.ws_ml[2 * prow] = m_used;
          P.ws_ml[2 * prow + 1] = l;
        }
      }
      if (ok) {
        if (u.slot >= 0) {
          slots_used |= 1 << u.slot;
          if (tid == 0)
            P.ws_meta[2 * blockIdx.x + u.slot] = make_int4(1 | (u.last ? 2 : 0), u.tok0, u.ntok, u.h);
        }
        // O may now be overwritten by the next unit's first P V
        tc_fence_before();
        mbar_arrive(smem_u32(&sm.o_free));
      }
      ++ui;
    }
    if (tid == 0)
      for (int s = 0; s < 2; ++s)
        if (!(slots_used >> s & 1)) P.ws_meta[2 * blockIdx.x + s] = make_int4(0, 0, 0, 0);
    if (!ok && !*abort_flag) set_abort(sm, status);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kCtlWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Merge the partials of the unit that CTA c begins and leaves unfinished: its
// own, then the continuing slots of the CTAs after it up to the unit's last.
//   o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s
constexpr int kMergeThreads = 256, kMergeY = 8;
template <bool BF, int D>
__global__ void __launch_bounds__(kMergeThreads) chunk_attn_merge(const __grid_constant__ Params P) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kLanes = D / 4, kPass = kMergeThreads / kLanes;
  __shared__ int list[kMergeThreads + 1], flags[kMergeThreads], n_list;
  const int c = blockIdx.x, grid = gridDim.x;
  const int4 meta = P.ws_meta[2 * c + 1];
  if (!(meta.x & 1)) return;
  const dft_chunk_attn_args& a = P.a;
  const int rows = meta.z * P.G, e = threadIdx.x % kLanes;
  if (blockIdx.y * kPass >= rows) return;
  // the unit's partials: slot 2c + 1, then the used even slots after it to the unit's last
  for (int k = threadIdx.x; k < grid; k += kMergeThreads) flags[k] = P.ws_meta[2 * k].x;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    list[n++] = 2 * c + 1;
    for (int k = c + 1; k < grid; ++k) {
      if (flags[k] & 1) list[n++] = 2 * k;
      if (flags[k] & 2) break;
    }
    n_list = n;
  }
  __syncthreads();
  const int n = n_list;
  for (int r = blockIdx.y * kPass + threadIdx.x / kLanes; r < rows; r += kMergeY * kPass) {
    float M = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < n; ++k) M = fmaxf(M, P.ws_ml[2 * ((int64_t)list[k] * kRows + r)]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const int64_t prow = (int64_t)list[k] * kRows + r;
      const float2 ml = reinterpret_cast<const float2*>(P.ws_ml)[prow];
      const float4 v = reinterpret_cast<const float4*>(P.ws_o + prow * D)[e];
      // a sum of 0: the row sees none of these keys (a NaN sum goes on)
      const float wgt = ml.y == 0.f ? 0.f : ex2(ml.x - M);
      acc.x += wgt * v.x;
      acc.y += wgt * v.y;
      acc.z += wgt * v.z;
      acc.w += wgt * v.w;
      L += wgt * ml.y;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int tok = r / P.G;
    unsigned char* orow = static_cast<unsigned char*>(a.o) +
                          ((int64_t)(meta.y + tok) * a.o_st + (int64_t)(meta.w * P.G + (r - tok * P.G)) * a.o_sh) * 2;
    reinterpret_cast<uint2*>(orow)[e] =
        make_uint2(pack2<BF>(acc.x * inv, acc.y * inv), pack2<BF>(acc.z * inv, acc.w * inv));
  }
}

// ------------------------------------------------------------------ host --
using gtile::al16;

int check_args(const dft_chunk_attn_args* a) {
  if (!a || a->B < 0 || a->T < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->n_slots < 0 || a->n_kv < 0)
    return DFT_ERR_INVALID;
  if (a->dtype != DFT_BF16 && a->dtype != DFT_F16) return DFT_ERR_INVALID;
  if (!(a->sm_scale > 0.f) || a->sm_scale > 3e38f) return DFT_ERR_INVALID;
  if ((a->D != 64 && a->D != 128 && a->D != 256) || a->Hq / a->Hkv > 128 || a->B > kMaxB) return DFT_ERR_UNSUPPORTED;
  if (a->B == 0 || a->T == 0) return DFT_OK;
  if (!a->q || !a->o || !a->qo_indptr || !a->kv_indptr || !a->k_cache || !a->v_cache || a->n_slots < 1 ||
      (a->n_kv > 0 && !a->kv_indices))
    return DFT_ERR_INVALID;
  if (!al16(a->q) || !al16(a->o) || !al16(a->k_cache) || !al16(a->v_cache)) return DFT_ERR_UNSUPPORTED;
  if (a->q_st % 8 || a->q_sh % 8 || a->o_st % 8 || a->o_sh % 8 || a->kv_st % 8 || a->kv_sh % 8)
    return DFT_ERR_UNSUPPORTED;
  if (a->q_st < 0 || a->q_sh < 0 || (a->T > 1 && a->o_st < a->D) || (a->Hq > 1 && a->o_sh < a->D) ||
      a->kv_st < a->D || (a->Hkv > 1 && a->kv_sh < a->D))
    return DFT_ERR_INVALID;
  // the cache as rows of one 2-D tensor map: a head is a column offset where a
  // slot's heads lie inside its stride, a row offset where heads are outermost
  const int64_t span = (a->Hkv - 1) * a->kv_sh + a->D;
  if (span > a->kv_st && a->kv_sh % a->kv_st) return DFT_ERR_UNSUPPORTED;
  const int64_t rows = span <= a->kv_st ? a->n_slots : a->n_slots + (a->Hkv - 1) * (a->kv_sh / a->kv_st);
  if (rows > 0x7FFFFFFF || span > 0x7FFFFFFF || a->kv_st >= ((int64_t)1 << 38)) return DFT_ERR_UNSUPPORTED;
  return DFT_OK;
}

// one CTA per SM; the merge keeps a flag per CTA
int grid_size() {
  const int n = gtile::sm_count();
  return n < kMergeThreads ? n : kMergeThreads;
}

struct Workspace {
  int64_t o, ml, meta, total;
};
Workspace workspace(const dft_chunk_attn_args* a, int grid) {
  Workspace w;
  w.meta = 0;
  w.ml = up256(2 * (int64_t)grid * sizeof(int4));
  w.o = w.ml + up256(2 * (int64_t)grid * kRows * 2 * sizeof(float));
  w.total = w.o + 2 * (int64_t)grid * kRows * a->D * sizeof(float);
  return w;
}

bool encode(CUtensorMap* m, const dft_chunk_attn_args* a, const void* base, bool inner) {
  const cuuint64_t dims[2] = {(cuuint64_t)(inner ? (a->Hkv - 1) * a->kv_sh + a->D : a->D),
                              (cuuint64_t)(inner ? a->n_slots : a->n_slots + (a->Hkv - 1) * (a->kv_sh / a->kv_st))};
  const cuuint64_t strides[1] = {(cuuint64_t)a->kv_st * 2};
  const cuuint32_t box[2] = {64, 16}, estr[2] = {1, 1};
  return gtile::encode_fn() &&
         gtile::encode_fn()(m, a->dtype == DFT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF, int D>
int launch(const Params& P, int grid, const CUtensorMap& k_map, const CUtensorMap& v_map, int32_t* status,
           cudaStream_t st) {
  DFT_CUDA_CHECK(cudaFuncSetAttribute(chunk_attn_kernel<BF, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)smem_bytes<D>()));
  chunk_attn_kernel<BF, D><<<(unsigned)grid, kThreads, smem_bytes<D>(), st>>>(k_map, v_map, P, status);
  DFT_LAUNCH_CHECK();
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)grid, kMergeY);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DFT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, chunk_attn_merge<BF, D>, P));
  return DFT_OK;
}

}  // namespace

extern "C" int64_t dft_chunk_attn_workspace_bytes(const dft_chunk_attn_args* a) {
  if (check_args(a)) return -1;
  if (a->B == 0 || a->T == 0) return 0;
  return workspace(a, grid_size()).total;
}

extern "C" int dft_chunk_attn(const dft_chunk_attn_args* a, void* ws, int32_t* dev_status, void* stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  if (a->B == 0 || a->T == 0) return DFT_OK;
  if (!ws || !al16(ws)) return DFT_ERR_INVALID;
  const int grid = grid_size();
  const Workspace w = workspace(a, grid);
  Params P;
  memset(&P, 0, sizeof(P));
  P.a = *a;
  P.G = a->Hq / a->Hkv;
  P.TQ = kRows / P.G;
  const bool inner = (a->Hkv - 1) * a->kv_sh + a->D <= a->kv_st;
  P.x_head = inner ? (int)a->kv_sh : 0;
  P.row_head = inner ? 0 : (int)(a->kv_sh / a->kv_st);
  P.ws_meta = reinterpret_cast<int4*>(static_cast<char*>(ws) + w.meta);
  P.ws_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + w.ml);
  P.ws_o = reinterpret_cast<float*>(static_cast<char*>(ws) + w.o);
  CUtensorMap k_map, v_map;
  if (!encode(&k_map, a, a->k_cache, inner) || !encode(&v_map, a, a->v_cache, inner)) return DFT_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a->dtype == DFT_BF16;
#define DFT_GO(D_) \
  return bf ? launch<true, D_>(P, grid, k_map, v_map, dev_status, st) : launch<false, D_>(P, grid, k_map, v_map, dev_status, st)
  if (a->D == 64) DFT_GO(64);
  if (a->D == 128) DFT_GO(128);
  DFT_GO(256);
#undef DFT_GO
}
