// Paged KV cache of the attention layers: page tables and slot maps from
// request lengths, K / V rows written to their slots, and the accepted path's
// rows compacted after a verify.  The reference leaves these to SGLang (the
// req_to_token rows and out_cache_loc behind fc1_branch64.py:31-34, the page
// size 1 plan of fc1_plan.py:16-33); here they are the device-side state that
// dft_tree_attn and dft_chunk_attn read, with no host round trip, so a step
// can be captured once and replayed at any lengths.
#include "dft_common.cuh"

using namespace dft;

namespace {

// ================================================================= plan ==
// Two launches.  plan_kernel is one CTA, a thread per request: needs and
// offsets are four block-wide prefix sums (pages given back, pages taken, new
// tokens, keys), then the page moves, spread over the threads by their flat
// index.  expand_kernel turns the tables into slots over the whole GPU.
constexpr int kMaxB = 1024;
constexpr int kPlanThreads = 1024;

struct PlanShared {
  int64_t warp_sum[4][32];
  int row[kMaxB], need[kMaxB], have[kMaxB];
  int back_off[kMaxB + 1], take_off[kMaxB + 1];
};

// inclusive sum over the CTA of four values at once (64-bit: lengths are the
// caller's and may be anything until they are checked)
__device__ __forceinline__ void block_scan4(int64_t (&v)[4], PlanShared& sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, v[q], d);
      if (lane >= d) v[q] += o;
    }
    if (lane == 31) sm.warp_sum[q][warp] = v[q];
  }
  __syncthreads();
  if (warp < 4) {
    int64_t s = sm.warp_sum[warp][lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += o;
    }
    sm.warp_sum[warp][lane] = s;
  }
  __syncthreads();
  if (warp > 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += sm.warp_sum[q][warp - 1];
  }
}

// the request of flat index i: off is an exclusive sum, off[0] = 0, i < off[n]
__device__ __forceinline__ int owner(const int* off, int n, int i) {
  int lo = 0, hi = n;  // off[lo] <= i < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ dft_page_plan_args a,
                                                            int page_shift, int32_t* status) {
  __shared__ PlanShared sm;
  const int b = threadIdx.x;
  const bool live = b < a.B;
  bool bad = false;
  int64_t cached = 0, fresh = 0, row = 0;
  int have = 0, need = 0;
  const int n_free = *a.n_free;
  if (live) {
    cached = a.cached[b];
    fresh = a.fresh[b];
    row = a.rows ? a.rows[b] : b;
    const int64_t most = (int64_t)a.max_pages << page_shift;
    if (row < 0 || row >= a.n_rows || cached < 0 || fresh < 0 || cached > most || fresh > most - cached) {
      bad = true;
    } else {
      have = a.held[row];
      // written so that no check overflows: have is at most max_pages first
      bad = have < 0 || have > a.max_pages || cached > ((int64_t)have << page_shift);
      need = (int)((cached + fresh + a.page_size - 1) >> page_shift);
    }
    sm.row[b] = bad ? -1 - b : (int)row;
  }
  if (bad) cached = fresh = 0, have = need = 0;
  bad |= n_free < 0 || n_free > a.n_pages;
  int64_t v[4] = {have > need ? have - need : 0, need > have ? need - have : 0, fresh, cached + fresh};
  block_scan4(v, sm);  // also orders sm.row
  int64_t total[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) total[q] = sm.warp_sum[q][31];
  if (live && !bad)
    for (int j = 0; j < b; ++j) bad |= sm.row[j] == (int)row;  // a row named twice
  const int64_t depth = n_free + total[0];  // of the stack once everything is given back
  bad |= depth > a.n_pages || total[2] > a.token_capacity || total[3] > a.kv_capacity || total[3] > 0x7FFFFFFF;
  const bool any_bad = __syncthreads_or(bad);
  const bool short_of_pages = total[1] > depth;
  if (any_bad || short_of_pages) {  // uniform: nothing moves
    if (threadIdx.x == 0) {
      raise_status(status, any_bad ? DFT_DEV_BAD_INDEX : DFT_DEV_NO_PAGES);
      a.qo_indptr[0] = 0;
      a.kv_indptr[0] = 0;
    }
    if (live) {
      a.qo_indptr[b + 1] = 0;
      a.kv_indptr[b + 1] = 0;
    }
    return;
  }
  if (threadIdx.x == 0) {
    sm.back_off[0] = sm.take_off[0] = 0;
    a.qo_indptr[0] = 0;
    a.kv_indptr[0] = 0;
    *a.n_free = (int)(depth - total[1]);  // every thread read it before the barriers above
  }
  if (live) {
    sm.need[b] = need;
    sm.have[b] = have;
    sm.back_off[b + 1] = (int)v[0];
    sm.take_off[b + 1] = (int)v[1];
    a.qo_indptr[b + 1] = (int)v[2];
    a.kv_indptr[b + 1] = (int)v[3];
    a.held[row] = need;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < (int)total[0]; i += kPlanThreads) {
    const int r = owner(sm.back_off, a.B, i);
    a.free_pages[n_free + i] = a.block_table[(int64_t)sm.row[r] * a.bt_sr + sm.need[r] + (i - sm.back_off[r])];
  }
  __syncthreads();  // the pops below may take a page given back above
  for (int i = threadIdx.x; i < (int)total[1]; i += kPlanThreads) {
    const int r = owner(sm.take_off, a.B, i);
    a.block_table[(int64_t)sm.row[r] * a.bt_sr + sm.have[r] + (i - sm.take_off[r])] =
        a.free_pages[(int)depth - 1 - i];
  }
}

// Keys and new tokens to slots, grid-stride over both; the offsets sit in
// shared memory, one binary search per run of four entries.
constexpr int kExpandThreads = 256;

__global__ void __launch_bounds__(kExpandThreads) expand_kernel(const __grid_constant__ dft_page_plan_args a,
                                                                int page_shift, int32_t* status) {
  __shared__ int kv[kMaxB + 1], qo[kMaxB + 1];
  for (int i = threadIdx.x; i <= a.B; i += kExpandThreads) {
    kv[i] = a.kv_indptr[i];
    qo[i] = a.qo_indptr[i];
  }
  __syncthreads();
  const int keys = kv[a.B], tokens = qo[a.B];
  const int in_page = a.page_size - 1;
  const int64_t step = (int64_t)gridDim.x * kExpandThreads * 4;
  bool bad = false;
  auto slot_of = [&](int b, int64_t pos) -> int {
    const int64_t row = a.rows ? a.rows[b] : b;
    const int page = a.block_table[row * a.bt_sr + (pos >> page_shift)];
    const bool ok = page >= 0 && page < a.n_pages;
    bad |= !ok;
    return ok ? (page << page_shift) + (int)(pos & in_page) : -1;
  };
  const int64_t first = ((int64_t)blockIdx.x * kExpandThreads + threadIdx.x) * 4;
  for (int64_t i0 = first; i0 < keys; i0 += step) {
    int b = owner(kv, a.B, (int)i0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + q;
      if (i < keys) {
        while (i >= kv[b + 1]) ++b;
        a.kv_indices[i] = slot_of(b, i - kv[b]);
      }
    }
  }
  for (int64_t i0 = first; i0 < a.token_capacity; i0 += step) {
    int b = i0 < tokens ? owner(qo, a.B, (int)i0) : 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + q;
      if (i < tokens) {
        while (i >= qo[b + 1]) ++b;
        const int64_t pos = a.cached[b] + (i - qo[b]);
        a.slot_map[i] = slot_of(b, pos);
        a.positions[i] = pos;
      } else if (i < a.token_capacity) {
        a.slot_map[i] = -1;
        a.positions[i] = 0;
      }
    }
  }
  if (bad) raise_status(status, DFT_DEV_BAD_INDEX);
}

// =============================================================== append ==
// A copy: each of K and V is read once and written once, V-byte pieces, one
// thread per piece and turn.  Bound by HBM at prompt sizes, by the launch for
// a decode batch.
constexpr int kAppendThreads = 256;

template <typename V>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ dft_kv_append_args a,
                                                                int32_t* status) {
  constexpr int kElems = sizeof(V) / 2;
  const int per_head = a.D / kElems, per_row = a.Hkv * per_head;
  const int64_t pieces = a.T * per_row * 2;
  const uint16_t* src[2] = {static_cast<const uint16_t*>(a.k), static_cast<const uint16_t*>(a.v)};
  uint16_t* dst[2] = {static_cast<uint16_t*>(a.k_cache), static_cast<uint16_t*>(a.v_cache)};
  for (int64_t i = (int64_t)blockIdx.x * kAppendThreads + threadIdx.x; i < pieces;
       i += (int64_t)gridDim.x * kAppendThreads) {
    const int64_t t = i / (2 * per_row);
    int c = (int)(i - t * (2 * per_row));
    const int which = c >= per_row;
    c -= which * per_row;
    const int h = c / per_head, e = (c - h * per_head) * kElems;
    const int64_t slot = a.slot_map[t];
    if (slot < 0) continue;
    if (slot >= a.n_slots) {
      raise_status(status, DFT_DEV_BAD_INDEX);
      continue;
    }
    const int64_t from = which ? t * a.v_st + h * a.v_sh : t * a.k_st + h * a.k_sh;
    *reinterpret_cast<V*>(dst[which] + slot * a.kv_st + h * a.kv_sh + e) =
        *reinterpret_cast<const V*>(src[which] + from + e);
  }
}

// =============================================================== commit ==
// One CTA per (request, layer).  A thread owns columns of the row; it reads
// the path's rows eight at a time before it writes them: path ascends, so
// path[i] >= i and a later read never meets an earlier write.
constexpr int kCommitThreads = 256;
constexpr int kBatch = 8;

template <typename V>
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const __grid_constant__ dft_kv_commit_args a,
                                                                int32_t* status) {
  constexpr int kElems = sizeof(V) / 2;
  __shared__ int64_t src[kMaxNodes], dst[kMaxNodes];
  __shared__ int moves;
  const int b = blockIdx.x, l = blockIdx.y;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int64_t k0 = a.kv_indptr[b], k1 = a.kv_indptr[b + 1];
    const int64_t want = a.accept_len[b];
    const int n = (int)(want < 0 ? 0 : want < a.P ? want : a.P);
    const bool fits = k0 >= 0 && k1 - k0 >= a.N && k1 <= a.n_kv;
    bool bad = !fits;
    int count = 0;  // entries before the first negative one
    int64_t last = -1;
    bool open = true;
    for (int i0 = 0; open && !bad && i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const int64_t p = i < n ? a.path[(int64_t)b * a.P + i] : -1;
      const unsigned stop = __ballot_sync(0xffffffffu, p < 0);
      const int here = stop ? __ffs(stop) - 1 : 32;
      int64_t before = __shfl_up_sync(0xffffffffu, p, 1);
      if (lane == 0) before = last;
      const bool mine = lane < here;
      bad = __any_sync(0xffffffffu, mine && (p >= a.N || p <= before));
      if (!bad && mine) {  // strictly ascending in [0, N): i < N <= kMaxNodes
        const int64_t s = a.kv_indices[k1 - a.N + p], d = a.kv_indices[k1 - a.N + i];
        src[i] = s;
        dst[i] = d;
        bad = s < 0 || s >= a.n_slots || d < 0 || d >= a.n_slots;
      }
      bad = __any_sync(0xffffffffu, bad);
      last = __shfl_sync(0xffffffffu, p, 31);
      count += here;
      open = here == 32;
    }
    if (lane == 0) {
      if (bad) raise_status(status, DFT_DEV_BAD_INDEX);
      moves = bad ? 0 : count;
    }
  }
  __syncthreads();
  const int n = moves;
  const int per_head = a.D / kElems, per_row = a.Hkv * per_head;
  for (int c = threadIdx.x; c < 2 * per_row; c += kCommitThreads) {
    const int which = c >= per_row, cc = c - which * per_row;
    const int h = cc / per_head, e = (cc - h * per_head) * kElems;
    uint16_t* base = static_cast<uint16_t*>(which ? a.v_cache : a.k_cache) + l * a.kv_sl + h * a.kv_sh + e;
    for (int i0 = 0; i0 < n; i0 += kBatch) {
      V v[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (i0 + q < n) v[q] = *reinterpret_cast<const V*>(base + src[i0 + q] * a.kv_st);
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (i0 + q < n && src[i0 + q] != dst[i0 + q]) *reinterpret_cast<V*>(base + dst[i0 + q] * a.kv_st) = v[q];
    }
  }
}

// ------------------------------------------------------------------ host --
bool half_type(int d) { return d == DFT_BF16 || d == DFT_F16; }
bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool al2(const void* p) { return ((uintptr_t)p & 1) == 0; }

}  // namespace

extern "C" int dft_page_plan(const dft_page_plan_args* a, int32_t* dev_status, void* stream) {
  if (!a || a->B < 0 || !a->qo_indptr || !a->kv_indptr || !a->n_free || a->kv_capacity < 0 || a->token_capacity < 0 ||
      a->n_rows < 0 || a->max_pages < 0 || a->n_pages < 0 || a->bt_sr < a->max_pages)
    return DFT_ERR_INVALID;
  if (a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return DFT_ERR_INVALID;
  if (a->B > kMaxB || a->page_size > 1024) return DFT_ERR_UNSUPPORTED;
  if ((int64_t)a->n_pages * a->page_size > 0x7FFFFFFF || (int64_t)a->max_pages * a->page_size > 0x7FFFFFFF)
    return DFT_ERR_UNSUPPORTED;
  if (a->B > 0 && (!a->cached || !a->fresh || !a->held)) return DFT_ERR_INVALID;
  if (a->n_rows > 0 && a->max_pages > 0 && !a->block_table) return DFT_ERR_INVALID;
  if (a->n_pages > 0 && !a->free_pages) return DFT_ERR_INVALID;
  if ((a->kv_capacity > 0 && !a->kv_indices) || (a->token_capacity > 0 && (!a->slot_map || !a->positions)))
    return DFT_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int shift = 0;
  while ((1 << shift) < a->page_size) ++shift;
  plan_kernel<<<1, kPlanThreads, 0, st>>>(*a, shift, dev_status);
  DFT_LAUNCH_CHECK();
  const int64_t most = a->kv_capacity > a->token_capacity ? a->kv_capacity : a->token_capacity;
  int64_t grid = (most + kExpandThreads * 4 - 1) / (kExpandThreads * 4);
  grid = grid < 1 ? 1 : grid > 148 * 4 ? 148 * 4 : grid;
  expand_kernel<<<(unsigned)grid, kExpandThreads, 0, st>>>(*a, shift, dev_status);
  DFT_LAUNCH_CHECK();
  return DFT_OK;
}

extern "C" int dft_kv_append(const dft_kv_append_args* a, int32_t* dev_status, void* stream) {
  if (!a || a->T < 0 || a->Hkv <= 0 || a->D <= 0 || a->n_slots < 0 || !half_type(a->dtype)) return DFT_ERR_INVALID;
  if (a->T == 0) return DFT_OK;
  if (!a->k || !a->v || !a->slot_map || (a->n_slots > 0 && (!a->k_cache || !a->v_cache))) return DFT_ERR_INVALID;
  if (!al2(a->k) || !al2(a->v) || !al2(a->k_cache) || !al2(a->v_cache)) return DFT_ERR_INVALID;
  if ((int64_t)a->Hkv * a->D > (1 << 24) || a->T > ((int64_t)1 << 36)) return DFT_ERR_UNSUPPORTED;
  const bool wide = al16(a->k) && al16(a->v) && al16(a->k_cache) && al16(a->v_cache) && a->D % 8 == 0 &&
                    a->k_st % 8 == 0 && a->k_sh % 8 == 0 && a->v_st % 8 == 0 && a->v_sh % 8 == 0 &&
                    a->kv_st % 8 == 0 && a->kv_sh % 8 == 0;
  const int64_t pieces = a->T * a->Hkv * (wide ? a->D / 8 : a->D) * 2;
  int64_t grid = (pieces + kAppendThreads - 1) / kAppendThreads;
  if (grid > 148 * 32) grid = 148 * 32;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (wide) append_kernel<uint4><<<(unsigned)grid, kAppendThreads, 0, st>>>(*a, dev_status);
  else append_kernel<uint16_t><<<(unsigned)grid, kAppendThreads, 0, st>>>(*a, dev_status);
  DFT_LAUNCH_CHECK();
  return DFT_OK;
}

extern "C" int dft_kv_commit(const dft_kv_commit_args* a, int32_t* dev_status, void* stream) {
  if (!a || a->L < 0 || a->B < 0 || a->N <= 0 || a->P < 0 || a->Hkv <= 0 || a->D <= 0 || a->n_slots < 0 ||
      a->n_kv < 0 || !half_type(a->dtype))
    return DFT_ERR_INVALID;
  if (a->N > kMaxNodes || a->L > 65535 || (int64_t)a->Hkv * a->D > (1 << 24)) return DFT_ERR_UNSUPPORTED;
  if (a->L == 0 || a->B == 0 || a->P == 0) return DFT_OK;
  if (!a->k_cache || !a->v_cache || !a->kv_indptr || !a->path || !a->accept_len || (a->n_kv > 0 && !a->kv_indices))
    return DFT_ERR_INVALID;
  if (!al2(a->k_cache) || !al2(a->v_cache)) return DFT_ERR_INVALID;
  const bool wide = al16(a->k_cache) && al16(a->v_cache) && a->D % 8 == 0 && a->kv_sl % 8 == 0 && a->kv_st % 8 == 0 &&
                    a->kv_sh % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)a->B, (unsigned)a->L);
  if (wide) commit_kernel<uint4><<<grid, kCommitThreads, 0, st>>>(*a, dev_status);
  else commit_kernel<uint16_t><<<grid, kCommitThreads, 0, st>>>(*a, dev_status);
  DFT_LAUNCH_CHECK();
  return DFT_OK;
}
