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
// plan_kernel is one CTA, a thread per request: needs and offsets are four
// block-wide prefix sums (pages given back, pages taken, new tokens, keys), then
// the page moves, spread over the threads by their flat index.  The tables then
// turn into slots: in the same CTA where the maps' capacities are small (a turn
// of its 1024 threads is 4096 entries, about 0.5 us; a second launch costs 2.5),
// else by expand_kernel over the whole GPU.  A batch of 8 takes 4.4 us and 512
// requests of 8 K tokens (4.2 M keys, 17 MB) 13: latency throughout, of a launch,
// the scans' barriers and three loads that wait for one another.
constexpr int kMaxB = 1024;
constexpr int kPlanThreads = 1024;

struct PlanShared {
  int64_t warp_sum[4][32];
  int row[kMaxB], need[kMaxB], have[kMaxB];
  int back_off[kMaxB + 1], take_off[kMaxB + 1];
  int seen[2 * kMaxB];  // hash set of the rows
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

// Keys and new tokens to slots; thread `me` of `all`, four entries a turn with
// one binary search of the offsets (in shared memory).
__device__ __forceinline__ void expand(const dft_page_plan_args& a, int page_shift, const int* kv, const int* qo, int me,
                                       int all, int32_t* status) {
  const int keys = kv[a.B], tokens = qo[a.B];
  const int in_page = a.page_size - 1;
  const int64_t step = (int64_t)all * 4;
  const bool aligned = ((uintptr_t)a.kv_indices & 15) == 0;
  bool bad = false;
  auto slot_of = [&](int b, int64_t pos) -> int {
    const int64_t row = a.rows ? a.rows[b] : b;
    const int page = a.block_table[row * a.bt_sr + (pos >> page_shift)];
    const bool ok = page >= 0 && page < a.n_pages;
    bad |= !ok;
    return ok ? (page << page_shift) + (int)(pos & in_page) : -1;
  };
  for (int64_t i0 = (int64_t)me * 4; i0 < keys; i0 += step) {
    int b = owner(kv, a.B, (int)i0);
    const int64_t pos = i0 - kv[b];
    if (i0 + 3 < kv[b + 1] && page_shift >= 2) {
      // four keys of one request lie in at most two pages
      const int s0 = slot_of(b, pos), s3 = (pos & in_page) + 3 <= in_page ? s0 + 3 * (s0 >= 0) : slot_of(b, pos + 3);
      int s[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool here = (pos & in_page) + q <= in_page;
        s[q] = here ? (s0 < 0 ? -1 : s0 + q) : (s3 < 0 ? -1 : s3 - (3 - q));
      }
      if (aligned) {
        *reinterpret_cast<int4*>(a.kv_indices + i0) = make_int4(s[0], s[1], s[2], s[3]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) a.kv_indices[i0 + q] = s[q];
      }
      continue;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + q;
      if (i < keys) {
        while (i >= kv[b + 1]) ++b;
        a.kv_indices[i] = slot_of(b, i - kv[b]);
      }
    }
  }
  for (int64_t i = me; i < a.token_capacity; i += all) {
    int64_t slot = -1, pos = 0;
    if (i < tokens) {
      const int b = owner(qo, a.B, (int)i);
      pos = a.cached[b] + (i - qo[b]);
      slot = slot_of(b, pos);
    }
    a.slot_map[i] = slot;
    a.positions[i] = pos;
  }
  if (bad) raise_status(status, DFT_DEV_BAD_INDEX);
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ dft_page_plan_args a,
                                                            int page_shift, int solo, int32_t* status) {
  __shared__ PlanShared sm;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // expand_kernel's blocks wait for this grid's end
  const int b = threadIdx.x;
  sm.seen[b] = sm.seen[b + kMaxB] = -1;
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
  block_scan4(v, sm);  // also orders sm.seen
  int64_t total[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) total[q] = sm.warp_sum[q][31];
  if (live && !bad) {  // a row named twice: the second to arrive finds the first
    uint32_t at = (uint32_t)row * 2654435761u >> 21;
    for (int tries = 0; tries < 2 * kMaxB; ++tries, at = (at + 1) & (2 * kMaxB - 1)) {
      const int other = atomicCAS(&sm.seen[at], -1, (int)row);
      if (other == -1) break;
      if (other == (int)row) {
        bad = true;
        break;
      }
    }
  }
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
    if (solo)  // the new tokens' maps still say that there are none
      for (int64_t i = b; i < a.token_capacity; i += kPlanThreads) {
        a.slot_map[i] = -1;
        a.positions[i] = 0;
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
  if (!solo) return;
  // the offsets take the page counts' places
  int* const qo = sm.back_off;
  int* const kv = sm.take_off;
  __syncthreads();
  if (threadIdx.x == 0) qo[0] = kv[0] = 0;
  if (live) {
    qo[b + 1] = (int)v[2];
    kv[b + 1] = (int)v[3];
  }
  __syncthreads();
  expand(a, page_shift, kv, qo, threadIdx.x, kPlanThreads, status);
}

constexpr int kExpandThreads = 256;
constexpr int64_t kSoloEntries = 16384;  // of either map: up to this plan_kernel writes them itself

__global__ void __launch_bounds__(kExpandThreads) expand_kernel(const __grid_constant__ dft_page_plan_args a,
                                                                int page_shift, int32_t* status) {
  __shared__ int kv[kMaxB + 1], qo[kMaxB + 1];
  pdl_wait();
  for (int i = threadIdx.x; i <= a.B; i += kExpandThreads) {
    kv[i] = a.kv_indptr[i];
    qo[i] = a.qo_indptr[i];
  }
  __syncthreads();
  expand(a, page_shift, kv, qo, blockIdx.x * kExpandThreads + threadIdx.x, gridDim.x * kExpandThreads, status);
}

// =============================================================== append ==
// A copy: each of K and V is read once and written once.  A block takes eight
// tokens, a thread columns of the row (K's pieces of V bytes, then V's): where a
// column lies in its head is worked out once, and four tokens' pieces are in
// flight at a time.  Bound by HBM at prompt sizes (10.4 K rows of 2 x 4 x 256,
// 89 MB in all, 10.6 us with K and V in L2, 16 from HBM: 5.6 TB/s), by the launch
// for a decode batch (2.5 us).  A piece per thread and turn, each
// with its divisions and slot load, took 18.7 us.
constexpr int kAppendThreads = 256, kAppendTokens = 8, kAppendBatch = 4;

template <typename V>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ dft_kv_append_args a,
                                                                int32_t* status) {
  constexpr int kElems = sizeof(V) / 2;
  const int per_head = a.D / kElems, per_row = a.Hkv * per_head;
  __shared__ int64_t slots[kAppendTokens];
  for (int64_t t0 = (int64_t)blockIdx.x * kAppendTokens; t0 < a.T; t0 += (int64_t)gridDim.x * kAppendTokens) {
    const int n = (int)min((int64_t)kAppendTokens, a.T - t0);
    __syncthreads();
    if (threadIdx.x < n) {
      const int64_t slot = a.slot_map[t0 + threadIdx.x];
      if (slot >= a.n_slots) raise_status(status, DFT_DEV_BAD_INDEX);
      slots[threadIdx.x] = slot >= a.n_slots ? -1 : slot;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * per_row; c += kAppendThreads) {
      const int which = c >= per_row, cc = c - which * per_row;
      const int h = cc / per_head, e = (cc - h * per_head) * kElems;
      const int64_t step = which ? a.v_st : a.k_st;
      const uint16_t* src = static_cast<const uint16_t*>(which ? a.v : a.k) + t0 * step + h * (which ? a.v_sh : a.k_sh) + e;
      uint16_t* dst = static_cast<uint16_t*>(which ? a.v_cache : a.k_cache) + h * a.kv_sh + e;
#pragma unroll
      for (int i0 = 0; i0 < kAppendTokens; i0 += kAppendBatch) {
        V x[kAppendBatch];
#pragma unroll
        for (int i = 0; i < kAppendBatch; ++i)
          if (i0 + i < n) x[i] = *reinterpret_cast<const V*>(src + (i0 + i) * step);
#pragma unroll
        for (int i = 0; i < kAppendBatch; ++i)
          if (i0 + i < n && slots[i0 + i] >= 0) *reinterpret_cast<V*>(dst + slots[i0 + i] * a.kv_st) = x[i];
      }
    }
  }
}

// =============================================================== commit ==
// One CTA per (request, layer).  A thread owns columns of the row; it reads
// the path's rows eight at a time before it writes them: path ascends, so
// path[i] >= i and a later read never meets an earlier write.  Bound by the
// chain offsets -> path -> slots -> rows, about 4 us; 64 requests of 8 layers
// (50 MB) 9.5 us.
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
  const int64_t most = a->kv_capacity > a->token_capacity ? a->kv_capacity : a->token_capacity;
  const bool solo = most <= kSoloEntries;
  plan_kernel<<<1, kPlanThreads, 0, st>>>(*a, shift, solo, dev_status);
  DFT_LAUNCH_CHECK();
  if (solo) return DFT_OK;
  int64_t grid = (most + kExpandThreads * 4 - 1) / (kExpandThreads * 4);
  if (grid > 148 * 8) grid = 148 * 8;
  // its blocks come up while plan_kernel runs and wait for its end
  return launch_pdl(expand_kernel, dim3((unsigned)grid), dim3(kExpandThreads), 0, st, *a, shift, dev_status);
}

extern "C" int dft_kv_append(const dft_kv_append_args* a, int32_t* dev_status, void* stream) {
  if (!a || a->T < 0 || a->Hkv <= 0 || a->D <= 0 || a->n_slots < 0 || !half_type(a->dtype)) return DFT_ERR_INVALID;
  if (a->T == 0) return DFT_OK;
  if (!a->k || !a->v || !a->slot_map || (a->n_slots > 0 && (!a->k_cache || !a->v_cache))) return DFT_ERR_INVALID;
  if (!al2(a->k) || !al2(a->v) || !al2(a->k_cache) || !al2(a->v_cache)) return DFT_ERR_INVALID;
  if ((int64_t)a->Hkv * a->D > (1 << 24) || a->T > ((int64_t)1 << 36)) return DFT_ERR_UNSUPPORTED;
  if (!rows_apart(a->D, {a->n_slots, a->Hkv}, {a->kv_st, a->kv_sh})) return DFT_ERR_INVALID;
  const bool wide = al16(a->k) && al16(a->v) && al16(a->k_cache) && al16(a->v_cache) && a->D % 8 == 0 &&
                    a->k_st % 8 == 0 && a->k_sh % 8 == 0 && a->v_st % 8 == 0 && a->v_sh % 8 == 0 &&
                    a->kv_st % 8 == 0 && a->kv_sh % 8 == 0;
  int64_t grid = (a->T + kAppendTokens - 1) / kAppendTokens;
  if (grid > 65535 * 16) grid = 65535 * 16;
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
  if (!rows_apart(a->D, {a->L, a->n_slots, a->Hkv}, {a->kv_sl, a->kv_st, a->kv_sh})) return DFT_ERR_INVALID;
  const bool wide = al16(a->k_cache) && al16(a->v_cache) && a->D % 8 == 0 && a->kv_sl % 8 == 0 && a->kv_st % 8 == 0 &&
                    a->kv_sh % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)a->B, (unsigned)a->L);
  if (wide) commit_kernel<uint4><<<grid, kCommitThreads, 0, st>>>(*a, dev_status);
  else commit_kernel<uint16_t><<<grid, kCommitThreads, 0, st>>>(*a, dev_status);
  DFT_LAUNCH_CHECK();
  return DFT_OK;
}
