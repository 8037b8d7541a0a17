// Causal attention of new tokens over the paged KV cache (sm_100a).
//
// Per request b with n new tokens (its rows of q) and L keys, token i and
// q-head hq:  o = softmax_j(q . k_j * sm_scale | j <= L - n + i) . v_j.
//
// One warp per (token, q-head): the lanes split the head's dims, keys in turn,
// running maximum and sum in fp32.
#include "dft_common.cuh"

using namespace dft;

namespace {

constexpr int kMaxB = 1024;

template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_attn_simple(const __grid_constant__ dft_chunk_attn_args a,
                                                         int32_t* status) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.T * a.Hq) return;
  const int t = (int)(w / a.Hq), hq = (int)(w % a.Hq), h = hq / (a.Hq / a.Hkv);
  // the request whose rows hold t
  int b = -1;
  for (int i = lane; i < a.B; i += 32) {
    const int64_t q0 = a.qo_indptr[i], q1 = a.qo_indptr[i + 1], k0 = a.kv_indptr[i], k1 = a.kv_indptr[i + 1];
    if (q0 < 0 || q0 > q1 || q1 > a.T || k0 < 0 || k0 > k1 || k1 > a.n_kv) raise_status(status, DFT_DEV_BAD_INDEX);
    else if (q0 <= t && t < q1) b = i;
  }
  b = __reduce_max_sync(0xffffffffu, b);
  if (b < 0) return;
  const int q0 = a.qo_indptr[b], n = a.qo_indptr[b + 1] - q0;
  const int64_t k0 = a.kv_indptr[b];
  const int L = (int)(a.kv_indptr[b + 1] - k0);
  const int seen = L - n + (t - q0) + 1;
  float q[kPer], o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    q[e] = to_f32(static_cast<const T*>(a.q)[t * a.q_st + hq * a.q_sh + lane * kPer + e]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < seen; ++j) {
    const int slot = a.kv_indices[k0 + j];
    if (slot < 0 || slot >= a.n_slots) {
      if (lane == 0) raise_status(status, DFT_DEV_BAD_INDEX);
      continue;
    }
    const int64_t off = slot * a.kv_st + h * a.kv_sh + lane * kPer;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) x += q[e] * to_f32(static_cast<const T*>(a.k_cache)[off + e]);
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    x *= a.sm_scale;
    const float m_new = fmaxf(m, x), keep = m == m_new ? 1.f : __expf(m - m_new), p = __expf(x - m_new);
    m = m_new;
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = o[e] * keep + p * to_f32(static_cast<const T*>(a.v_cache)[off + e]);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    static_cast<T*>(a.o)[t * a.o_st + hq * a.o_sh + lane * kPer + e] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_args(const dft_chunk_attn_args* a) {
  if (!a || a->B < 0 || a->T < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->n_slots < 0 || a->n_kv < 0)
    return DFT_ERR_INVALID;
  if (a->dtype != DFT_BF16 && a->dtype != DFT_F16) return DFT_ERR_INVALID;
  if (!(a->sm_scale > 0.f) || a->sm_scale > 3e38f) return DFT_ERR_INVALID;
  if ((a->D != 64 && a->D != 128 && a->D != 256) || a->Hq / a->Hkv > 128 || a->B > kMaxB) return DFT_ERR_UNSUPPORTED;
  if (a->B == 0 || a->T == 0) return DFT_OK;
  if (!a->q || !a->o || !a->qo_indptr || !a->kv_indptr) return DFT_ERR_INVALID;
  if ((a->n_kv > 0 && !a->kv_indices) || (a->n_slots > 0 && (!a->k_cache || !a->v_cache))) return DFT_ERR_INVALID;
  if (!al16(a->q) || !al16(a->o) || !al16(a->k_cache) || !al16(a->v_cache)) return DFT_ERR_UNSUPPORTED;
  if (a->q_st % 8 || a->q_sh % 8 || a->o_st % 8 || a->o_sh % 8 || a->kv_st % 8 || a->kv_sh % 8)
    return DFT_ERR_UNSUPPORTED;
  return DFT_OK;
}

template <typename T>
void launch(const dft_chunk_attn_args* a, int32_t* status, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)a->T * a->Hq + 7) / 8);
  if (a->D == 64) chunk_attn_simple<T, 64><<<grid, 256, 0, st>>>(*a, status);
  else if (a->D == 128) chunk_attn_simple<T, 128><<<grid, 256, 0, st>>>(*a, status);
  else chunk_attn_simple<T, 256><<<grid, 256, 0, st>>>(*a, status);
}

}  // namespace

extern "C" int64_t dft_chunk_attn_workspace_bytes(const dft_chunk_attn_args* a) { return check_args(a) ? -1 : 0; }

extern "C" int dft_chunk_attn(const dft_chunk_attn_args* a, void* workspace, int32_t* dev_status, void* stream) {
  const int rc = check_args(a);
  if (rc) return rc;
  if (a->B == 0 || a->T == 0) return DFT_OK;
  (void)workspace;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == DFT_BF16) launch<__nv_bfloat16>(a, dev_status, st);
  else launch<__half>(a, dev_status, st);
  DFT_LAUNCH_CHECK();
  return DFT_OK;
}
