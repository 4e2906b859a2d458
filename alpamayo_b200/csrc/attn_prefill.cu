// attn_prefill.cu — causal attention over packed prompts with grouped heads.
//
//   o_i = sum_{j <= i + Lk - Lq} softmax_j(scale * q_i . k_j) v_j
//
// One warp per (query token, head): the lanes hold D / 32 columns each and
// walk the visible keys with a running maximum and sum.
#include "tc_ptx.cuh"

namespace paro {

struct PrefillParams {
  const void* q;
  const void* k;
  const void* v;
  int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, heads, group;
  int64_t rows, k_rows;
  float scale_log2;
  void* out;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) attn_prefill_kernel(PrefillParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= p.rows * p.heads) return;
  const int64_t row = w / p.heads;
  const int h = (int)(w - row * p.heads), hk = h / p.group;
  int b = 0;
  while (b < p.B && row >= p.cu_q[b + 1]) ++b;
  float o[E] = {}, m = -INFINITY, l = 0.f;
  if (b < p.B) {
    const int64_t lq = p.cu_q[b + 1] - p.cu_q[b], lk = p.cu_k[b + 1] - p.cu_k[b];
    const int64_t see = row - p.cu_q[b] + lk - lq + 1;
    float qf[E];
    for (int e = 0; e < E; ++e)
      qf[e] = to_f32(static_cast<const T*>(p.q)[row * p.sq_t + h * p.sq_h + lane * E + e]) * p.scale_log2;
    for (int64_t j = 0; j < see; ++j) {
      const T* k = static_cast<const T*>(p.k) + (p.cu_k[b] + j) * p.sk_t + hk * p.sk_h + lane * E;
      const T* v = static_cast<const T*>(p.v) + (p.cu_k[b] + j) * p.sv_t + hk * p.sv_h + lane * E;
      float s = 0.f;
      for (int e = 0; e < E; ++e) s = fmaf(qf[e], to_f32(k[e]), s);
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float mn = fmaxf(m, s), a = exp2f(m - mn), e0 = exp2f(s - mn);
      m = mn;
      l = fmaf(l, a, e0);
      for (int e = 0; e < E; ++e) o[e] = fmaf(e0, to_f32(v[e]), o[e] * a);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int e = 0; e < E; ++e) static_cast<T*>(p.out)[(row * p.heads + h) * D + lane * E + e] = from_f32<T>(o[e] * inv);
}

cudaError_t launch_attn_prefill(const void* q, const void* k, const void* v, int dtype, const int64_t* s,
                                const int32_t* cu_q, const int32_t* cu_k, int B, int64_t rows, int64_t k_rows,
                                int heads, int kv_heads, int dim, float scale, void* out, cudaStream_t st) {
  PrefillParams p{q, k, v, s[0], s[1], s[2], s[3], s[4], s[5], cu_q, cu_k, B, heads, heads / kv_heads, rows, k_rows,
                  scale * 1.4426950408889634f, out};
  const int64_t blocks = (rows * heads + 3) / 4;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (dtype == PARO_BF16) {
    if (dim == 128) attn_prefill_kernel<__nv_bfloat16, 128><<<(unsigned)blocks, 128, 0, st>>>(p);
    else attn_prefill_kernel<__nv_bfloat16, 64><<<(unsigned)blocks, 128, 0, st>>>(p);
  } else {
    if (dim == 128) attn_prefill_kernel<__half, 128><<<(unsigned)blocks, 128, 0, st>>>(p);
    else attn_prefill_kernel<__half, 64><<<(unsigned)blocks, 128, 0, st>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace paro
