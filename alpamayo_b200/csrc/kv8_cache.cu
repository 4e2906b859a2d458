// kv8_cache.cu — writing, reading back and compacting the paged int8
// key/value cache (layout: kv8.cuh).
//
// All three kernels move bytes: each reads its inputs once and writes its
// outputs once, a thread holding its share of one (page, head) tile in
// registers between the maximum and the quantisation.
//
//  * append: scale s = max|x| / 127 over the page's tokens of the head,
//    code = rint(x / s).  A page that already holds tokens keeps the larger
//    of its scale and the new one; its codes become rint(code * (old / s)).
//    Every operation is a single correctly rounded float32 one, so the codes
//    do not depend on how the work is split.
//  * gather: code * scale in float32, rounded once to the output type.
//  * compact (eviction's second half): code * scale of the kept tokens,
//    requantised per destination page.
#include "kv8.cuh"

namespace paro {

PARO_DEFINE_ERROR_ACCESSOR(kv8)

namespace {

template <typename T> struct Vec8;   // 8 elements as 16-byte words
template <> struct Vec8<__nv_bfloat16> { uint4 w; };
template <> struct Vec8<__half> { uint4 w; };
template <> struct Vec8<float> { uint4 w[2]; };

__device__ __forceinline__ void load8(Vec8<__nv_bfloat16>& v, const __nv_bfloat16* p) { v.w = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load8(Vec8<__half>& v, const __half* p) { v.w = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load8(Vec8<float>& v, const float* p) {
  v.w[0] = reinterpret_cast<const uint4*>(p)[0];
  v.w[1] = reinterpret_cast<const uint4*>(p)[1];
}
__device__ __forceinline__ void unpack(const Vec8<__nv_bfloat16>& v, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack(const Vec8<__half>& v, float (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v.w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack(const Vec8<float>& v, float (&f)[8]) {
  const float* s = reinterpret_cast<const float*>(v.w);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = s[i];
}

__device__ __forceinline__ void unpack_codes8(uint2 u, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = (float)(int8_t)(u.x >> (8 * i));
    f[4 + i] = (float)(int8_t)(u.y >> (8 * i));
  }
}

__device__ __forceinline__ uint32_t pack4(const int* c) {
  return (uint32_t)(c[0] & 0xff) | ((uint32_t)(c[1] & 0xff) << 8) | ((uint32_t)(c[2] & 0xff) << 16) |
         ((uint32_t)(c[3] & 0xff) << 24);
}

// Block-wide maximum of |x| given as the bits of a non-negative float
// (integers order them, and NaN above infinity, so a NaN shows in the
// result).  `slots`: one word per warp.
__device__ __forceinline__ float block_absmax(uint32_t bits, uint32_t* slots) {
  bits = __reduce_max_sync(0xffffffffu, bits);
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = bits;
  __syncthreads();
  for (int w = 0; w < warps; ++w) bits = max(bits, slots[w]);
  return __uint_as_float(bits);
}

constexpr int kVpt = 4;   // 8-element vectors per thread: page * dim / 32 threads hold a (page, head) tile

}  // namespace

struct AppendParams {
  Kv8View c;
  const void* src[2];          // new keys, values
  int64_t stride_t[2], stride_h[2];
  const int32_t* cu;           // [B + 1] rows of the new tokens
  const int32_t* starts;       // [B] tokens each sequence holds already
  int B;
  int64_t rows;
};

// Grid (touched pages, kv heads, 2: keys / values).  A CTA owns one page's
// tile of one head, so old codes and new tokens meet in its registers.
template <typename T>
__global__ void __launch_bounds__(512) kv8_append_kernel(AppendParams p) {
  __shared__ uint32_t slots[16];
  const Kv8View& c = p.c;
  const int page = 1 << c.page_shift, mask = page - 1;
  auto fresh = [&](int b) { return max(0, p.cu[b + 1] - p.cu[b]); };
  int64_t first = 0;
  const int b = warp_find_seq(blockIdx.x, p.B, [&](int i) -> int64_t {
    const int n = fresh(i);
    return n ? (int64_t)(((p.starts[i] & mask) + (int64_t)n + mask) >> c.page_shift) : 0;
  }, &first);
  if (b < 0) return;
  const int start = p.starts[b], n = fresh(b);
  const int64_t blk = (start >> c.page_shift) + ((int64_t)blockIdx.x - first);
  if (start < 0 || blk >= c.table_width || p.cu[b] < 0 || (int64_t)p.cu[b] + n > p.rows) {
    if (threadIdx.x == 0) report_error(kErrBadPage);
    return;
  }
  const int id = kv8_page(c, b, (int)blk);
  if (id < 0) return;
  const int h = blockIdx.y, which = blockIdx.z;
  const int64_t t0 = blk << c.page_shift;               // first token of the page
  const int old = (int)max((int64_t)0, start - t0);     // its tokens that were there before
  const int end = (int)min((int64_t)page, (int64_t)start + n - t0);
  const int per_tok = c.dim >> 3;                        // vectors per token (8 or 16)
  const T* src = static_cast<const T*>(which ? p.src[1] : p.src[0]);
  const int64_t st = which ? p.stride_t[1] : p.stride_t[0], sh = which ? p.stride_h[1] : p.stride_h[0];
  const int64_t row0 = (int64_t)p.cu[b] + (t0 - start);  // source row of the page's token 0
  int8_t* codes = (which ? c.v_codes : c.k_codes) + kv8_base(c, id, h);
  float* scale_at = (which ? c.v_scale : c.k_scale) + ((int64_t)id * c.kv_heads + h);
  const float prior = old ? *scale_at : 0.f;

  Vec8<T> v[kVpt];
  uint2 prev[kVpt];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x, tok = e / per_tok, d = (e - tok * per_tok) * 8;
    if (tok >= old && tok < end) load8(v[i], src + (row0 + tok) * st + h * sh + d);
    if (tok < old) prev[i] = *reinterpret_cast<const uint2*>(codes + (int64_t)e * 8);
  }
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int tok = (i * blockDim.x + threadIdx.x) / per_tok;
    if (tok >= old && tok < end) {
      float f[8];
      unpack(v[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(fabsf(f[k])));
    }
  }
  float s = __fdiv_rn(block_absmax(top, slots), kKv8Max);
  // every thread read the prior scale before the barrier inside
  // block_absmax, so thread 0 may overwrite it now
  if (old && !(s > prior) && !isnan(s)) s = prior;
  const float ratio = s > 0.f ? __fdiv_rn(prior, s) : 0.f;
  if (threadIdx.x == 0) *scale_at = s;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x, tok = e / per_tok;
    if (tok >= end) continue;
    int q[8];
    if (tok >= old) {
      float f[8];
      unpack(v[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k] = kv8_code(f[k], s);
    } else {
      if (ratio == 1.f) continue;
      float f[8];
      unpack_codes8(prev[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k] = __float2int_rn(__fmul_rn(f[k], ratio));
    }
    *reinterpret_cast<uint2*>(codes + (int64_t)e * 8) = make_uint2(pack4(q), pack4(q + 4));
  }
}

struct GatherParams {
  Kv8View c;
  const int32_t* starts;   // [B] first token of each range
  const int32_t* cu;       // [B + 1] output rows
  int B;
  int64_t rows;
  void* out[2];
};

constexpr int kGatherRows = 16;

// Grid (output rows / 16, 2: keys / values).  One thread turns 8 codes into
// 8 values at a time.
template <typename T>
__global__ void __launch_bounds__(256) kv8_gather_kernel(GatherParams p) {
  const Kv8View& c = p.c;
  __shared__ int s_b;
  const int64_t r0 = (int64_t)blockIdx.x * kGatherRows;
  if (threadIdx.x < 32) {
    int64_t first;
    const int b = warp_find_seq(r0, p.B, [&](int i) -> int64_t { return max(0, p.cu[i + 1] - p.cu[i]); }, &first);
    if (threadIdx.x == 0) s_b = b;
  }
  __syncthreads();
  const int b0 = s_b, which = blockIdx.y;
  const int8_t* codes = which ? c.v_codes : c.k_codes;
  const float* scales = which ? c.v_scale : c.k_scale;
  T* out = static_cast<T*>(which ? p.out[1] : p.out[0]);
  const int per_tok = c.kv_heads * (c.dim >> 3);
  const int rows = (int)min((int64_t)kGatherRows, p.rows - r0);
  for (int e = threadIdx.x; e < rows * per_tok; e += blockDim.x) {
    const int r = e / per_tok, in_tok = e - r * per_tok;
    const int h = in_tok / (c.dim >> 3), d = (in_tok - h * (c.dim >> 3)) * 8;
    const int64_t row = r0 + r;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    int b = b0;
    while (b >= 0 && b < p.B && row >= p.cu[b + 1]) ++b;
    if (b >= 0 && b < p.B) {   // rows past the last sequence read as zeros
      const int64_t tok = (int64_t)p.starts[b] + (row - p.cu[b]);
      const int64_t blk = tok >> c.page_shift;
      if (tok < 0 || blk >= c.table_width) {
        report_error(kErrBadPage);
      } else {
        const int id = kv8_page(c, b, (int)blk);
        if (id >= 0) {
          const float s = scales[(int64_t)id * c.kv_heads + h];
          unpack_codes8(*reinterpret_cast<const uint2*>(codes + kv8_base(c, id, h) +
                                                        (tok & ((1 << c.page_shift) - 1)) * c.dim + d), f);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] *= s;
        }
      }
    }
    T* dst = out + (row * c.kv_heads + h) * c.dim + d;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      T o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = from_f32<T>(f[k]);
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
    }
  }
}

struct EvictParams {
  Kv8View c;
  const float* weights;    // [B][kv_heads][cap]
  int64_t cap;
  const int32_t* lens;     // [B]
  int budget, sink, recent;
  int32_t* kept;           // [B][kv_heads][budget]
  float* new_weights;      // [B][kv_heads][budget]
  int32_t* new_lens;       // [B]
  const int32_t* out_table;  // [B][out_width]
  int out_width;
};

// Integer whose order is the float's: NaN above everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// Block-wide exclusive prefix sum of two 16-bit counts packed in a word;
// *total: their sums.  `slots`: 32 words.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* slots, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  __syncthreads();   // the slots of the previous call have been read
  if (lane == 31) slots[warp] = incl;
  __syncthreads();
  uint32_t w = slots[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += up;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, w, warp) - slots[warp];
  return before + incl - v;
}

// One CTA per (sequence, KV head): radix select (three digits of 11, 11 and
// 10 bits, most significant first) of the smallest key still kept, then one
// ordered pass that writes the kept tokens.
__global__ void __launch_bounds__(kSelThreads) kv8_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t slots[32];
  __shared__ uint32_t s_digit, s_above;
  const int bh = blockIdx.x, b = bh / p.c.kv_heads, tid = threadIdx.x;
  int len = kv8_len(p.c, p.lens[b]);
  const float* w = p.weights + (int64_t)bh * p.cap;
  int32_t* kept = p.kept + (int64_t)bh * p.budget;
  float* nw = p.new_weights + (int64_t)bh * p.budget;
  const int n = min(len, p.budget);
  if (bh % p.c.kv_heads == 0 && tid == 0) p.new_lens[b] = n;
  for (int i = n + tid; i < p.budget; i += kSelThreads) {
    kept[i] = -1;
    nw[i] = 0.f;
  }
  if (len <= p.budget) {
    for (int i = tid; i < n; i += kSelThreads) {
      kept[i] = i;
      nw[i] = w[i];
    }
    return;
  }
  const int lo = p.sink, hi = len - p.recent;   // tokens that compete: lo <= t < hi (len > budget >= sink + recent)
  uint32_t need = p.budget - p.sink - p.recent; // how many of them stay
  uint32_t prefix = 0, known = 0;               // key digits found so far and their mask
  if (need > 0) {
    const int shifts[3] = {21, 10, 0};
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = shifts[pass], digits = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t k = order_key(w[i]);
        if ((k & known) == prefix) atomicAdd(&hist[(k >> shift) & (digits - 1)], 1u);
      }
      __syncthreads();
      // thread i holds digits 2i and 2i + 1 from the top: find where the
      // running count reaches `need`
      const int d0 = digits - 1 - 2 * tid, d1 = d0 - 1;
      const uint32_t c0 = d0 >= 0 ? hist[d0] : 0u, c1 = d1 >= 0 ? hist[d1] : 0u;
      uint32_t incl = c0 + c1;
      const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (lane == 31) slots[warp] = incl;
      __syncthreads();
      uint32_t ws = slots[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, ws, o);
        if (lane >= o) ws += up;
      }
      const uint32_t base = __shfl_sync(0xffffffffu, ws, warp) - slots[warp];
      const uint32_t before = base + incl - c0 - c1;
      if (before < need && before + c0 >= need) {
        s_digit = d0;
        s_above = before;
      } else if (before + c0 < need && before + c0 + c1 >= need) {
        s_digit = d1;
        s_above = before + c0;
      }
      __syncthreads();
      prefix |= s_digit << shift;
      known |= (uint32_t)(digits - 1) << shift;
      need -= s_above;      // still to take among the keys with this prefix
      __syncthreads();
    }
  }
  // ordered pass: keys above `prefix` stay, of those equal to it the first
  // `need`; the low half of a count is the kept tokens, the high half the equal ones
  const uint32_t thr = prefix;
  const bool any = p.budget > p.sink + p.recent;
  uint32_t out = 0, ties = 0;
  for (int base = 0; base < len; base += kSelThreads) {
    const int i = base + tid;
    const float x = i < len ? w[i] : 0.f;
    const bool fixed = i < len && (i < lo || i >= hi);
    const uint32_t k = order_key(x);
    const bool cand = any && i >= lo && i < hi;
    const bool above = fixed || (cand && k > thr), equal = cand && k == thr;
    uint32_t total;
    const uint32_t at = block_scan((above ? 1u : 0u) | (equal ? 0x10000u : 0u), slots, &total);
    // equal tokens before this one that stay: at most `need` in all
    const uint32_t eq_before = ties + (at >> 16);
    const uint32_t taken_before = min(eq_before, need) - min(ties, need);
    const uint32_t pos = out + (at & 0xffffu) + taken_before;
    if (above || (equal && eq_before < need)) {
      kept[pos] = i;
      nw[pos] = x;
    }
    out += (total & 0xffffu) + (min(ties + (total >> 16), need) - min(ties, need));
    ties += total >> 16;
  }
}

// Grid (destination pages per sequence, kv heads, 2 B: keys / values).
__global__ void __launch_bounds__(512) kv8_compact_kernel(EvictParams p) {
  __shared__ uint32_t slots[16];
  __shared__ int64_t s_src[128];
  __shared__ float s_scale[128];
  const Kv8View& c = p.c;
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, h = blockIdx.y, blk = blockIdx.x;
  const int page = 1 << c.page_shift;
  const int n = min(kv8_len(c, p.lens[b]), p.budget);
  const int cnt = min(page, n - blk * page);
  if (cnt <= 0) return;
  const int id = p.out_table[(int64_t)b * p.out_width + blk];
  if (id < 0 || id >= c.num_pages) {
    if (threadIdx.x == 0) report_error(kErrBadPage);
    return;
  }
  const int8_t* codes = which ? c.v_codes : c.k_codes;
  const float* scales = which ? c.v_scale : c.k_scale;
  const int32_t* kept = p.kept + ((int64_t)b * c.kv_heads + h) * p.budget + blk * page;
  for (int t = threadIdx.x; t < cnt; t += blockDim.x) {
    const int tok = kept[t];
    const int src = kv8_page(c, b, tok >> c.page_shift);
    s_src[t] = src < 0 ? -1 : kv8_base(c, src, h) + (int64_t)(tok & (page - 1)) * c.dim;
    s_scale[t] = src < 0 ? 0.f : scales[(int64_t)src * c.kv_heads + h];
  }
  __syncthreads();
  const int per_tok = c.dim >> 3;
  uint2 v[kVpt];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x, tok = e / per_tok, d = (e - tok * per_tok) * 8;
    v[i] = make_uint2(0u, 0u);
    if (tok < cnt && s_src[tok] >= 0) v[i] = *reinterpret_cast<const uint2*>(codes + s_src[tok] + d);
  }
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int tok = (i * blockDim.x + threadIdx.x) / per_tok;
    if (tok < cnt) {
      float f[8];
      unpack_codes8(v[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(fabsf(__fmul_rn(f[k], s_scale[tok]))));
    }
  }
  const float s = __fdiv_rn(block_absmax(top, slots), kKv8Max);
  int8_t* dst = (which ? c.v_codes : c.k_codes) + kv8_base(c, id, h);
  if (threadIdx.x == 0) (which ? c.v_scale : c.k_scale)[(int64_t)id * c.kv_heads + h] = s;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x, tok = e / per_tok;
    if (tok >= cnt) continue;
    float f[8];
    int q[8];
    unpack_codes8(v[i], f);
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = kv8_code(__fmul_rn(f[k], s_scale[tok]), s);
    *reinterpret_cast<uint2*>(dst + (int64_t)e * 8) = make_uint2(pack4(q), pack4(q + 4));
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int tile_threads(const Kv8View& c) { return (c.dim << c.page_shift) / (8 * kVpt); }

cudaError_t launch_kv8_append(const Kv8View& c, const void* k, const void* v, int dtype, const int64_t* strides,
                              const int32_t* cu, const int32_t* starts, int B, int64_t rows, cudaStream_t st) {
  AppendParams p{c, {k, v}, {strides[0], strides[2]}, {strides[1], strides[3]}, cu, starts, B, rows};
  // a sequence's n tokens touch at most n / page + 2 pages, and at most n
  const int64_t items = rows / (1 << c.page_shift) + 2 * (int64_t)B < rows ? rows / (1 << c.page_shift) + 2 * (int64_t)B : rows;
  if (items > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)items, (unsigned)c.kv_heads, 2);
  const int threads = tile_threads(c);
  if (dtype == PARO_BF16) kv8_append_kernel<__nv_bfloat16><<<grid, threads, 0, st>>>(p);
  else if (dtype == PARO_F16) kv8_append_kernel<__half><<<grid, threads, 0, st>>>(p);
  else kv8_append_kernel<float><<<grid, threads, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv8_gather(const Kv8View& c, const int32_t* starts, const int32_t* cu, int B, int64_t rows, void* k,
                              void* v, int dtype, cudaStream_t st) {
  GatherParams p{c, starts, cu, B, rows, {k, v}};
  const int64_t blocks = (rows + kGatherRows - 1) / kGatherRows;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, 2);
  if (dtype == PARO_BF16) kv8_gather_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  else if (dtype == PARO_F16) kv8_gather_kernel<__half><<<grid, 256, 0, st>>>(p);
  else kv8_gather_kernel<float><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv8_evict(const Kv8View& c, const float* weights, int64_t cap, const int32_t* lens, int B,
                             int budget, int sink, int recent, int32_t* kept, float* new_weights, int32_t* new_lens,
                             const int32_t* out_table, int out_width, cudaStream_t st) {
  EvictParams p{c, weights, cap, lens, budget, sink, recent, kept, new_weights, new_lens, out_table, out_width};
  kv8_select_kernel<<<(unsigned)(B * c.kv_heads), kSelThreads, 0, st>>>(p);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  const int blocks = (budget + (1 << c.page_shift) - 1) >> c.page_shift;
  kv8_compact_kernel<<<dim3((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)(2 * B)), tile_threads(c), 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace paro
