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
//
// 4 heads of 128, bf16: 8192 tokens of six prompts appended in 12 us (25 MB),
// appended and read back in 20 (51 MB); one token of 64 clips in 5, and with
// its pages read back in 11; 64 clips with 262144 tokens cut to 2048 each, and
// read back, in 170 us (614 MB; compaction 78, selection 30); one clip of
// 32768 cut to 4096, and read back, in 34, most of it the selection's chain of
// barriers.
#include <cooperative_groups.h>

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

// (Assembling 2^23 + code with byte permutes instead of converting was
// slower: the read-back of 131072 tokens 82 against 61 us.)
__device__ __forceinline__ void unpack_codes8(uint2 u, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = (float)(int8_t)(u.x >> (8 * i));
    f[4 + i] = (float)(int8_t)(u.y >> (8 * i));
  }
}

// Four elements' codes by division, out of line: 16 of these inline per piece
// of the compaction filled the instruction cache (its largest stall).
__device__ __noinline__ uint32_t codes_div(float a, float b, float c, float d, float scale) {
  return (uint32_t)(kv8_code(a, scale) & 0xff) | ((uint32_t)(kv8_code(b, scale) & 0xff) << 8) |
         ((uint32_t)(kv8_code(c, scale) & 0xff) << 16) | ((uint32_t)(kv8_code(d, scale) & 0xff) << 24);
}

// Codes of N elements under `scale`, as kv8_code gives them, without a
// division each: x times the reciprocal is within 1.6e-5 of the rounded
// quotient (two units in the last place below 128), so both round to the
// same integer unless the product is that close to the middle between two;
// where one is, all N are divided.  Adding 1.5 * 2^23 rounds to an integer
// (ties to even) that stands in the low bits.
struct CodeScale {
  float scale, inv;
  bool slow;       // reciprocal or quotients out of range, zero, not finite
  __device__ __forceinline__ explicit CodeScale(float s) : scale(s) {
    slow = !(s > 1e-30f && s < 1e30f);
    inv = slow ? 0.f : __fdiv_rn(1.f, s);
  }
};
template <int N>
__device__ __forceinline__ void codes_of(const float (&x)[N], const CodeScale& cs, uint32_t (&out)[N / 4]) {
  const float2 inv2 = make_float2(cs.inv, cs.inv), magic = make_float2(12582912.f, 12582912.f);
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    uint32_t q[4];
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const float2 v = make_float2(x[i + k], x[i + k + 1]);
      const float2 z = __ffma2_rn(v, inv2, magic);
      const float2 d = __ffma2_rn(v, inv2, __ffma2_rn(z, make_float2(-1.f, -1.f), magic));   // from the integer
      q[k] = __float_as_uint(z.x);
      q[k + 1] = __float_as_uint(z.y);
      far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
    }
    out[i / 4] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  }
  if (cs.slow || far > 0.49996f) {
#pragma unroll
    for (int i = 0; i < N; i += 4) out[i / 4] = codes_div(x[i], x[i + 1], x[i + 2], x[i + 3], cs.scale);
  }
}

// Codes under `cs` of 16 old codes c under the scale `sc`: those of the
// float32 products c * sc, as codes_of gives them.  c times fl(sc / s) is
// within 3.1e-5 of their rounded quotient.
__device__ __forceinline__ void recodes_of(const float (&c)[16], float sc, const CodeScale& cs, uint32_t (&out)[4]) {
  const float r = __fmul_rn(sc, cs.inv);
  const float2 r2 = make_float2(r, r), magic = make_float2(12582912.f, 12582912.f);
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    uint32_t q[4];
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const float2 v = make_float2(c[i + k], c[i + k + 1]);
      const float2 z = __ffma2_rn(v, r2, magic);
      const float2 d = __ffma2_rn(v, r2, __ffma2_rn(z, make_float2(-1.f, -1.f), magic));   // from the integer
      q[k] = __float_as_uint(z.x);
      q[k + 1] = __float_as_uint(z.y);
      far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
    }
    out[i / 4] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  }
  if (cs.slow || !(far <= 0.4999f) || !(r < 1e30f)) {
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      out[i / 4] = codes_div(__fmul_rn(c[i], sc), __fmul_rn(c[i + 1], sc), __fmul_rn(c[i + 2], sc),
                             __fmul_rn(c[i + 3], sc), cs.scale);
  }
}

// Running maximum of |x|: of 16-bit types as two 16-bit lanes of a word (the
// bits of non-negative floats are ordered as integers, NaN above infinity,
// so a NaN shows in the result), of float32 as a word.
__device__ __forceinline__ uint32_t absmax8(uint32_t top, const uint4& w) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(__vmaxu2(top, w.x & kAbs), __vmaxu2(w.y & kAbs, w.z & kAbs)), w.w & kAbs);
}
__device__ __forceinline__ uint32_t absmax(uint32_t top, const Vec8<__nv_bfloat16>& v) { return absmax8(top, v.w); }
__device__ __forceinline__ uint32_t absmax(uint32_t top, const Vec8<__half>& v) { return absmax8(top, v.w); }
__device__ __forceinline__ uint32_t absmax(uint32_t top, const Vec8<float>& v) {
  constexpr uint32_t kAbs = 0x7fffffffu;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    top = max(max(max(top, v.w[i].x & kAbs), max(v.w[i].y & kAbs, v.w[i].z & kAbs)), v.w[i].w & kAbs);
  return top;
}
// The same as the bits of a float32.
template <typename T> __device__ __forceinline__ uint32_t absmax_f32(uint32_t top);
template <> __device__ __forceinline__ uint32_t absmax_f32<float>(uint32_t top) { return top; }
template <> __device__ __forceinline__ uint32_t absmax_f32<__nv_bfloat16>(uint32_t top) { return max(top & 0xffffu, top >> 16) << 16; }
template <> __device__ __forceinline__ uint32_t absmax_f32<__half>(uint32_t top) {
  return __float_as_uint(fabsf(half_bits_to_f32((uint16_t)max(top & 0xffffu, top >> 16))));
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
  const int id = c.table[(int64_t)b * c.table_width + blk];   // checked below, behind the new tokens' loads
  const int h = blockIdx.y, which = blockIdx.z;
  const int64_t t0 = blk << c.page_shift;               // first token of the page
  const int old = (int)max((int64_t)0, start - t0);     // its tokens that were there before
  const int end = (int)min((int64_t)page, (int64_t)start + n - t0);
  const int tok_shift = c.dim == 128 ? 4 : 3;            // 16 or 8 vectors per token
  const T* src = static_cast<const T*>(which ? p.src[1] : p.src[0]);
  const int64_t st = which ? p.stride_t[1] : p.stride_t[0], sh = which ? p.stride_h[1] : p.stride_h[0];
  const int64_t row0 = (int64_t)p.cu[b] + (t0 - start);  // source row of the page's token 0
  Vec8<T> v[kVpt];
  uint2 prev[kVpt];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x, tok = e >> tok_shift, d = (e - (tok << tok_shift)) * 8;
    if (tok >= old && tok < end) load8(v[i], src + (row0 + tok) * st + h * sh + d);
  }
  if (id < 0 || id >= c.num_pages) {
    if (threadIdx.x == 0) report_error(kErrBadPage);
    return;
  }
  int8_t* codes = (which ? c.v_codes : c.k_codes) + kv8_base(c, id, h);
  float* scale_at = (which ? c.v_scale : c.k_scale) + ((int64_t)id * c.kv_heads + h);
  const float prior = old ? *scale_at : 0.f;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x;
    if (e >> tok_shift < old) prev[i] = *reinterpret_cast<const uint2*>(codes + (int64_t)e * 8);
  }
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int tok = (i * blockDim.x + threadIdx.x) >> tok_shift;
    if (tok >= old && tok < end) top = absmax(top, v[i]);
  }
  float s = __fdiv_rn(block_absmax(absmax_f32<T>(top), slots), kKv8Max);
  // every thread read the prior scale before the barrier inside
  // block_absmax, so thread 0 may overwrite it now
  if (old && !(s > prior) && !isnan(s)) s = prior;
  const float ratio = s > 0.f ? __fdiv_rn(prior, s) : 0.f;
  const CodeScale cs(s);
  if (threadIdx.x == 0) *scale_at = s;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int e = i * blockDim.x + threadIdx.x, tok = e >> tok_shift;
    if (tok >= end) continue;
    float f[8];
    uint32_t q[2];
    if (tok >= old) {
      unpack(v[i], f);
      codes_of(f, cs, q);
    } else {
      if (ratio == 1.f) continue;
      unpack_codes8(prev[i], f);
      int r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = __float2int_rn(__fmul_rn(f[k], ratio));
      q[0] = pack4(r);
      q[1] = pack4(r + 4);
    }
    *reinterpret_cast<uint2*>(codes + (int64_t)e * 8) = make_uint2(q[0], q[1]);
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

constexpr int kGatherRows = 32;
constexpr int kGatherThreads = 256;
constexpr int kGatherFlight = 4;   // pieces of 16 codes in flight per thread

__device__ __forceinline__ void unpack_codes16(const uint4& u, float (&f)[16]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3)));
}

__device__ __forceinline__ uint32_t max_s16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.s16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_s16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.s16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Largest |code| of 16.  As signed 16-bit lanes a word orders by its odd
// bytes, shifted left by 8 by its even ones (the byte below only breaks ties).
__device__ __forceinline__ int code_absmax(const uint4& v) {
  const uint32_t e[4] = {v.x << 8, v.y << 8, v.z << 8, v.w << 8};
  const uint32_t hi = max_s16x2(max_s16x2(max_s16x2(v.x, v.y), max_s16x2(v.z, v.w)),
                                max_s16x2(max_s16x2(e[0], e[1]), max_s16x2(e[2], e[3])));
  const uint32_t lo = min_s16x2(min_s16x2(min_s16x2(v.x, v.y), min_s16x2(v.z, v.w)),
                                min_s16x2(min_s16x2(e[0], e[1]), min_s16x2(e[2], e[3])));
  const int up = max((int)hi >> 24, (int)(hi << 16) >> 24), down = min((int)lo >> 24, (int)(lo << 16) >> 24);
  return max(up, -down);
}

template <typename T>
__device__ __forceinline__ void store16(T* dst, const float (&f)[16]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float4*>(dst)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  } else {
    __align__(16) T o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = from_f32<T>(f[i]);
    reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<const uint4*>(o)[0];
    reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<const uint4*>(o)[1];
  }
}

// Grid (output rows / 32).  One warp finds the rows' tokens; then every
// thread has several pieces of 16 codes of keys and values on their way.
template <typename T>
__global__ void __launch_bounds__(kGatherThreads) kv8_gather_kernel(GatherParams p) {
  const Kv8View& c = p.c;
  __shared__ int s_page[kGatherRows], s_at[kGatherRows];   // page (-1: zeros) and place in it
  const int64_t r0 = (int64_t)blockIdx.x * kGatherRows;
  if (threadIdx.x < 32) {
    int64_t first;
    // the sequence of the first row here, or the first with rows behind it
    const int64_t into = max((int64_t)0, r0 - p.cu[0]);
    int b = warp_find_seq(into, p.B, [&](int i) -> int64_t { return max(0, p.cu[i + 1] - p.cu[i]); }, &first);
    const int64_t row = r0 + threadIdx.x;
    int page = -1, at = 0;
    while (b >= 0 && b < p.B && row >= p.cu[b + 1]) ++b;
    if (row < p.rows && b >= 0 && b < p.B && row >= p.cu[b]) {   // rows outside the sequences read as zeros
      const int64_t tok = (int64_t)p.starts[b] + (row - p.cu[b]), blk = tok >> c.page_shift;
      if (tok < 0 || blk >= c.table_width) report_error(kErrBadPage);
      else page = kv8_page(c, b, (int)blk);
      at = (int)(tok & ((1 << c.page_shift) - 1));
    }
    s_page[threadIdx.x] = page;
    s_at[threadIdx.x] = at;
  }
  __syncthreads();
  const int head_shift = c.dim == 128 ? 3 : 2, per_tok = c.kv_heads << head_shift;   // pieces of a head, of a token
  const int rows = (int)min((int64_t)kGatherRows, p.rows - r0), side = rows * per_tok;
  for (int e0 = threadIdx.x; e0 < 2 * side; e0 += kGatherFlight * kGatherThreads) {
    uint4 w[kGatherFlight];
    float s[kGatherFlight];
#pragma unroll
    for (int x = 0; x < kGatherFlight; ++x) {
      const int e = e0 + x * kGatherThreads;
      w[x] = make_uint4(0u, 0u, 0u, 0u);
      s[x] = 0.f;
      if (e < 2 * side) {
        const int which = e >= side, i = e - (which ? side : 0), r = i / per_tok, in_tok = i - r * per_tok;
        const int h = in_tok >> head_shift, d = (in_tok - (h << head_shift)) * 16, page = s_page[r];
        if (page >= 0) {
          w[x] = *reinterpret_cast<const uint4*>((which ? c.v_codes : c.k_codes) + kv8_base(c, page, h) + s_at[r] * c.dim + d);
          s[x] = (which ? c.v_scale : c.k_scale)[(int64_t)page * c.kv_heads + h];
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kGatherFlight; ++x) {
      const int e = e0 + x * kGatherThreads;
      if (e >= 2 * side) break;
      const int which = e >= side;
      float f[16];
      unpack_codes16(w[x], f);
#pragma unroll
      for (int k = 0; k < 16; ++k) f[k] *= s[x];
      // a row's pieces are contiguous: [row][head][dim]
      store16(static_cast<T*>(which ? p.out[1] : p.out[0]) + (r0 * per_tok + (e - (which ? side : 0))) * 16, f);
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

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelFlight = 8;      // weights in flight per thread
constexpr int kSelCached = 40960;  // keys of a CTA kept in shared memory, at most
constexpr int kSelBins = 2048;

// One cluster of CTAs per (sequence, KV head), each CTA with a run of its
// tokens: radix select (three digits of 11, 11 and 10 bits, most significant
// first) of the smallest key still kept, on the sum of the CTAs' counts, then
// an ordered pass: every warp counts its own run of tokens, the counts are
// added up across warps and CTAs, and the warps write.  The keys are read
// from global memory once and kept in shared memory as far as they fit
// (`cached`, from the front of the CTA's run).  Bound by one SM's instruction
// rate where there are few (sequence, head)s: 32768 tokens of 4 heads took
// 42 us on one CTA each.
__global__ void __launch_bounds__(kSelThreads) kv8_select_kernel(EvictParams p, int cached, int with_masks) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t keys[];           // [cached] keys, then two words per 32 tokens of the CTA's run
  __shared__ __align__(16) uint32_t hist[3][kSelBins];
  __shared__ uint32_t slots[kSelWarps], slots2[kSelWarps];
  __shared__ uint32_t s_digit, s_above, s_total[2];
  const cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int bh = blockIdx.x / cs, b = bh / p.c.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = kv8_len(p.c, p.lens[b]);
  const float* w = p.weights + (int64_t)bh * p.cap;
  int32_t* kept = p.kept + (int64_t)bh * p.budget;
  float* nw = p.new_weights + (int64_t)bh * p.budget;
  const int n = min(len, p.budget);
  if (bh % p.c.kv_heads == 0 && rank == 0 && tid == 0) p.new_lens[b] = n;
  for (int i = n + rank * kSelThreads + tid; i < p.budget; i += cs * kSelThreads) {
    kept[i] = -1;
    nw[i] = 0.f;
  }
  if (len <= p.budget) {
    for (int i = rank * kSelThreads + tid; i < n; i += cs * kSelThreads) {
      kept[i] = i;
      nw[i] = w[i];
    }
    return;
  }
  const int lo = p.sink, hi = len - p.recent;   // tokens that compete: lo <= t < hi (len > budget >= sink + recent)
  uint32_t need = p.budget - p.sink - p.recent; // how many of them stay
  const bool any = need > 0;
  // this CTA's tokens, and inside it each warp's
  const int slice = (len + cs * 32 - 1) / (cs * 32) * 32, a0 = min(len, rank * slice), a1 = min(len, a0 + slice);
  const int run = (slice + 32 * kSelWarps - 1) / (32 * kSelWarps) * 32;
  const int t0 = min(a1, a0 + warp * run), t1 = min(a1, t0 + run);
  uint32_t* masks = keys + cached;
  uint32_t prefix = 0, known = 0;               // key digits found so far and their mask
  if (any) {
    for (int i = tid; i < 3 * kSelBins; i += kSelThreads) hist[0][i] = 0;
    __syncthreads();
  }
  for (int pass = 0; pass < 3 && any; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, digits = pass == 2 ? 1024 : kSelBins;
    const int from = max(a0, lo), to = min(a1, hi);
    for (int i0 = from + tid; i0 < to; i0 += kSelFlight * kSelThreads) {
      uint32_t k[kSelFlight];
#pragma unroll
      for (int x = 0; x < kSelFlight; ++x) {
        const int i = i0 + x * kSelThreads;
        if (i < to) k[x] = pass > 0 && i - a0 < cached ? keys[i - a0] : order_key(w[i]);
      }
#pragma unroll
      for (int x = 0; x < kSelFlight; ++x) {
        const int i = i0 + x * kSelThreads;
        if (i < to) {
          if (pass == 0 && i - a0 < cached) keys[i - a0] = k[x];
          if ((k[x] & known) == prefix) atomicAdd(&hist[pass][(k[x] >> shift) & (digits - 1)], 1u);
        }
      }
    }
    cluster.sync();
    // thread i holds the four digits from 4 i below the top on: find where
    // the running count reaches `need`
    const int d0 = digits - 4 - 4 * tid;
    uint32_t cnt[4] = {0u, 0u, 0u, 0u};         // from the highest digit down
    if (d0 >= 0)
      for (int r = 0; r < cs; ++r) {
        const uint4 v = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&hist[pass][d0], r));
        cnt[0] += v.w;
        cnt[1] += v.z;
        cnt[2] += v.y;
        cnt[3] += v.x;
      }
    const uint32_t mine = cnt[0] + cnt[1] + cnt[2] + cnt[3];
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) slots[warp] = incl;
    __syncthreads();
    uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? slots[lane] : 0u) + incl - mine;
    if (before < need && before + mine >= need) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (before < need && before + cnt[x] >= need) {
          s_digit = d0 + 3 - x;
          s_above = before;
          before = need;   // found
        } else {
          before += cnt[x];
        }
      }
    }
    __syncthreads();
    prefix |= s_digit << shift;
    known |= (uint32_t)(digits - 1) << shift;
    need -= s_above;      // still to take among the keys with this prefix
    __syncthreads();
  }
  // Keys above `prefix` stay, of those equal to it the first `need`.
  // masks of the 32 tokens from i0 on that stay, and that are equal to the last kept
  auto judge = [&](int i0) {
    const int i = i0 + lane;
    bool stays = i < t1 && (i < lo || i >= hi), tie = false;
    if (any && i < t1 && !stays) {
      const uint32_t k = i - a0 < cached ? keys[i - a0] : order_key(w[i]);
      stays = k > prefix;
      tie = k == prefix;
    }
    return make_uint2(__ballot_sync(0xffffffffu, stays), __ballot_sync(0xffffffffu, tie));
  };
  uint32_t above = 0, equal = 0;
#pragma unroll 4
  for (int i0 = t0; i0 < t1; i0 += 32) {
    const uint2 m = judge(i0);
    above += __popc(m.x);
    equal += __popc(m.y);
    if (with_masks && lane == 0) *reinterpret_cast<uint2*>(masks + (i0 - a0) / 32 * 2) = m;
  }
  if (lane == 0) {
    slots[warp] = above;
    slots2[warp] = equal;
  }
  __syncthreads();
  uint32_t out = __reduce_add_sync(0xffffffffu, lane < warp ? slots[lane] : 0u);
  uint32_t ties = __reduce_add_sync(0xffffffffu, lane < warp ? slots2[lane] : 0u);
  if (tid == kSelThreads - 1) {
    s_total[0] = out + above;
    s_total[1] = ties + equal;
  }
  cluster.sync();
  uint32_t out_cta = 0, ties_cta = 0;
  if (lane < rank) {
    const uint32_t* o = cluster.map_shared_rank(s_total, lane);
    out_cta = o[0];
    ties_cta = o[1];
  }
  out += __reduce_add_sync(0xffffffffu, out_cta);
  ties += __reduce_add_sync(0xffffffffu, ties_cta);
  out += min(ties, need);
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
  for (int i0 = t0; i0 < t1; i0 += 32) {
    const uint2 m = with_masks ? *reinterpret_cast<const uint2*>(masks + (i0 - a0) / 32 * 2) : judge(i0);
    const uint32_t tie_at = ties + __popc(m.y & below);
    const uint32_t taken = min(tie_at, need) - min(ties, need);   // equal ones before this lane that stay
    if ((m.x >> lane & 1u) || ((m.y >> lane & 1u) && tie_at < need)) {
      const uint32_t pos = out + __popc(m.x & below) + taken;
      kept[pos] = i0 + lane;
      nw[pos] = w[i0 + lane];
    }
    const uint32_t ties_after = ties + __popc(m.y);
    out += __popc(m.x) + min(ties_after, need) - min(ties, need);
    ties = ties_after;
  }
  cluster.sync();          // the other CTAs have read this one's counts
}

// One task per (destination page, keys or values, head, sequence), taken by
// a team of as many warps as its pieces of 16 codes need at 8 to a lane, all
// of them in flight at once.  With a block of 256 threads per task, an index
// list in shared memory and two barriers, the same work took 90 us instead of
// 78 for 64 sequences cut to 2048 tokens (warps in blocks of 128: 89, of 512:
// 107; teams that walk the tasks with the grid's stride: 117).
constexpr int kCmpThreads = 256;
constexpr int kCmpPieces = 8;

template <int D>
__global__ void __launch_bounds__(kCmpThreads) kv8_compact_kernel(EvictParams p, int pages) {
  constexpr int kShift = D == 128 ? 3 : 2;       // 8 or 4 pieces per token
  constexpr int kTok = kCmpPieces >> kShift;     // tokens per lane
  constexpr int kPer = 32 >> kShift;             // tokens per piece index
  __shared__ uint32_t s_top[kCmpThreads / 32];
  const Kv8View& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int page = 1 << c.page_shift;
  // log2 of the warps to a task: 1, 2 or 4 of them
  const int team_shift = max(0, c.page_shift + kShift - 8), team = 1 << team_shift;
  static_assert(32 * kCmpPieces == 256, "2^8 pieces to a warp");
  const int task = (blockIdx.x * (kCmpThreads / 32) + warp) >> team_shift, which = task & 1, blk = task >> 1;
  const int h = blockIdx.y, b = blockIdx.z, bh = b * c.kv_heads + h;
  int cnt = 0, id = -1;
  if (blk < pages) {
    id = p.out_table[(int64_t)b * p.out_width + blk];
    cnt = min(page, min(kv8_len(c, p.lens[b]), p.budget) - blk * page);
    if (cnt > 0 && (id < 0 || id >= c.num_pages)) {
      report_error(kErrBadPage);
      cnt = 0;
    }
  }
  const int share = page >> team_shift, first = (warp & (team - 1)) * share;             // this warp's tokens of the page
  const int mine = max(0, min(share, cnt - first));
  const float* scales = which ? c.v_scale : c.k_scale;
  const int8_t* codes = which ? c.v_codes : c.k_codes;
  // lane l knows the source rows of the warp's tokens l, l + 32, ...
  int src_page[kTok], src_at[kTok];
  float src_scale[kTok];
#pragma unroll
  for (int x = 0; x < kTok; ++x) {
    const int t = x * 32 + lane;
    src_at[x] = t < mine ? p.kept[(int64_t)bh * p.budget + blk * page + first + t] : 0;
  }
#pragma unroll
  for (int x = 0; x < kTok; ++x) {
    src_page[x] = x * 32 + lane < mine ? kv8_page(c, b, src_at[x] >> c.page_shift) : -1;
    src_at[x] &= page - 1;
  }
#pragma unroll
  for (int x = 0; x < kTok; ++x)
    src_scale[x] = src_page[x] >= 0 ? scales[(int64_t)src_page[x] * c.kv_heads + h] : 0.f;
  // piece i of a lane belongs to token (i * 32 + lane) >> kShift, known to
  // lane (token & 31) as its token x(i)
  auto owner = [&](int i) { return ((i * 32 + lane) >> kShift) & 31; };
  uint4 v[kCmpPieces];
#pragma unroll
  for (int i = 0; i < kCmpPieces; ++i) {
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (i * kPer >= share) continue;
    const int x = i * kPer / 32;
    const int pg = __shfl_sync(0xffffffffu, src_page[x], owner(i)), at = __shfl_sync(0xffffffffu, src_at[x], owner(i));
    if (pg >= 0)
      v[i] = *reinterpret_cast<const uint4*>(codes + kv8_base(c, pg, h) + at * D + (lane & ((1 << kShift) - 1)) * 16);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kCmpPieces; ++i) {
    if (i * kPer >= share) break;
    const float sc = __shfl_sync(0xffffffffu, src_scale[i * kPer / 32], owner(i));
    // |code * scale| is largest where |code| is
    top = max(top, __float_as_uint(fabsf(__fmul_rn((float)code_absmax(v[i]), sc))));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (team > 1) {
    if (lane == 0) s_top[warp] = top;
    named_barrier(1 + (warp >> team_shift), 32 * team);
    for (int x = 0; x < team; ++x) top = max(top, s_top[(warp & ~(team - 1)) + x]);
  }
  if (cnt <= 0) return;
  const float s = __fdiv_rn(__uint_as_float(top), kKv8Max);
  const CodeScale cs(s);
  int8_t* dst = (which ? c.v_codes : c.k_codes) + kv8_base(c, id, h) + (int64_t)first * D;
  if (lane == 0 && first == 0) (which ? c.v_scale : c.k_scale)[(int64_t)id * c.kv_heads + h] = s;
#pragma unroll
  for (int i = 0; i < kCmpPieces; ++i) {
    if (i * kPer >= share) break;
    const float sc = __shfl_sync(0xffffffffu, src_scale[i * kPer / 32], owner(i));
    float f[16];
    uint32_t q[4];
    unpack_codes16(v[i], f);
    recodes_of(f, sc, cs, q);
    if ((i * 32 + lane) >> kShift < mine)
      *reinterpret_cast<uint4*>(dst + (int64_t)(i * 32 + lane) * 16) = make_uint4(q[0], q[1], q[2], q[3]);
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Threads that hold a (page, head) tile, kVpt vectors of 8 elements each.
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
  if (dtype == PARO_BF16) kv8_gather_kernel<__nv_bfloat16><<<(unsigned)blocks, kGatherThreads, 0, st>>>(p);
  else if (dtype == PARO_F16) kv8_gather_kernel<__half><<<(unsigned)blocks, kGatherThreads, 0, st>>>(p);
  else kv8_gather_kernel<float><<<(unsigned)blocks, kGatherThreads, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv8_evict(const Kv8View& c, const float* weights, int64_t cap, const int32_t* lens, int B,
                             int budget, int sink, int recent, int32_t* kept, float* new_weights, int32_t* new_lens,
                             const int32_t* out_table, int out_width, cudaStream_t st) {
  EvictParams p{c, weights, cap, lens, budget, sink, recent, kept, new_weights, new_lens, out_table, out_width};
  // CTAs to a (sequence, head): as many as the GPU holds at once (two to an
  // SM, by registers), at most 8
  int cs = 1;
  while (cs < 8 && (int64_t)B * c.kv_heads * cs * 2 <= 2 * sm_count()) cs *= 2;
  // as many keys in shared memory as a CTA can get, up to 160 KB of them,
  // and the masks of its run (8 bytes per 32 tokens) up to 40 KB; a longer
  // run makes them twice
  const int64_t most = (((int64_t)c.table_width << c.page_shift) + cs * 32 - 1) / (cs * 32) * 32;
  const int cached = (int)(most < kSelCached ? most : kSelCached);
  const int with_masks = most / 32 * 8 <= 40 * 1024;
  const int64_t smem = (int64_t)cached * 4 + (with_masks ? most / 32 * 8 : 0);
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kv8_select_kernel), (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * c.kv_heads * cs));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cs, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, kv8_select_kernel, p, cached, with_masks)) != cudaSuccess) return e;
  const int blocks = (budget + (1 << c.page_shift) - 1) >> c.page_shift;
  const int pieces = (c.dim << c.page_shift) / 16, team = pieces > 32 * kCmpPieces ? pieces / (32 * kCmpPieces) : 1;
  const int64_t ctas = ((int64_t)blocks * 2 * team + kCmpThreads / 32 - 1) / (kCmpThreads / 32);
  const dim3 grid((unsigned)ctas, (unsigned)c.kv_heads, (unsigned)B);
  if (c.dim == 128) kv8_compact_kernel<128><<<grid, kCmpThreads, 0, st>>>(p, blocks);
  else kv8_compact_kernel<64><<<grid, kCmpThreads, 0, st>>>(p, blocks);
  return cudaGetLastError();
}

}  // namespace paro
