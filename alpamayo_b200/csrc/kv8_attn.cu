// kv8_attn.cu — attention of the newest 1..T tokens of each sequence over
// the paged int8 cache (layout: kv8.cuh).
//
//   o_r = sum_t p_rt vs_t V_t,  p_rt = softmax_t(scale * ks_t * q_r . K_t)
//
// over the tokens t that row r = (new token i, query head) may see
// (t <= len - T + i); ks_t, vs_t are the scales of t's page.
//
// Bound by the cache's bytes: 2 * dim per token and KV head, each read once
// for all the query heads that share the head.  The work is cut into units
// of 32 tokens of one (sequence, KV head); the grid's CTAs take equal runs
// of consecutive units (the lengths are read on the device), so ragged
// lengths and few long sequences balance alike.  Inside a CTA teams of 1, 2 or
// 4 warps (16 query rows each) take units in turn, each team with its own
// ring of cp.async stages, laid out so that a lane reads back the 16-byte
// places of its own lane number: no bank conflicts, and for teams of one
// warp no barrier between the copy and its use.  The page table is read a
// unit ahead of the copies.
//
// The products run on mma.sync m16n8k16 in fp16 with float32 sums: int8
// codes are exact in fp16, q is scaled per row by a power of two to fill
// fp16's range, the page scales enter in float32.  The probabilities are
// rounded to fp16 (11 bits, finer than the bf16 output) after a power-of-two
// shift that keeps them normal 29 binades below the row's largest term: the
// running maximum M is of score + e_t, with 2^e_t the power of two below
// vs_t, so the rounded value exp2(score + e_t - M + 14) * (vs_t / 2^e_t)
// stays below 2^15 whatever the page scales are (e_t is kept within -60 and
// 121: a page of smaller values loses bits, and no finite input has a scale of
// 2^122).  The denominator keeps the unrounded float32 terms, but
// for those of pages whose scale (2^-60 for a page of zeros) is below 2^-126
// of the largest.
//
// A CTA that meets the end of its run inside a (sequence, head) leaves a
// partial (M, sum, weighted values) that the second kernel joins; that
// kernel also turns the stored scores into softmax weights where the caller
// accumulates them, one writer per element, so every result is independent
// of timing.
//
// A page that the table does not have in the pool is copied from page 0 with
// key scales of zero, and minus infinity is added to its scores.  A row that
// sees a token has a finite maximum, whatever its scores are: it tells a row
// of nothing but minus infinity (NaN) from one that sees nothing (zeros).
//
// 28 query over 4 key/value heads of 128, bf16: one clip of 131072 tokens 42 us
// (134 MB, 3.2 TB/s over all, some 5 in the steady part: 8 us go into start-up
// and join), 64 clips with 262144 tokens and weights 90 us (278 MB; first
// kernel 74, join 16), one clip of 300 tokens 10 us; 8 verify tokens of 8
// clips with 32000, fp16, 50 us.  Bound by the instructions per unit (some
// 820, 12 warps per SM), and with many rows by mma.sync and the widening.
#include <cfloat>

#include "kv8.cuh"

namespace paro {

PARO_DEFINE_ERROR_ACCESSOR(kv8a)

constexpr int kDecWarps = 4;
constexpr int kUnit = 32;         // tokens per unit
constexpr int kMinUnits = 4;      // least units per CTA: one per warp
constexpr float kPShift = 14.f;   // probabilities are kept as multiples of 2^-14 below the maximum

struct DecodeParams {
  Kv8View c;
  const void* q;               // [B][T][heads][dim]
  int64_t q_sb, q_st, q_sh;    // element strides
  void* out;                   // [B][T][heads][dim], contiguous
  const int32_t* lens;
  int B, T, heads, group;      // group = heads / kv_heads
  int rows;                    // T * group
  float scale_log2;            // softmax scale * log2(e)
  int ctas;                    // grid.x of the first kernel
  // workspace
  float* part_o;               // [row blocks][slots][RB][dim]
  float2* part_ml;             // [row blocks][slots][RB] (M, sum)
  int slots;                   // B * kv_heads + ctas
  int lanes, out_blocks;       // second kernel: threads per output column group, blocks of output rows,
  int row_groups;              // threads that share a weight's rows
  int2* range;                 // [B * kv_heads] first and last CTA with a partial
  float* scores;               // [B * kv_heads][rows][score_cap] log2-scaled scores, or null
  int64_t score_cap;
  const float* weights;        // [B][kv_heads][cap] or null
  float* weights_out;
  int64_t cap;
};

namespace {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t dst, float x) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst), "f"(x) : "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two code bytes (biased by 128, in bytes `sel`) as two exact fp16 values:
// 0x64uu is 1024 + u.
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t biased, uint32_t sel) {
  const uint32_t w = __byte_perm(biased, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6480)));  // 1152
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Units of sequence b per KV head.  All sequences' units together fit 31
// bits (the launch refuses more).
__device__ __forceinline__ int seq_units(const DecodeParams& p, int b) {
  const int cap = p.c.table_width << p.c.page_shift;
  return (int)(((unsigned)max(0, min(p.lens[b], cap)) + kUnit - 1) / kUnit);
}

// Units per CTA; *total: units of all sequences and heads.
__device__ __forceinline__ int units_per_cta(const DecodeParams& p, int* total) {
  int u = 0;
  for (int b = threadIdx.x & 31; b < p.B; b += 32) u += seq_units(p, b);
  u = __reduce_add_sync(0xffffffffu, u) * p.c.kv_heads;
  *total = u;
  return max(kMinUnits, (u + p.ctas - 1) / p.ctas);
}

// The sequence that unit `u` lies in; *first: the sequence's first unit.
// All lanes of a warp call it, with u inside the total.
__device__ __forceinline__ int find_unit(const DecodeParams& p, int u, int* first) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int mine = b0 + lane < p.B ? seq_units(p, b0 + lane) * p.c.kv_heads : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
    if (hit) {
      const int src = __ffs(hit) - 1;
      *first = before + __shfl_sync(0xffffffffu, incl - mine, src);
      return b0 + src;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}

}  // namespace

// Warps of a CTA: WR of them share a unit and hold 16 rows each (8 for RB =
// 8), and 4 / WR such teams take units in turn.  More rows than one warp's
// mean that every team member expands the unit's codes for itself; the
// cache's bytes still come once.
template <int D, int RB>
struct DecodeTile {
  static constexpr int kWr = RB <= 16 ? 1 : RB / 16;     // warps of a team
  static constexpr int kTeams = kDecWarps / kWr;
  static constexpr int kWarpRows = RB / kWr;             // 8 or 16
  static constexpr int kSlots = D / 8;                   // 16-byte slots per lane and stage (K and V)
  static constexpr int kStage = kSlots * 512 + 32;       // + the unit's four scales and a term of the scores of either half
  static constexpr int kCtas = 3;                        // CTAs per SM
  static constexpr int kStages = kWr == 4 ? 4 : kWr == 2 ? 3 : D == 128 ? 2 : 4;
  // Teams of four: the expanded codes, shared by the team, as the 16-byte
  // fragments of the products ([K, V][16 or 8 slots][lanes]) and the scales;
  // two buffers, so that one barrier per unit will do.
  static constexpr bool kShare = kWr == 4;
  static constexpr int kFrag = 2 * (D / 8) * 512 + 32;
  static constexpr int kRing = kTeams * kStages * kStage + (kShare ? 2 * kFrag : 0);
  static constexpr int kComb = kTeams > 1 ? RB * D * 4 + RB * 32 : 0;   // one team's partial on its way to the next
  static constexpr int kSmem = kRing + kComb;
};

template <typename T, int D, int RB>
__global__ void __launch_bounds__(kDecWarps * 32, (DecodeTile<D, RB>::kCtas)) kv8_attn_kernel(const __grid_constant__ DecodeParams p) {
  using C = DecodeTile<D, RB>;
  constexpr bool kUpper = RB > 8;           // rows g + 8 of the m16 tile in use
  constexpr int kHalves = kUpper ? 2 : 1;
  constexpr int KS = D / 16;                // k16 steps of the score product
  // Value product.  RB = 8: V^T is the 16-row operand and P^T the 8-column
  // one, O^T comes out (columns (D / 8) g + 2 n + {0, 1} of rows 2t, 2t + 1
  // in tile n); otherwise P is the 16-row operand (rows g, g + 8, columns
  // (D / 8) (2t + {0, 1}) + n in tile n).
  constexpr int NT = kUpper ? D / 8 : D / 16;
  constexpr int VW = D / 32;                // 4-byte words of a lane's piece of a V token
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int team = warp / C::kWr, wr = warp % C::kWr;
  uint8_t* ring = smem + team * (C::kStages * C::kStage);
  [[maybe_unused]] uint8_t* frags = smem + C::kTeams * C::kStages * C::kStage;
  float4* comb = reinterpret_cast<float4*>(smem + C::kRing) + wr * (NT * 32);   // [NT][lanes]
  float2* comb_ml = reinterpret_cast<float2*>(smem + C::kRing + RB * D * 4) + wr * (kHalves * 32);
  const Kv8View& c = p.c;
  const int page = 1 << c.page_shift;

  int total;
  const int per = units_per_cta(p, &total);
  const int u0 = min(total, (int)blockIdx.x * per), u1 = min(total, u0 + per);
  asm volatile("griddepcontrol.launch_dependents;");
  if (u0 >= u1) return;
  int first;
  int b = find_unit(p, u0, &first);
  int su = seq_units(p, b);
  int h = (u0 - first) / su;
  int unit0 = u0 - first - h * su;          // first unit within (b, h)
  const int row0 = blockIdx.y * RB + wr * C::kWarpRows;

  // The copies run ahead of the products, and the page table two units
  // ahead of the copies: look_up() loads a unit's two pages (its 32 tokens
  // lie in at most two), issue() copies the unit that was looked up before
  // the last one.
  struct Pages {
    int id[2], tok, head;
    bool any;
  };
  int pb = b, ph = h, plen = kv8_len(c, p.lens[b]);
  int psu = su, pu = u0 + team, pfirst = first + h * su;   // pfirst: flat index of (pb, ph)'s unit 0
  Pages ahead[2] = {};
  auto look_up = [&]() {
    Pages r{};
    r.any = pu < u1;
    if (r.any) {
      while (pu >= pfirst + psu) {          // next (sequence, head) that has units
        pfirst += psu;
        if (++ph == c.kv_heads) {
          ph = 0;
          do ++pb; while (seq_units(p, pb) == 0);
          psu = seq_units(p, pb);
          plen = kv8_len(c, p.lens[pb]);
        }
      }
      r.tok = (pu - pfirst) * kUnit;
      r.head = ph;
      const int32_t* row = c.table + (int64_t)pb * c.table_width;
      const int last = (plen - 1) >> c.page_shift;
#pragma unroll
      for (int i = 0; i < 2; ++i) r.id[i] = row[min((r.tok + 16 * i) >> c.page_shift, last)];
    }
    pu += C::kTeams;
    return r;
  };
  auto issue = [&](int stage) {
    Pages n = ahead[0];
    ahead[0] = ahead[1];
    ahead[1] = look_up();
    if (n.any) {
      int64_t kb[2];                        // element offsets of tokens tok and tok + 16
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (n.id[i] < 0 || n.id[i] >= c.num_pages) {
          report_error(kErrBadPage);
          n.id[i] = -1;                     // page 0 is copied in its place, and nothing of it seen
        }
        kb[i] = kv8_base(c, max(0, n.id[i]), n.head) + (int64_t)((n.tok + 16 * i) & (page - 1)) * D;
      }
      const uint32_t at = smem_u32(ring + stage * C::kStage), dst = at + lane * 16;
      // the team's warps take the pieces in turn
      // K: slot (j, i) = token 8 j + g, bytes 64 i + 16 t
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j % C::kWr != wr) continue;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
          cp_async16(dst + (j * (D / 64) + i) * 512,
                     c.k_codes + kb[j >> 1] + ((j & 1) * 8 + g) * D + i * 64 + t * 16);
      }
      // V: slot (kk, x) = token 16 kk + {2t, 2t + 1, 2t + 8, 2t + 9}[x], bytes of lane g's D / 8 columns
      if constexpr (C::kShare) {
        // what this warp will expand: one kk, half of the columns
        const int kk = wr >> 1;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int64_t off = (kk ? kb[1] : kb[0]) + (2 * t + (x & 1) + (x >> 1) * 8) * D + g * (D / 8) + (wr & 1) * (D / 16);
          const uint32_t to = at + (D / 16) * 512 + (wr * 4 + x) * (2 * D) + lane * (D / 16);
          if constexpr (D == 128) cp_async8(to, c.v_codes + off);
          else cp_async4(to, c.v_codes + off);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if ((kk * 4 + x) % C::kWr != wr) continue;
            const int64_t off = kb[kk] + (2 * t + (x & 1) + (x >> 1) * 8) * D + g * (D / 8);
            if constexpr (D == 128) cp_async16(dst + (D / 16 + kk * 4 + x) * 512, c.v_codes + off);
            else cp_async8(at + 4 * 512 + (kk * 4 + x) * 256 + lane * 8, c.v_codes + off);
          }
      }
      if (lane < 6 && wr == 0) {
        const int id = (lane & 1) ? n.id[1] : n.id[0];
        const float* sc = (lane < 2 ? c.k_scale : c.v_scale) + (int64_t)id * c.kv_heads + n.head;
        // a half without a page: keys of zero, and minus infinity for its scores
        if (lane < 4 && id >= 0) cp_async4(at + C::kSlots * 512 + lane * 4, sc);
        else st_shared(at + C::kSlots * 512 + lane * 4, lane < 4 || id >= 0 ? 0.f : -INFINITY);
      }
    }
    cp_commit();
  };
  ahead[0] = look_up();
  ahead[1] = look_up();
  // A warp that reads its own copies alone refills a stage when it has used
  // it; otherwise when the barrier of the next unit says that the team has.
  constexpr bool kAlone = C::kWr == 1 || C::kShare;
#pragma unroll
  for (int s = 0; s < C::kStages - (kAlone ? 0 : 1); ++s) issue(s);

  uint32_t qf[KS][4];
  float qs[2];                         // row factor: scale * log2(e) / the power of two q was multiplied by
  int lim[2];                          // tokens the row may see
  float o[NT][4], m[2], l[2];   // m: running maximum - kPShift, l: this lane's part of the sum
  // o = o * f for the rows of half hf; f is the row's (lanes 4 g ..)
  auto scale_rows = [&](int hf, float f) {
    if constexpr (kUpper) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][hf * 2] *= f;
        o[n][hf * 2 + 1] *= f;
      }
    } else {
      const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][0] *= f0;
        o[n][1] *= f1;
        o[n][2] *= f0;
        o[n][3] *= f1;
      }
    }
  };
  int stage = 0;
  [[maybe_unused]] int buf = 0;
  int cu = u0 + team;                       // this team's next unit
  int seg0 = u0;                            // current segment: units [seg0, seg1) of (b, h)
  int seg_first = u0 - unit0;               // flat index of (b, h)'s unit 0

  while (seg0 < u1) {
    const int seg1 = min(u1, seg_first + su);
    if (threadIdx.x == 0 && blockIdx.y == 0) {
      int* at = reinterpret_cast<int*>(p.range + b * c.kv_heads + h);
      if (seg0 == seg_first) at[0] = blockIdx.x;
      if (seg1 == seg_first + su) at[1] = blockIdx.x;
    }
    const int len = kv8_len(c, p.lens[b]);
    // query fragments and row state
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      m[hf] = -INFINITY;
      l[hf] = 0.f;
      const int r = row0 + hf * 8 + g;
      const bool live = r < p.rows && (kUpper || hf == 0);
      float f[D / 4];
      float top = 0.f;
      const int i_tok = r / p.group, head = h * p.group + r % p.group;
      lim[hf] = live ? len - p.T + i_tok + 1 : 0;
      const T* src = static_cast<const T*>(p.q) + b * p.q_sb + i_tok * p.q_st + head * p.q_sh;
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) f[i * 16 + e] = 0.f;
      if (live) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + i * 64 + t * 16 + v * 8);
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[i * 16 + v * 8 + k] = to_f32(e[k]);
          }
      }
#pragma unroll
      for (int e = 0; e < D / 4; ++e) top = fmaxf(top, fabsf(f[e]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^k that brings the row's largest value to [2^14, 2^15)
      int k = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
      k = max(-113, min(100, k));
      const float up = __uint_as_float((uint32_t)(k + 127) << 23);
      qs[hf] = p.scale_log2 * __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qf[i * 4 + w][hf + 2 * x] =
                hf < kHalves ? pack_f16x2(f[i * 16 + w * 4 + x * 2] * up, f[i * 16 + w * 4 + x * 2 + 1] * up) : 0u;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (; cu < seg1; cu += C::kTeams) {
      // the other lanes' copies (the scales) and the other warps' are in
      cp_wait<C::kStages - (kAlone ? 1 : 2)>();
      if constexpr (C::kShare) {
        // this warp's quarter of the unit, expanded once for the team
        const uint8_t* raw = ring + stage * C::kStage;
        uint4* fk = reinterpret_cast<uint4*>(frags + buf * C::kFrag) + lane;
        uint4* fv = fk + (D / 8) * 32;
        __syncwarp();                        // the scales are other lanes' copies
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint4 kw = *reinterpret_cast<const uint4*>(raw + (wr * (D / 64) + i) * 512 + lane * 16);
          const uint32_t w4[4] = {kw.x ^ 0x80808080u, kw.y ^ 0x80808080u, kw.z ^ 0x80808080u, kw.w ^ 0x80808080u};
#pragma unroll
          for (int w = 0; w < 4; w += 2)
            fk[((wr * (D / 64) + i) * 2 + w / 2) * 32] =
                make_uint4(codes_f16x2(w4[w], 0x4140), codes_f16x2(w4[w], 0x4342), codes_f16x2(w4[w + 1], 0x4140),
                           codes_f16x2(w4[w + 1], 0x4342));
        }
        uint32_t vw[4][VW / 2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint8_t* from = raw + (D / 16) * 512 + (wr * 4 + x) * (2 * D) + lane * (D / 16);
          if constexpr (D == 128) {
            const uint2 w = *reinterpret_cast<const uint2*>(from);
            vw[x][0] = w.x;
            vw[x][1] = w.y;
          } else {
            vw[x][0] = *reinterpret_cast<const uint32_t*>(from);
          }
        }
#pragma unroll
        for (int w = 0; w < VW / 2; ++w) {
          const uint32_t a_lo = __byte_perm(vw[0][w], vw[1][w], 0x5140) ^ 0x80808080u;
          const uint32_t a_hi = __byte_perm(vw[0][w], vw[1][w], 0x7362) ^ 0x80808080u;
          const uint32_t c_lo = __byte_perm(vw[2][w], vw[3][w], 0x5140) ^ 0x80808080u;
          const uint32_t c_hi = __byte_perm(vw[2][w], vw[3][w], 0x7362) ^ 0x80808080u;
          const int slot = ((wr >> 1) * VW + (wr & 1) * (VW / 2) + w) * 2;
          fv[slot * 32] = make_uint4(codes_f16x2(a_lo, 0x4140), codes_f16x2(c_lo, 0x4140), codes_f16x2(a_lo, 0x4342),
                                     codes_f16x2(c_lo, 0x4342));
          fv[(slot + 1) * 32] = make_uint4(codes_f16x2(a_hi, 0x4140), codes_f16x2(c_hi, 0x4140),
                                           codes_f16x2(a_hi, 0x4342), codes_f16x2(c_hi, 0x4342));
        }
        if (wr == 0 && lane < 6)
          reinterpret_cast<float*>(frags + buf * C::kFrag + 2 * (D / 8) * 512)[lane] =
              reinterpret_cast<const float*>(raw + C::kSlots * 512)[lane];
        __syncwarp();
        issue(stage);
        named_barrier(1 + team, C::kWr * 32);
      } else if constexpr (kAlone) {
        __syncwarp();
      } else {
        named_barrier(1 + team, C::kWr * 32);
        issue(stage == 0 ? C::kStages - 1 : stage - 1);
      }
      const uint8_t* st = ring + stage * C::kStage;
      const float* sc = reinterpret_cast<const float*>(C::kShare ? frags + buf * C::kFrag + 2 * (D / 8) * 512
                                                                 : st + C::kSlots * 512);
      [[maybe_unused]] const uint4* fk = reinterpret_cast<const uint4*>(frags + buf * C::kFrag) + lane;
      const float ks[2] = {sc[0], sc[1]}, vs[2] = {sc[2], sc[3]};
      const int tok0 = (cu - seg_first) * kUnit;
      // scores
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
        if constexpr (C::kShare) {
#pragma unroll
          for (int w = 0; w < D / 32; ++w) {
            const uint4 f = fk[(j * (D / 32) + w) * 32];
            mma_f16(s[j], qf[2 * w], f.x, f.y);
            mma_f16(s[j], qf[2 * w + 1], f.z, f.w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const uint4 kw = *reinterpret_cast<const uint4*>(st + (j * (D / 64) + i) * 512 + lane * 16);
            const uint32_t w4[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t bi = w4[w] ^ 0x80808080u;
              mma_f16(s[j], qf[i * 4 + w], codes_f16x2(bi, 0x4140), codes_f16x2(bi, 0x4342));
            }
          }
        }
      }
      // page scales: 2^e <= |vs| < 2^(e + 1), e kept within -60 and 121
      float ve[2], vf[2], vi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = max(-60, min(121, (int)((__float_as_uint(vs[i]) >> 23) & 0xff) - 127));
        ve[i] = (float)e + sc[4 + i];                         // - infinity: left out
        vi[i] = __uint_as_float((uint32_t)(127 - e) << 23);   // 2^-e
        vf[i] = vs[i] * vi[i];
      }
      uint32_t pa[2][4];
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        float x[4][2];
        // A row that sees a token has a finite maximum, so that one whose
        // scores are all minus infinity (0 / 0: NaN) differs from one that
        // sees nothing (zeros).
        float top = fmaxf(tok0 < lim[hf] ? ve[0] - FLT_MAX : -INFINITY, tok0 + 16 < lim[hf] ? ve[1] - FLT_MAX : -INFINITY);
        const int r = row0 + hf * 8 + g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = tok0 + j * 8 + 2 * t + e;
            const float v = s[j][hf * 2 + e] * (ks[j >> 1] * qs[hf]);
            s[j][hf * 2 + e] = v;
            x[j][e] = tok < lim[hf] ? v + ve[j >> 1] : -INFINITY;
            top = fmaxf(top, x[j][e]);
          }
        }
        if (p.scores && r < p.rows) {
          float* dst = p.scores + (((int64_t)b * c.kv_heads + h) * p.rows + r) * p.score_cap + tok0 + 2 * t;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(dst + j * 8) = make_float2(s[j][hf * 2], s[j][hf * 2 + 1]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[hf], top - kPShift);
        const float base = mn == -INFINITY ? 0.f : mn;            // nothing seen yet: every term is exp2(-inf)
        const float alpha = mn == -INFINITY ? 1.f : ex2(m[hf] - mn);
        m[hf] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float pv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ex = ex2(x[j][e] - base);
            sum = fmaf(ex, vi[j >> 1], sum);
            pv[e] = ex > 0.f ? ex * vf[j >> 1] : 0.f;   // a masked token's page scale does not matter
          }
          pa[j >> 1][(j & 1) * 2 + hf] = pack_f16x2(pv[0], pv[1]);
        }
        l[hf] = fmaf(l[hf], alpha, sum);
        if (__any_sync(0xffffffffu, alpha != 1.f)) scale_rows(hf, alpha);
      }
      // values
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        if constexpr (C::kShare) {
#pragma unroll
          for (int w = 0; w < VW * 2; ++w) {
            const uint4 f = fk[(D / 8 + kk * VW * 2 + w) * 32];
            mma_f16(o[2 * w], pa[kk], f.x, f.y);
            mma_f16(o[2 * w + 1], pa[kk], f.z, f.w);
          }
        } else {
          uint32_t vw[4][VW];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if constexpr (D == 128) {
              const uint4 w = *reinterpret_cast<const uint4*>(st + (D / 16 + kk * 4 + x) * 512 + lane * 16);
              vw[x][0] = w.x;
              vw[x][1] = w.y;
              vw[x][2] = w.z;
              vw[x][3] = w.w;
            } else {
              const uint2 w = *reinterpret_cast<const uint2*>(st + 4 * 512 + (kk * 4 + x) * 256 + lane * 8);
              vw[x][0] = w.x;
              vw[x][1] = w.y;
            }
          }
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            [[maybe_unused]] uint32_t va[4];
            const uint32_t a_lo = __byte_perm(vw[0][w], vw[1][w], 0x5140) ^ 0x80808080u;
            const uint32_t a_hi = __byte_perm(vw[0][w], vw[1][w], 0x7362) ^ 0x80808080u;
            const uint32_t c_lo = __byte_perm(vw[2][w], vw[3][w], 0x5140) ^ 0x80808080u;
            const uint32_t c_hi = __byte_perm(vw[2][w], vw[3][w], 0x7362) ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t b0 = codes_f16x2(e < 2 ? a_lo : a_hi, (e & 1) ? 0x4342 : 0x4140);
              const uint32_t b1 = codes_f16x2(e < 2 ? c_lo : c_hi, (e & 1) ? 0x4342 : 0x4140);
              if constexpr (kUpper) {
                mma_f16(o[w * 4 + e], pa[kk], b0, b1);
              } else {
                va[(e & 1)] = b0;
                va[2 + (e & 1)] = b1;
                if (e & 1) mma_f16(o[w * 2 + (e >> 1)], va, pa[kk][0], pa[kk][2]);
              }
            }
          }
        }
      }
      if constexpr (C::kShare) {
        buf ^= 1;
      } else if constexpr (kAlone) {
        __syncwarp();                        // every lane has read the stage's scales
        issue(stage);
      }
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
    }

    // Join the teams' partials of this segment: the last team hands its own
    // to the one before, that one the sum to the one before it and so on,
    // lane by lane (every lane writes and reads the same 16-byte places, so
    // no bank conflicts and one buffer); team 0 stores the segment's partial
    // in its slot.
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
    }
#pragma unroll 1
    for (int w = C::kTeams - 1; w >= 0; --w) {
      if (team == w) {
        if (w < C::kTeams - 1) {
          float fb[2] = {0.f, 0.f};
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            const float2 ml = comb_ml[hf * 32 + lane];
            const float mx = fmaxf(m[hf], ml.x);
            const float fa = l[hf] == 0.f ? 0.f : exp2f(m[hf] - mx);
            fb[hf] = ml.y == 0.f ? 0.f : exp2f(ml.x - mx);
            l[hf] = l[hf] * fa + ml.y * fb[hf];
            m[hf] = mx;
            scale_rows(hf, fa);
          }
          const float f0 = kUpper ? fb[0] : __shfl_sync(0xffffffffu, fb[0], 8 * t);
          const float f1 = kUpper ? fb[0] : __shfl_sync(0xffffffffu, fb[0], 8 * t + 4);
          const float f2 = kUpper ? fb[1] : f0, f3 = kUpper ? fb[1] : f1;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float4 v = comb[n * 32 + lane];
            o[n][0] = fmaf(v.x, f0, o[n][0]);
            o[n][1] = fmaf(v.y, f1, o[n][1]);
            o[n][2] = fmaf(v.z, f2, o[n][2]);
            o[n][3] = fmaf(v.w, f3, o[n][3]);
          }
        }
        if (w > 0) {
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) comb_ml[hf * 32 + lane] = make_float2(m[hf], l[hf]);
#pragma unroll
          for (int n = 0; n < NT; ++n) comb[n * 32 + lane] = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
        } else {
          const int64_t slot = (int64_t)blockIdx.y * p.slots + b * c.kv_heads + h + blockIdx.x;
          const int64_t at = slot * RB + wr * C::kWarpRows;
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            if (row0 + hf * 8 + g < p.rows && t == 0) p.part_ml[at + hf * 8 + g] = make_float2(m[hf], l[hf]);
          }
          if constexpr (kUpper) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
              if (row0 + hf * 8 + g < p.rows) {
                float* dst = p.part_o + (at + hf * 8 + g) * D + (D / 8) * 2 * t;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                  for (int n = 0; n < NT; n += 4)
                    *reinterpret_cast<float4*>(dst + x * (D / 8) + n) = make_float4(
                        o[n][hf * 2 + x], o[n + 1][hf * 2 + x], o[n + 2][hf * 2 + x], o[n + 3][hf * 2 + x]);
              }
          } else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (row0 + 2 * t + x < p.rows) {
                float* dst = p.part_o + (at + 2 * t + x) * D + (D / 8) * g;
#pragma unroll
                for (int n = 0; n < NT; n += 2)
                  *reinterpret_cast<float4*>(dst + 2 * n) = make_float4(o[n][x], o[n][2 + x], o[n + 1][x], o[n + 1][2 + x]);
              }
          }
        }
      }
      if constexpr (C::kTeams > 1) __syncthreads();   // the next team may read, or the next segment write
    }
    // next (sequence, head) with units
    seg0 = seg1;
    if (seg0 < u1) {
      seg_first += su;
      if (++h == c.kv_heads) {
        h = 0;
        do ++b; while (seq_units(p, b) == 0);
        su = seq_units(p, b);
      }
    }
  }
  cp_wait<0>();
}

// Second kernel: grid (B * kv_heads, output blocks + weight blocks).  An
// output block joins the partials of kJoinThreads / lanes groups of four
// columns of one (sequence, head), `lanes` threads taking every lanes-th
// partial of the same group (a long sequence has one partial per CTA of the
// first kernel, and reading them one after the other would cost more than
// the attention).  A weight block turns the scores of kJoinTokens tokens
// into weights (where there are many rows, of fewer tokens, with several
// threads to share a token's rows).
constexpr int kJoinTokens = 1024;
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 8;                  // rows of scores in flight per thread
constexpr int kMaxRows = 512;

// (m, l) joined with (m2, l2); f, f2: what the two sides' values are scaled
// by.  A side that has seen nothing has l = 0, m = -infinity; one that has seen
// scores of minus infinity alone l = 0 and a finite m; a NaN stays NaN.
__device__ __forceinline__ void join_stats(float& m, float& l, float m2, float l2, float& f, float& f2) {
  const float mx = fmaxf(m, m2);
  f = l == 0.f ? 0.f : exp2f(m - mx);
  f2 = l2 == 0.f ? 0.f : exp2f(m2 - mx);
  l = l * f + l2 * f2;
  m = mx;
}

// 1 / sum of a row's terms, with what it has seen as above.
__device__ __forceinline__ float inv_sum(float m, float l) {
  return l != 0.f ? 1.f / l : m == -INFINITY ? 0.f : __uint_as_float(0x7fffffffu);
}

template <typename T, int D, int RB>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float2 s_ml[kMaxRows];           // weights: (M - kPShift, 1 / sum) per row; 0: the row sees nothing
  __shared__ int s_see[kMaxRows];             // tokens the row sees
  __shared__ float4 s_part[kJoinThreads];
  constexpr int kCols = D / 4;                // column groups of a row
  const Kv8View& c = p.c;
  const int bh = blockIdx.x, b = bh / c.kv_heads, h = bh - b * c.kv_heads;
  const int chunk = (int)blockIdx.y - p.out_blocks;
  const int len = kv8_len(c, p.lens[b]);
  const int tokens = kJoinTokens / p.row_groups;   // a weight block's
  if (chunk >= 0 && (int64_t)chunk * tokens >= len) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the CTAs of the first kernel that hold partials of (b, h): c0 .. c1
  const int2 range = len > 0 ? p.range[bh] : make_int2(0, -1);
  const int c0 = range.x, c1 = range.y;

  if (chunk < 0) {
    const int groups = kJoinThreads / p.lanes;
    const int part = threadIdx.x / groups, item = blockIdx.y * groups + threadIdx.x % groups;
    const int r = item / kCols, col = item - r * kCols;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    if (r < p.rows) {
      const int64_t at = ((int64_t)(r / RB) * p.slots + bh) * RB + r % RB;
      const float2* mls = p.part_ml + at;
      const float4* os = reinterpret_cast<const float4*>(p.part_o + at * D) + col;
      for (int i0 = c0 + part; i0 <= c1; i0 += 4 * p.lanes) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int64_t i = i0 + x * p.lanes;
          ml[x] = make_float2(-INFINITY, 0.f);
          v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i <= c1) {
            ml[x] = mls[i * RB];
            v[x] = os[i * RB * kCols];
          }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float f, f2;
          join_stats(m, l, ml[x].x, ml[x].y, f, f2);
          acc.x = acc.x * f + v[x].x * f2;
          acc.y = acc.y * f + v[x].y * f2;
          acc.z = acc.z * f + v[x].z * f2;
          acc.w = acc.w * f + v[x].w * f2;
        }
      }
    }
    if (p.lanes > 1) {
      s_part[threadIdx.x] = acc;
      s_ml[threadIdx.x] = make_float2(m, l);
      __syncthreads();
      if (part == 0)
        for (int i = 1; i < p.lanes; ++i) {
          const float4 v = s_part[threadIdx.x + i * groups];
          const float2 ml = s_ml[threadIdx.x + i * groups];
          float f, f2;
          join_stats(m, l, ml.x, ml.y, f, f2);
          acc.x = acc.x * f + v.x * f2;
          acc.y = acc.y * f + v.y * f2;
          acc.z = acc.z * f + v.z * f2;
          acc.w = acc.w * f + v.w * f2;
        }
    }
    if (part == 0 && r < p.rows) {
      const float inv = inv_sum(m, l);   // zeros where the row sees nothing
      T* dst = static_cast<T*>(p.out) + (((int64_t)b * p.T + r / p.group) * p.heads + h * p.group + r % p.group) * D + col * 4;
      const T o[4] = {from_f32<T>(acc.x * inv), from_f32<T>(acc.y * inv), from_f32<T>(acc.z * inv),
                      from_f32<T>(acc.w * inv)};
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
    }
    return;
  }
  // Four tokens per thread, and every row_groups-th row.  The first rows'
  // scores and the old weights are on their way while the statistics are
  // joined; a masked or padded score is loaded (inside its row) but never
  // used.
  const int quads = tokens / 4, rg = threadIdx.x / quads, tok = chunk * tokens + threadIdx.x % quads * 4;
  bool live = tok < len;
  if (live) {                                 // a page (of four tokens at least) outside the pool: nothing is seen
    const int id = c.table[(int64_t)b * c.table_width + (tok >> c.page_shift)];
    live = id >= 0 && id < c.num_pages;
  }
  const float* s = p.scores + (int64_t)bh * p.rows * p.score_cap + tok;
  const int64_t wat = (int64_t)bh * p.cap + tok;
  float4 v[kJoinRows];
  auto fetch = [&](int r0) {
    const float* at = s + (int64_t)(r0 + rg) * p.score_cap;
    const int64_t step = (int64_t)p.row_groups * p.score_cap;
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i, at += step)
      if (live && r0 + i * p.row_groups + rg < p.rows) v[i] = *reinterpret_cast<const float4*>(at);
  };
  fetch(0);
  float w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = rg == 0 && tok + e < len ? p.weights[wat + e] : 0.f;
  // `per_row` lanes join a row's statistics: no more than there are partials,
  // nor than let the block take all rows at once
  int per_row = 1;
  while (per_row < 32 && per_row < c1 - c0 + 1 && kJoinThreads / (2 * per_row) >= p.rows) per_row <<= 1;
  for (int r0 = 0; r0 < p.rows; r0 += kJoinThreads / per_row) {
    const int r = r0 + threadIdx.x / per_row;
    float m = -INFINITY, l = 0.f, f, f2;
    if (r < p.rows) {
      const float2* mls = p.part_ml + ((int64_t)(r / RB) * p.slots + bh) * RB + r % RB;
#pragma unroll 4
      for (int i = c0 + threadIdx.x % per_row; i <= c1; i += per_row) {
        const float2 ml = mls[(int64_t)i * RB];
        join_stats(m, l, ml.x, ml.y, f, f2);
      }
    }
    for (int o = per_row >> 1; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
      join_stats(m, l, m2, l2, f, f2);
    }
    if (r < p.rows && threadIdx.x % per_row == 0) {
      s_ml[r] = make_float2(m, inv_sum(m, l));
      s_see[r] = m == -INFINITY && l == 0.f ? 0 : len - p.T + r / p.group + 1;
    }
  }
  __syncthreads();
  float mass[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < p.rows; r0 += kJoinRows * p.row_groups) {
    if (r0) fetch(r0);
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i) {
      const int r = r0 + i * p.row_groups + rg;
      if (r >= p.rows) break;
      const float2 row = s_ml[r];
      const int see = s_see[r];
      const float x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (live && tok + e < see) mass[e] = fmaf(ex2(x[e] - row.x), row.y, mass[e]);
    }
  }
  if (p.row_groups > 1) {
    s_part[threadIdx.x] = make_float4(mass[0], mass[1], mass[2], mass[3]);
    __syncthreads();
    if (rg == 0)
      for (int i = 1; i < p.row_groups; ++i) {
        const float4 o = s_part[threadIdx.x + i * quads];
        mass[0] += o.x;
        mass[1] += o.y;
        mass[2] += o.z;
        mass[3] += o.w;
      }
  }
  if (rg) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (tok + e < len) p.weights_out[wat + e] = w[e] + mass[e];
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Rows per CTA; beyond 64 the cache is read once for each 64.
static int row_block(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

// Workspace: partials, their (M, sum), and the scores where weights are kept.
static void decode_plan(DecodeParams& p, size_t* bytes) {
  const int rb = row_block(p.rows), blocks = (p.rows + rb - 1) / rb;
  const int64_t cap_units = (((int64_t)p.c.table_width << p.c.page_shift) + kUnit - 1) / kUnit;
  const int64_t most = (cap_units * p.B * p.c.kv_heads + kMinUnits - 1) / kMinUnits;
  int64_t ctas = (int64_t)sm_count() * 3;                    // DecodeTile's kCtas
  ctas = (ctas + blocks - 1) / blocks;
  p.ctas = (int)(most < ctas ? most : ctas);
  if (p.ctas < 1) p.ctas = 1;
  p.slots = p.B * p.c.kv_heads + p.ctas;
  p.score_cap = cap_units * kUnit;
  // a (sequence, head) has about ctas / (B * kv_heads) partials; more lanes
  // than keep the output blocks to one wave (four to an SM) cost more than
  // they save (8 verify tokens of 8 sequences: 8 lanes 13 us, 2 lanes 5 us)
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes * p.B * p.c.kv_heads * 2 <= p.ctas &&
         (int64_t)p.lanes * 2 * p.B * p.c.kv_heads * p.rows * (p.c.dim / 4) <= (int64_t)kJoinThreads * 4 * sm_count())
    p.lanes *= 2;
  p.row_groups = p.rows <= 8 ? 1 : p.rows <= 16 ? 2 : 4;
  const int groups = kJoinThreads / p.lanes;
  p.out_blocks = (p.rows * (p.c.dim / 4) + groups - 1) / groups;
  const size_t part_rows = (size_t)blocks * p.slots * rb;
  uint8_t* w = reinterpret_cast<uint8_t*>(p.part_o);
  auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t off = al(part_rows * p.c.dim * 4);
  p.part_ml = reinterpret_cast<float2*>(w + off);
  off += al(part_rows * 8);
  p.range = reinterpret_cast<int2*>(w + off);
  off += al((size_t)p.B * p.c.kv_heads * 8);
  p.scores = p.weights ? reinterpret_cast<float*>(w + off) : nullptr;
  if (p.weights) off += (size_t)p.B * p.c.kv_heads * p.rows * p.score_cap * 4;
  *bytes = off;
}

int kv8_attn_max_rows() { return kMaxRows; }

size_t kv8_attn_workspace(const Kv8View& c, int B, int T, int heads, int with_weights) {
  DecodeParams p{};
  p.c = c;
  p.B = B;
  p.T = T;
  p.heads = heads;
  p.group = heads / c.kv_heads;
  p.rows = T * p.group;
  float dummy;
  p.weights = with_weights ? &dummy : nullptr;
  size_t bytes;
  decode_plan(p, &bytes);
  return bytes;
}

template <typename T, int D, int RB>
static cudaError_t launch_decode(const DecodeParams& p, cudaStream_t st) {
  using C = DecodeTile<D, RB>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kv8_attn_kernel<T, D, RB>), C::kSmem);
  if (e != cudaSuccess) return e;
  const int blocks = (p.rows + RB - 1) / RB;
  kv8_attn_kernel<T, D, RB><<<dim3((unsigned)p.ctas, (unsigned)blocks), kDecWarps * 32, C::kSmem, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t cap = (int64_t)p.c.table_width << p.c.page_shift;
  const int64_t chunks = p.weights ? (cap * p.row_groups + kJoinTokens - 1) / kJoinTokens : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.c.kv_heads), (unsigned)(p.out_blocks + chunks));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv8_join_kernel<T, D, RB>, p);
}

template <typename T>
static cudaError_t launch_decode_dim(const DecodeParams& p, cudaStream_t st) {
  const int rb = row_block(p.rows);
  if (p.c.dim == 128)
    return rb == 8    ? launch_decode<T, 128, 8>(p, st)
           : rb == 16 ? launch_decode<T, 128, 16>(p, st)
           : rb == 32 ? launch_decode<T, 128, 32>(p, st)
                      : launch_decode<T, 128, 64>(p, st);
  return rb == 8    ? launch_decode<T, 64, 8>(p, st)
         : rb == 16 ? launch_decode<T, 64, 16>(p, st)
         : rb == 32 ? launch_decode<T, 64, 32>(p, st)
                    : launch_decode<T, 64, 64>(p, st);
}

cudaError_t launch_kv8_attn(const Kv8View& c, const void* q, int dtype, const int64_t* strides, int B, int T, int heads,
                            const int32_t* lens, float scale, const float* weights, float* weights_out, int64_t cap,
                            void* out, void* workspace, cudaStream_t st) {
  DecodeParams p{};
  p.c = c;
  p.q = q;
  p.q_sb = strides[0];
  p.q_st = strides[1];
  p.q_sh = strides[2];
  p.out = out;
  p.lens = lens;
  p.B = B;
  p.T = T;
  p.heads = heads;
  p.group = heads / c.kv_heads;
  p.rows = T * p.group;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part_o = static_cast<float*>(workspace);
  p.weights = weights;
  p.weights_out = weights_out;
  p.cap = cap;
  size_t bytes;
  decode_plan(p, &bytes);
  return dtype == PARO_BF16 ? launch_decode_dim<__nv_bfloat16>(p, st) : launch_decode_dim<__half>(p, st);
}

}  // namespace paro
