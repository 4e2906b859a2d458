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
// stays below 2^15 whatever the page scales are.  The denominator keeps the
// unrounded float32 terms.
//
// A CTA that meets the end of its run inside a (sequence, head) leaves a
// partial (M, sum, weighted values) that the second kernel joins; that
// kernel also turns the stored scores into softmax weights where the caller
// accumulates them, one writer per element, so every result is independent
// of timing.
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
  int lanes, out_blocks;       // second kernel: threads per output column group, blocks of output rows
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

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// units of sequence b per KV head
__device__ __forceinline__ int64_t seq_units(const DecodeParams& p, int b) {
  const int64_t cap = (int64_t)p.c.table_width << p.c.page_shift;
  const int64_t len = max((int64_t)0, min((int64_t)p.lens[b], cap));
  return (len + kUnit - 1) / kUnit;
}

// Units of all sequences together, and per CTA.
__device__ __forceinline__ int64_t units_per_cta(const DecodeParams& p, int64_t* total) {
  const int lane = threadIdx.x & 31;
  int64_t u = 0;
  for (int b = lane; b < p.B; b += 32) u += seq_units(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
  *total = u * p.c.kv_heads;
  const int64_t per = (*total + p.ctas - 1) / p.ctas;
  return per < kMinUnits ? kMinUnits : per;
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
  static constexpr int kStage = kSlots * 512 + 32;       // + the unit's four scales
  static constexpr int kStages = kWr == 1 ? (D == 128 ? 3 : 4) : 4;
  static constexpr int kRing = kTeams * kStages * kStage;
  static constexpr int kComb = kTeams > 1 ? RB * D * 4 + RB * 32 : 0;   // one team's partial on its way to the next
  static constexpr int kSmem = kRing + kComb;
};

template <typename T, int D, int RB>
__global__ void __launch_bounds__(kDecWarps * 32, 2) kv8_attn_kernel(const __grid_constant__ DecodeParams p) {
  using C = DecodeTile<D, RB>;
  constexpr bool kUpper = RB > 8;           // rows g + 8 of the m16 tile in use
  constexpr int kHalves = kUpper ? 2 : 1;
  constexpr int KS = D / 16;                // k16 steps of the score product
  constexpr int NT = D / 8;                 // n8 tiles of the value product
  constexpr int VW = D / 32;                // 4-byte words of a lane's piece of a V token
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int team = warp / C::kWr, wr = warp % C::kWr;
  uint8_t* ring = smem + team * (C::kStages * C::kStage);
  float4* comb = reinterpret_cast<float4*>(smem + C::kRing) + wr * (kHalves * (NT / 2) * 32);   // [halves][NT / 2][lanes]
  float2* comb_ml = reinterpret_cast<float2*>(smem + C::kRing + RB * D * 4) + wr * (kHalves * 32);
  const Kv8View& c = p.c;
  const int page = 1 << c.page_shift;

  int64_t total;
  const int64_t per = units_per_cta(p, &total);
  const int64_t u0 = blockIdx.x * per, u1 = min(total, u0 + per);
  asm volatile("griddepcontrol.launch_dependents;");
  if (u0 >= u1) return;
  int64_t first;
  int b = warp_find_seq(u0, p.B, [&](int i) { return seq_units(p, i) * c.kv_heads; }, &first);
  int64_t su = seq_units(p, b);
  int h = (int)((u0 - first) / su);
  int64_t unit0 = u0 - first - h * su;      // first unit within (b, h)
  const int row0 = blockIdx.y * RB + wr * C::kWarpRows;

  // The copies run ahead of the products, and the page table ahead of the
  // copies: look_up() loads the next unit's two pages (a unit's 32 tokens
  // lie in at most two), issue() copies the unit that was looked up before.
  int pb = b, ph = h, plen = kv8_len(c, p.lens[b]);
  int64_t psu = su, pu = u0 + team, pfirst = first + h * su;   // pfirst: flat index of (pb, ph)'s unit 0
  int n_id[2] = {0, 0}, n_tok = 0, n_head = 0;
  bool n_any = false;
  auto look_up = [&]() {
    n_any = pu < u1;
    if (n_any) {
      while (pu >= pfirst + psu) {          // next (sequence, head) that has units
        pfirst += psu;
        if (++ph == c.kv_heads) {
          ph = 0;
          do ++pb; while (seq_units(p, pb) == 0);
          psu = seq_units(p, pb);
          plen = kv8_len(c, p.lens[pb]);
        }
      }
      n_tok = (int)(pu - pfirst) * kUnit;
      n_head = ph;
      const int32_t* row = c.table + (int64_t)pb * c.table_width;
      const int last = (plen - 1) >> c.page_shift;
#pragma unroll
      for (int i = 0; i < 2; ++i) n_id[i] = row[min((n_tok + 16 * i) >> c.page_shift, last)];
    }
    pu += C::kTeams;
  };
  auto issue = [&](int stage) {
    if (n_any) {
      int64_t kb[2];                        // element offsets of tokens n_tok and n_tok + 16
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (n_id[i] < 0 || n_id[i] >= c.num_pages) {
          report_error(kErrBadPage);
          n_id[i] = 0;
        }
        kb[i] = kv8_base(c, n_id[i], n_head) + (int64_t)((n_tok + 16 * i) & (page - 1)) * D;
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
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if ((kk * 4 + x) % C::kWr != wr) continue;
          const int64_t off = kb[kk] + (2 * t + (x & 1) + (x >> 1) * 8) * D + g * (D / 8);
          if constexpr (D == 128) cp_async16(dst + (D / 16 + kk * 4 + x) * 512, c.v_codes + off);
          else cp_async8(at + 4 * 512 + (kk * 4 + x) * 256 + lane * 8, c.v_codes + off);
        }
      if (lane < 4 && wr == 0) {
        const float* sc = (lane < 2 ? c.k_scale : c.v_scale) + (int64_t)((lane & 1) ? n_id[1] : n_id[0]) * c.kv_heads + n_head;
        cp_async4(at + C::kSlots * 512 + lane * 4, sc);
      }
    }
    cp_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) {
    issue(s);
    look_up();
  }

  uint32_t qf[KS][4];
  float qs[2];                         // row factor: scale * log2(e) / the power of two q was multiplied by
  int lim[2];                          // tokens the row may see
  float o[NT][4], m[2], l[2];   // m: running maximum - kPShift, l: this lane's part of the sum
  int stage = 0;
  int64_t cu = u0 + team;                   // this team's next unit
  int64_t seg0 = u0;                        // current segment: units [seg0, seg1) of (b, h)
  int64_t seg_first = u0 - unit0;           // flat index of (b, h)'s unit 0

  while (seg0 < u1) {
    const int64_t seg1 = min(u1, seg_first + su);
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
      k = max(-100, min(100, k));
      const float up = __uint_as_float((uint32_t)(k + 127) << 23);
      qs[hf] = p.scale_log2 * __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qf[i * 4 + w][hf + 2 * x] =
                pack_f16x2(f[i * 16 + w * 4 + x * 2] * up, f[i * 16 + w * 4 + x * 2 + 1] * up);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (; cu < seg1; cu += C::kTeams) {
      cp_wait<C::kStages - 2>();
      // the other lanes' copies (the scales) and the other warps' are in, and
      // everyone is done with the stage that is filled next
      if constexpr (C::kWr == 1) __syncwarp();
      else named_barrier(1 + team, C::kWr * 32);
      issue(stage == 0 ? C::kStages - 1 : stage - 1);
      look_up();
      const uint8_t* st = ring + stage * C::kStage;
      const float* sc = reinterpret_cast<const float*>(st + C::kSlots * 512);
      const float ks[2] = {sc[0], sc[1]}, vs[2] = {sc[2], sc[3]};
      const int tok0 = (int)(cu - seg_first) * kUnit;
      // scores
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
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
      // page scales: 2^e <= |vs| < 2^(e + 1), e kept within +-60
      float ve[2], vf[2], vi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = max(-60, min(60, (int)((__float_as_uint(vs[i]) >> 23) & 0xff) - 127));
        ve[i] = (float)e;
        vi[i] = __uint_as_float((uint32_t)(127 - e) << 23);   // 2^-e
        vf[i] = vs[i] * vi[i];
      }
      uint32_t pa[2][4];
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        float x[4][2];
        float top = -INFINITY;
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
        const float alpha = mn == -INFINITY ? 1.f : exp2f(m[hf] - mn);
        m[hf] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float pv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ex = exp2f(x[j][e] - base);
            sum = fmaf(ex, vi[j >> 1], sum);
            pv[e] = ex > 0.f ? ex * vf[j >> 1] : 0.f;   // a masked token's page scale does not matter
          }
          pa[j >> 1][(j & 1) * 2 + hf] = pack_f16x2(pv[0], pv[1]);
        }
        l[hf] = fmaf(l[hf], alpha, sum);
        if (alpha != 1.f) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][hf * 2] *= alpha;
            o[n][hf * 2 + 1] *= alpha;
          }
        }
      }
      if constexpr (!kUpper) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) pa[kk][1] = pa[kk][3] = 0u;
      }
      // values
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
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
          const uint32_t a_lo = __byte_perm(vw[0][w], vw[1][w], 0x5140) ^ 0x80808080u;
          const uint32_t a_hi = __byte_perm(vw[0][w], vw[1][w], 0x7362) ^ 0x80808080u;
          const uint32_t c_lo = __byte_perm(vw[2][w], vw[3][w], 0x5140) ^ 0x80808080u;
          const uint32_t c_hi = __byte_perm(vw[2][w], vw[3][w], 0x7362) ^ 0x80808080u;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t b0 = codes_f16x2(e < 2 ? a_lo : a_hi, (e & 1) ? 0x4342 : 0x4140);
            const uint32_t b1 = codes_f16x2(e < 2 ? c_lo : c_hi, (e & 1) ? 0x4342 : 0x4140);
            mma_f16(o[w * 4 + e], pa[kk], b0, b1);
          }
        }
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
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
          if (w < C::kTeams - 1) {
            const float2 ml = comb_ml[hf * 32 + lane];
            const float mx = fmaxf(m[hf], ml.x);
            const float fa = l[hf] == 0.f ? 0.f : exp2f(m[hf] - mx);
            const float fb = ml.y == 0.f ? 0.f : exp2f(ml.x - mx);
            l[hf] = l[hf] * fa + ml.y * fb;
            m[hf] = mx;
#pragma unroll
            for (int n = 0; n < NT / 2; ++n) {
              const float4 v = comb[(hf * (NT / 2) + n) * 32 + lane];
              o[2 * n][hf * 2] = fmaf(v.x, fb, o[2 * n][hf * 2] * fa);
              o[2 * n][hf * 2 + 1] = fmaf(v.y, fb, o[2 * n][hf * 2 + 1] * fa);
              o[2 * n + 1][hf * 2] = fmaf(v.z, fb, o[2 * n + 1][hf * 2] * fa);
              o[2 * n + 1][hf * 2 + 1] = fmaf(v.w, fb, o[2 * n + 1][hf * 2 + 1] * fa);
            }
          }
          if (w > 0) {
            comb_ml[hf * 32 + lane] = make_float2(m[hf], l[hf]);
#pragma unroll
            for (int n = 0; n < NT / 2; ++n)
              comb[(hf * (NT / 2) + n) * 32 + lane] = make_float4(o[2 * n][hf * 2], o[2 * n][hf * 2 + 1],
                                                                  o[2 * n + 1][hf * 2], o[2 * n + 1][hf * 2 + 1]);
          } else {
            const int r = hf * 8 + g;
            if (row0 + r < p.rows) {
              const int64_t slot = (int64_t)blockIdx.y * p.slots + b * c.kv_heads + h + blockIdx.x;
              const int64_t at = slot * RB + wr * C::kWarpRows + r;
              if (t == 0) p.part_ml[at] = make_float2(m[hf], l[hf]);
              // column n of value tile i is value column (D / 8) n + i
              float* dst = p.part_o + at * D + (D / 8) * 2 * t;
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NT; n += 4)
                  *reinterpret_cast<float4*>(dst + x * (D / 8) + n) = make_float4(
                      o[n][hf * 2 + x], o[n + 1][hf * 2 + x], o[n + 2][hf * 2 + x], o[n + 3][hf * 2 + x]);
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
// output block joins the partials of a few rows of one (sequence, head),
// `lanes` threads taking every lanes-th partial of the same four columns (a
// long sequence has one partial per CTA of the first kernel, and reading
// them one after the other would cost more than the attention); a weight
// block turns the scores of kJoinTokens tokens into weights.
constexpr int kJoinTokens = 1024;
constexpr int kJoinThreads = 256;
constexpr int kMaxRows = 512;

template <typename T, int D, int RB>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float2 s_ml[kMaxRows];           // (M - kPShift, 1 / sum) per row; 1 / sum = 0: the row sees nothing
  __shared__ float4 s_part[kJoinThreads];
  constexpr int kCols = D / 4;                // threads across a row
  const Kv8View& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bh = blockIdx.x, b = bh / c.kv_heads, h = bh - b * c.kv_heads;
  const int64_t tok0 = (int64_t)((int)blockIdx.y - p.out_blocks) * kJoinTokens;
  const int len = kv8_len(c, p.lens[b]);
  if (tok0 >= len && tok0 >= 0) return;
  // the CTAs of the first kernel that hold partials of (b, h): c0 .. c1
  int64_t total;
  const int64_t per = units_per_cta(p, &total);
  int64_t before = 0;
  for (int i = lane; i < b; i += 32) before += seq_units(p, i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const int64_t su = seq_units(p, b), ub = before * c.kv_heads + h * su;
  const int c0 = (int)(ub / per), c1 = su ? (int)((ub + su - 1) / per) : c0 - 1;
  // rows whose statistics this block needs
  const int per_block = kJoinThreads / kCols / p.lanes;
  const int ra = tok0 < 0 ? blockIdx.y * per_block : 0, rz = tok0 < 0 ? min(p.rows, ra + per_block) : p.rows;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  for (int r = ra + warp; r < rz; r += kJoinThreads / 32) {
    const float2* ml = p.part_ml + ((int64_t)(r / RB) * p.slots + bh) * RB + r % RB;
    float mx = -INFINITY, sum = 0.f;
    for (int i = c0 + lane; i <= c1; i += 32) {
      const float2 v = ml[(int64_t)i * RB];
      if (v.y == 0.f) continue;
      const float m = fmaxf(mx, v.x);
      sum = (sum == 0.f ? 0.f : sum * exp2f(mx - m)) + v.y * exp2f(v.x - m);
      mx = m;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, mx, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
      const float m = fmaxf(mx, om);
      sum = (sum == 0.f ? 0.f : sum * exp2f(mx - m)) + (os == 0.f ? 0.f : os * exp2f(om - m));
      mx = m;
    }
    // a sum that is NaN (a page scale that is not finite) stays NaN
    if (lane == 0) s_ml[r] = make_float2(mx, sum == 0.f ? 0.f : 1.f / sum);
  }
  __syncthreads();
  if (tok0 < 0) {
    const int col = threadIdx.x % kCols, rest = threadIdx.x / kCols, part = rest % p.lanes, r = ra + rest / p.lanes;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rz) {
      const int64_t at = ((int64_t)(r / RB) * p.slots + bh) * RB + r % RB;
      const float mx = s_ml[r].x;
#pragma unroll 4
      for (int i = c0 + part; i <= c1; i += p.lanes) {
        const float2 ml = p.part_ml[at + (int64_t)i * RB];
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + (at + (int64_t)i * RB) * D + col * 4);
        const float f = ml.y == 0.f ? 0.f : exp2f(ml.x - mx);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
      }
    }
    if (p.lanes > 1) {
      s_part[threadIdx.x] = acc;
      __syncthreads();
      if (part == 0)
        for (int i = 1; i < p.lanes; ++i) {
          const float4 v = s_part[threadIdx.x + i * kCols];
          acc.x += v.x;
          acc.y += v.y;
          acc.z += v.z;
          acc.w += v.w;
        }
    }
    if (part == 0 && r < rz) {
      const float inv = s_ml[r].y;
      T* dst = static_cast<T*>(p.out) + (((int64_t)b * p.T + r / p.group) * p.heads + h * p.group + r % p.group) * D + col * 4;
      const T o[4] = {from_f32<T>(acc.x * inv), from_f32<T>(acc.y * inv), from_f32<T>(acc.z * inv),
                      from_f32<T>(acc.w * inv)};
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
    }
    return;
  }
  // four tokens per thread; a masked or padded score is never used
  const int64_t tok = tok0 + threadIdx.x * 4;
  if (tok >= len) return;
  const float* s = p.scores + (int64_t)bh * p.rows * p.score_cap + tok;
  float mass[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int r = 0; r < p.rows; ++r) {
    const float4 v = *reinterpret_cast<const float4*>(s + (int64_t)r * p.score_cap);
    const float2 row = s_ml[r];
    const int see = row.y == 0.f ? 0 : len - p.T + r / p.group + 1;
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (tok + e < see) mass[e] = fmaf(exp2f(x[e] - row.x), row.y, mass[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (tok + e < len) {
      const int64_t at = (int64_t)bh * p.cap + tok + e;
      p.weights_out[at] = p.weights[at] + mass[e];
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Rows per CTA; beyond 64 the cache is read once for each 64.
static int row_block(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
constexpr int kDecodeCtasPerSm = 2;

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

// Workspace: partials, their (M, sum), and the scores where weights are kept.
static void decode_plan(DecodeParams& p, size_t* bytes) {
  const int rb = row_block(p.rows), blocks = (p.rows + rb - 1) / rb;
  const int64_t cap_units = (((int64_t)p.c.table_width << p.c.page_shift) + kUnit - 1) / kUnit;
  const int64_t most = (cap_units * p.B * p.c.kv_heads + kMinUnits - 1) / kMinUnits;
  int64_t ctas = (int64_t)sm_count() * kDecodeCtasPerSm;
  ctas = (ctas + blocks - 1) / blocks;
  p.ctas = (int)(most < ctas ? most : ctas);
  if (p.ctas < 1) p.ctas = 1;
  p.slots = p.B * p.c.kv_heads + p.ctas;
  p.score_cap = cap_units * kUnit;
  // a (sequence, head) has about ctas / (B * kv_heads) partials
  p.lanes = 1;
  while (p.lanes < 8 && p.lanes * p.B * p.c.kv_heads * 2 <= p.ctas) p.lanes *= 2;
  const int per_block = kJoinThreads / (p.c.dim / 4) / p.lanes;
  p.out_blocks = (p.rows + per_block - 1) / per_block;
  const size_t part_rows = (size_t)blocks * p.slots * rb;
  uint8_t* w = reinterpret_cast<uint8_t*>(p.part_o);
  auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t off = al(part_rows * p.c.dim * 4);
  p.part_ml = reinterpret_cast<float2*>(w + off);
  off += al(part_rows * 8);
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
  const int64_t chunks = p.weights ? (cap + kJoinTokens - 1) / kJoinTokens : 0;
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
