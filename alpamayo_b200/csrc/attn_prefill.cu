// attn_prefill.cu — causal attention over packed prompts with grouped heads,
// on the 5th-generation tensor cores (sm_100a).
//
//   o_i = sum_{j <= i + Lk - Lq} softmax_j(scale * q_i . k_j) v_j
//
// One CTA per (256 query rows of one sequence, head): two tiles of 128 rows
// that share every key/value tile of 128 tokens, walked with a running
// maximum and sum.  Bound by the tensor cores (4 * dim flops per pair) and,
// nearly as much, by the exponentials: a 128 x 128 tile takes 2 * 512 clocks
// of tcgen05.mma (dim 128) and 1024 clocks of the SM's 16 exp2 lanes.
//
//  * warps 0-3 / 4-7: softmax of tile 0 / 1, one thread per row.  The scores
//    come from tensor memory into registers; the probabilities go back over
//    the same columns in 16 bits (the value product takes them from there).
//    The output is rescaled only when a row's maximum has grown by more than
//    2^8 since the reference maximum in use (any exact common factor of
//    terms and sum cancels), so nearly never.
//  * warp 8: TMA loads, K_0 V_0 K_1 V_1 ... through one ring of tiles.
//  * warp 9: MMAs, one thread: S = Q K^T (both K-major in shared memory) and
//    O += P V (P in tensor memory, V with its columns contiguous, i.e.
//    MN-major).  In issue order ... O_0 += P_0(j) V_j, S_0 = Q_0 K_(j+1),
//    O_1 += P_1(j) V_j, S_1 = Q_1 K_(j+1) ..., so one tile's softmax runs
//    under the other's MMAs.  tcgen05 operations of one thread complete in
//    order: S(j + 1) being ready says that O has taken in P(j).
//  * warps 10-11: the value tiles that some row of the CTA sees only in part
//    (at most three: the diagonal ones).  A product with a zero probability
//    is not zero where the value is not finite, so these warps zero the rows
//    behind the last key and every value that is not finite, and note the
//    keys concerned; the epilogue adds those values back, each to the rows
//    that see it.  What a row does not see has no effect on it.
//
// Probabilities are rounded to the inputs' type for the value product (the
// relative error of 2^-9 that bf16 operands of the tensor core have anyhow;
// it is of the size of the output's own rounding); sums, maxima and the
// output stay in float32, and the denominator adds the unrounded terms.
#include "umma.cuh"

namespace paro {

PARO_DEFINE_ERROR_ACCESSOR(attn)

constexpr int kPfRows = 128;       // query rows per tile, keys per tile
constexpr int kPfThreads = 384;
constexpr int kPfSplits = 8;       // splits of an item's keys, at most
constexpr int kPfMasked = 3;       // key tiles that a CTA's rows see in part, at most

struct PrefillParams {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, heads, group;
  int rows, k_rows;
  float scale_log2;
  void* out;
  const void* v;                   // for the values that are not finite
  int64_t sv_t, sv_h;
  int splits;                      // CTAs that share the keys of one item; > 1: partial results
  float* part_o;                   // [splits][rows][heads][dim] sums of terms times values
  float2* part_ml;                 // [splits][rows][heads] (reference maximum, sum of terms), in log2 units
};

template <int D>
struct PrefillTile {
  static constexpr int kAtoms = D / 64;                    // 128-byte wide columns of a tile
  static constexpr int kTileBytes = kPfRows * D * 2;       // one Q, K or V tile
  static constexpr int kSlots = 5;
  static constexpr int kOffKv = 2 * kTileBytes;
  static constexpr int kOffBar = kOffKv + kSlots * kTileBytes;
  static constexpr int kSmem = kOffBar + 512 + 1024;
  static constexpr int kTmemO = 256;                       // S_0, S_1: columns 0 and 128; O_0, O_1: from 256
};

namespace {

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
      "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The MMA warp runs as a whole and issues under a predicate that one lane
// has: in code that only one lane executes, every descriptor has to be moved
// to the uniform registers that tcgen05 instructions take, some 100 clocks
// per MMA (measured), against the 64 that it executes for.

// D[tmem] (+)= A[smem] * B[smem], one CTA
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                           uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                           uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
// Arrives on `bar` when every tcgen05 operation issued so far by the leader is done.
__device__ __forceinline__ void umma_commit(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(r));
  return r;
}

// MN-major operand with 128-byte swizzle: 64 columns (128 bytes) by 8 rows
// per 1024-byte atom; the next 8 rows 1024 bytes on (stride byte offset), the
// next 64 columns a whole 128-row column block on (leading byte offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((kPfRows * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> struct Type16;
template <> struct Type16<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;                 // instruction descriptor's operand type
  static constexpr uint32_t kExp = 0x7F807F80u, kOne = 0x00800080u;   // exponent bits, their lowest
  static constexpr float kShift = 0.f;
};
template <> struct Type16<__half> {
  static constexpr uint32_t kFmt = 0;
  static constexpr uint32_t kExp = 0x7C007C00u, kOne = 0x04000400u;
  // terms are kept times 2^6: up to 2^14 with the lazy maximum, and normal
  // fp16 numbers down to 2^-20 of the reference maximum
  static constexpr float kShift = 6.f;
};

// Whether either half of the word is infinite or NaN: the exponent bits all
// set carry into the sign bit.
template <typename T> __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & Type16<T>::kExp) + Type16<T>::kOne) & 0x80008000u;
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kPfThreads, 1)
attn_prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PrefillParams p) {
  using C = PrefillTile<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);  // [2]
  uint64_t* full = q_full + 2;                                        // [slots] a K or V tile has landed
  uint64_t* empty = full + C::kSlots;                                 // [slots] its MMAs are done
  uint64_t* s_full = empty + C::kSlots;                               // [2] scores ready (and O up to date)
  uint64_t* p_ready = s_full + 2;                                     // [2][2] half a tile's probabilities written
  uint64_t* o_full = p_ready + 4;                                     // [2] output complete
  uint64_t* v_full = o_full + 2;                                      // [3] partly seen value tile has landed
  uint64_t* v_ok = v_full + kPfMasked;                                // [3] ... and is cleaned
  uint64_t* done = v_ok + kPfMasked;                                  // [1] every MMA is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  uint32_t* poison = tmem_slot + 1;                                   // [3][4] keys with values that are not finite
  // the item, for the softmax warps: read where it is used, so that it takes
  // no registers in their loop (a few spilled ones there cost 4 %)
  volatile int* ctx = reinterpret_cast<volatile int*>(poison + 4 * kPfMasked);
  enum { kCtxQ0, kCtxLq, kCtxR0, kCtxH, kCtxOff, kCtxLk, kCtxJm, kCtxK0, kCtxNk };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 256) {   // the tensor maps' descriptors, fetched while the item is found
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  // This CTA's item: rows r0 .. of sequence b, head h.  Items are taken in
  // order of the tile's place in its sequence, the last places of all
  // sequences first (they see the most keys, and the longest work starts
  // earliest).  left(t) items lie at place t or later; b = B stands for the
  // rows behind the last sequence.
  const int split = blockIdx.x % p.splits;
  const int item = blockIdx.x / p.splits;
  auto tiles_of = [&](int i) {
    if (i > p.B) return 0;
    const int lo = min(max(p.cu_q[i], 0), p.rows), hi = i < p.B ? min(max(p.cu_q[i + 1], lo), p.rows) : p.rows;
    return (hi - lo + 2 * kPfRows - 1) / (2 * kPfRows);
  };
  const int mine0 = tiles_of(lane);            // sequences 0 .. 31 are kept in registers
  auto left = [&](int t) {
    int n = max(0, mine0 - t);
    for (int b0 = 32; b0 <= p.B; b0 += 32) n += max(0, tiles_of(b0 + lane) - t);
    return __reduce_add_sync(0xffffffffu, n);
  };
  int place = 0, b = -1, h = 0;
  {
    if (item >= left(0) * p.heads) return;
    int most = mine0;
    for (int b0 = 32; b0 <= p.B; b0 += 32) most = max(most, tiles_of(b0 + lane));
    int hi = __reduce_max_sync(0xffffffffu, most);   // left(hi) = 0
    while (hi - place > 1) {                         // the largest place with left(place) * heads > item
      const int mid = (place + hi) >> 1;
      if (left(mid) * p.heads > item) place = mid;
      else hi = mid;
    }
    const int rest = item - left(place + 1) * p.heads;
    int nth = rest / p.heads;                        // of the sequences that have such a place
    h = rest - nth * p.heads;
    for (int b0 = 0; b0 <= p.B && b < 0; b0 += 32) {
      unsigned has = __ballot_sync(0xffffffffu, (b0 ? tiles_of(b0 + lane) : mine0) > place);
      if (nth >= __popc(has)) {
        nth -= __popc(has);
        continue;
      }
      for (; nth > 0; --nth) has &= has - 1;
      b = b0 + __ffs(has) - 1;
    }
  }
  const int hk = h / p.group;
  const int q0 = min(max(p.cu_q[b], 0), p.rows);
  const int lq = (b < p.B ? min(max(p.cu_q[b + 1], q0), p.rows) : p.rows) - q0;
  int k0 = b < p.B ? min(max(p.cu_k[b], 0), p.k_rows) : 0;
  int lk = b < p.B ? min(max(p.cu_k[b + 1], k0), p.k_rows) - k0 : 0;
  if (threadIdx.x == 0 && b < p.B && (q0 != p.cu_q[b] || lq != p.cu_q[b + 1] - q0 || k0 != p.cu_k[b] ||
                                      lk != p.cu_k[b + 1] - k0))
    report_error(kErrBadPage);
  const int r0 = place * 2 * kPfRows;
  int off = lk - lq;                                 // row i sees keys j <= i + off
  // key tiles of each row tile (0: no rows, or none that sees a key)
  int nk[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int begin = r0 + s * kPfRows, end = min(lq, begin + kPfRows);
    nk[s] = begin < lq && end + off > 0 ? (end + off + kPfRows - 1) / kPfRows : 0;
  }
  T* out = static_cast<T*>(p.out);
  // this split's key tiles are j0 .. : from here on keys are counted from there
  if (p.splits > 1) {
    const int all = max(nk[0], nk[1]), share = (all + p.splits - 1) / p.splits, j0 = min(all, split * share);
#pragma unroll
    for (int s = 0; s < 2; ++s) nk[s] = max(0, min(nk[s], j0 + share) - j0);
    k0 += j0 * kPfRows;
    lk -= j0 * kPfRows;
    off -= j0 * kPfRows;
  }
  const int nmax = max(nk[0], nk[1]);
  const int jm = min(nmax, max(0, (r0 + off + 1) / kPfRows));   // tiles from jm on are seen in part by some row
  if (nmax == 0) {                                         // nothing to see: zeros
    const int n = min(2 * kPfRows, lq - r0);
    if (p.splits > 1) {
      for (int r = threadIdx.x; r < n; r += kPfThreads)
        p.part_ml[((int64_t)split * p.rows + q0 + r0 + r) * p.heads + h] = make_float2(-INFINITY, 0.f);
      return;
    }
    for (int e = threadIdx.x; e < n * (D / 8); e += kPfThreads) {
      const int r = e / (D / 8), d = (e - r * (D / 8)) * 8;
      *reinterpret_cast<uint4*>(out + ((int64_t)(q0 + r0 + r) * p.heads + h) * D + d) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }

  // the loader's thread sets up the barriers and starts the first copies
  // before the CTA meets
  auto load = [&](const CUtensorMap* map, uint8_t* dst, int head, int row, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, C::kTileBytes);
#pragma unroll
    for (int a = 0; a < C::kAtoms; ++a) tma_load_3d(dst + a * kPfRows * 128, map, a * 64, head, row, bar);
  };
  if (threadIdx.x == 256) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[2 * s], 4);
      mbar_init(&p_ready[2 * s + 1], 4);
      mbar_init(&o_full[s], 1);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kPfMasked; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ok[i], 2);
    }
    mbar_init(done, 1);
    fence_mbar_init();
    if (nk[0]) load(&qmap, smem, h, q0 + r0, &q_full[0]);
    load(&kmap, smem + C::kOffKv, hk, k0, &full[0]);
    if (nk[1]) load(&qmap, smem + C::kTileBytes, h, q0 + r0 + kPfRows, &q_full[1]);
  }
  if (threadIdx.x < 4 * kPfMasked) poison[threadIdx.x] = 0u;
  if (threadIdx.x == 0) {
    ctx[kCtxQ0] = q0;
    ctx[kCtxLq] = lq;
    ctx[kCtxR0] = r0;
    ctx[kCtxH] = h;
    ctx[kCtxOff] = off;
    ctx[kCtxLk] = lk;
    ctx[kCtxJm] = jm;
    ctx[kCtxK0] = k0;
    ctx[kCtxNk] = nk[0];
    ctx[kCtxNk + 1] = nk[1];
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8 && lane == 0) {
      // loader: ring position 2 j holds K_j, 2 j + 1 holds V_j; K_0 and the
      // queries are on their way
      int n = 1;
      for (; n < 2 * nmax; ++n) {
        const int s = n % C::kSlots;
        if (n >= C::kSlots && !mbar_wait(&empty[s], ((n / C::kSlots) - 1) & 1)) break;
        // a partly seen value tile goes to the cleaning warps: it has a
        // barrier of its own, and the slot's passes on to the next phase
        const bool masked = (n & 1) && (n >> 1) >= jm;
        if (masked) mbar_arrive(&full[s]);
        load((n & 1) ? &vmap : &kmap, smem + C::kOffKv + s * C::kTileBytes, hk, k0 + (n >> 1) * kPfRows,
             masked ? &v_full[(n >> 1) - jm] : &full[s]);
      }
      // no copy is left in flight, whatever became of its readers
      for (int i = max(0, n - C::kSlots); i < n; ++i)
        mbar_wait((i & 1) && (i >> 1) >= jm ? &v_full[(i >> 1) - jm] : &full[i % C::kSlots],
                  (i & 1) && (i >> 1) >= jm ? 0 : (i / C::kSlots) & 1);
      if (nk[0]) mbar_wait(&q_full[0], 0);
      if (nk[1]) mbar_wait(&q_full[1], 0);
    } else if (warp == 9) {
      constexpr uint32_t kFmt = (1u << 4) | (Type16<T>::kFmt << 7) | (Type16<T>::kFmt << 10) |
                                ((uint32_t)(kPfRows >> 4) << 24);
      constexpr uint32_t kIdS = kFmt | ((uint32_t)(kPfRows >> 3) << 17);
      constexpr uint32_t kIdO = kFmt | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // B is MN-major
      const uint32_t leader = elect_one();
      // warp-uniform copies of what the loop depends on
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const int un[2] = {__shfl_sync(0xffffffffu, nk[0], 0), __shfl_sync(0xffffffffu, nk[1], 0)};
      const int umax = max(un[0], un[1]), um = __shfl_sync(0xffffffffu, jm, 0);
      const uint64_t dq = umma_desc_sw128(base), dk = umma_desc_sw128(base + C::kOffKv), dv = umma_desc_mn_sw128(base + C::kOffKv);
      constexpr uint32_t kStep = C::kTileBytes >> 4;
      auto scores = [&](int s, uint32_t slot) {            // S_s = Q_s K^T, K in ring slot `slot`
        const uint64_t da = dq + s * kStep, db = dk + slot * kStep;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = ((k >> 2) * (kPfRows * 128) + (k & 3) * 32) >> 4;
          mma_f16_ss(tm + s * kPfRows, da + o, db + o, kIdS, k > 0, leader);
        }
        umma_commit(&s_full[s], leader);
      };
      auto values = [&](int s, uint32_t slot, int half, uint32_t acc) {   // O_s += P_s V, one half of the keys
        const uint64_t db = dv + slot * kStep;
#pragma unroll
        for (int i = 0; i < kPfRows / 32; ++i) {
          const int k = half * (kPfRows / 32) + i;
          mma_f16_ts(tm + C::kTmemO + s * 128, tm + s * kPfRows + k * 8, db + k * (2048 >> 4), kIdO, acc | (k > 0), leader);
        }
      };
      // ring slot and phase of the tile that is waited for next
      uint32_t slot = 0, phase = 0;
      auto advance = [&]() {
        if (++slot == (uint32_t)C::kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      // V_j and, unless it is the last, K_(j + 1) are in their slots
      uint32_t vslot = 0, kslot = 0;
      auto landed = [&](int j, uint32_t& v, uint32_t& k) {
        v = slot;
        bool r = j < um ? mbar_wait(&full[slot], phase) : mbar_wait(&v_ok[j - um], 0);
        advance();
        k = slot;
        if (r && j + 1 < umax) r = mbar_wait(&full[slot], phase);
        advance();
        return r;
      };
      bool ok = mbar_wait(&full[0], 0);
      advance();
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (ok && un[s]) {
          ok = mbar_wait(&q_full[s], 0);
          if (ok) scores(s, 0);
        }
      if (ok) umma_commit(&empty[0], leader);
      ok = ok && landed(0, vslot, kslot);
      for (int j = 0; j < umax && ok; ++j) {
        uint32_t vnext = 0, knext = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (j < un[s] && ok) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && mbar_wait(&p_ready[2 * s + half], j & 1);
              tc_fence_after();
              if (ok) values(s, vslot, half, j > 0);
            }
            if (ok) {
              if (j + 1 < un[s]) scores(s, kslot);
              else umma_commit(&o_full[s], leader);
            }
          }
          // the next tiles are waited for while the tensor core is busy
          if (s == 0 && ok && j + 1 < umax) ok = landed(j + 1, vnext, knext);
        }
        if (!ok) break;
        umma_commit(&empty[vslot], leader);
        if (j + 1 < umax) umma_commit(&empty[kslot], leader);
        vslot = vnext;
        kslot = knext;
      }
      umma_commit(done, leader);               // the tensor memory is not freed under an MMA
      mbar_wait(done, 0);
    } else if (warp >= 10) {
      for (int j = jm; j < nmax; ++j) {
        const int n = 2 * j + 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&v_full[j - jm], 0))) break;
        uint8_t* tile = smem + C::kOffKv + (n % C::kSlots) * C::kTileBytes;
        const int keys = min(kPfRows, lk - j * kPfRows);
        // 16-byte pieces, 8 to a 128-byte row, eight of them at a time: one
        // by one this took longer than a tile's MMAs and softmax
        constexpr int kBatch = 8;
        uint4* at = reinterpret_cast<uint4*>(tile) + (threadIdx.x - 320);
#pragma unroll 1
        for (int c0 = 0; c0 < C::kTileBytes / 16; c0 += 64 * kBatch, at += 64 * kBatch) {
          uint4 w[kBatch];
          uint32_t bad = 0;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) w[i] = at[i * 64];
          auto key_of = [&](int i) { return ((c0 + i * 64 + (int)threadIdx.x - 320) >> 3) % kPfRows; };
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const uint32_t b = not_finite<T>(w[i].x) | not_finite<T>(w[i].y) | not_finite<T>(w[i].z) | not_finite<T>(w[i].w);
            if (key_of(i) < keys) bad |= b;
            else at[i * 64] = make_uint4(0u, 0u, 0u, 0u);
          }
          if (bad) {
#pragma unroll 1
            for (int i = 0; i < kBatch; ++i) {
              const int key = key_of(i);
              uint4 v = at[i * 64];
              if (key >= keys || !(not_finite<T>(v.x) | not_finite<T>(v.y) | not_finite<T>(v.z) | not_finite<T>(v.w))) continue;
              atomicOr(&poison[(j - jm) * 4 + (key >> 5)], 1u << (key & 31));
              uint32_t* x = &v.x;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t b = not_finite<T>(x[k]);
                if (b & 0x8000u) x[k] &= 0xffff0000u;
                if (b & 0x80000000u) x[k] &= 0x0000ffffu;
              }
              at[i * 64] = v;
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[j - jm]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int s = warp >> 2, quarter = warp & 3;
    const uint32_t t_s = tmem + s * kPfRows + ((uint32_t)(quarter * 32) << 16);
    const uint32_t t_o = tmem + C::kTmemO + s * 128 + ((uint32_t)(quarter * 32) << 16);
    const int n = ctx[kCtxNk + s];
    // keys this row sees, and the tile's first row
    const int seen_by_all = ctx[kCtxR0] + s * kPfRows + ctx[kCtxOff] + 1;
    const int see = min(ctx[kCtxLk], seen_by_all + quarter * 32 + lane);
    float m = -INFINITY, sum = 0.f;                              // reference maximum of the raw scores, sum of terms
    const float scale = p.scale_log2;
    bool fail = false;
    for (int j = 0; j < n; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[s], j & 1))) {
        fail = true;
        break;
      }
      tc_fence_after();
      uint32_t x[4][32];
      const int here = see - j * kPfRows;
      const bool masked = (j + 1) * kPfRows > seen_by_all;
      float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, x[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[c][i] = c * 32 + i < here ? x[c][i] : 0xff800000u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            top4[k] = fmaxf(fmaxf(top4[k], __uint_as_float(x[c][i + 2 * k])), __uint_as_float(x[c][i + 2 * k + 1]));
      }
      const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
      // a new reference maximum where the terms would pass 2^8
      const bool grow = top > m && (m == -INFINITY || (top - m) * scale > 8.f);
      if (__any_sync(0xffffffffu, grow)) {
        const float a = grow ? (m == -INFINITY ? 0.f : ex2((m - top) * scale)) : 1.f;
        if (grow) {
          m = top;
          sum *= a;
        }
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(t_o + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
            tmem_st16(t_o + c * 16, o);
          }
        }
      }
      const float neg = m == -INFINITY ? 0.f : Type16<T>::kShift - m * scale;
      const float2 scale2 = make_float2(scale, scale), neg2 = make_float2(neg, neg);
      float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      // the first half of the keys goes to the tensor core while the second
      // half's exponentials are computed
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 v = __ffma2_rn(
                make_float2(__uint_as_float(x[half * 2 + c][i]), __uint_as_float(x[half * 2 + c][i + 1])), scale2, neg2);
            const float2 e = make_float2(ex2(v.x), ex2(v.y));
            part[(i >> 1) & 1] = __fadd2_rn(part[(i >> 1) & 1], e);
            w[c * 16 + (i >> 1)] = pack16<T>(e.x, e.y);
          }
        tmem_st32(t_s + half * 32, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * s + half]);
      }
      sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
    }
    const int e_q0 = ctx[kCtxQ0], e_lq = ctx[kCtxLq], e_h = ctx[kCtxH], e_k0 = ctx[kCtxK0], e_jm = ctx[kCtxJm];
    const int first = ctx[kCtxR0] + s * kPfRows + quarter * 32, row = first + lane;   // within the sequence
    const bool live = row < e_lq;
    const int64_t at = ((int64_t)(blockIdx.x % p.splits) * p.rows + e_q0 + row) * p.heads + e_h;   // splits: partial row
    T* dst = static_cast<T*>(p.out) + ((int64_t)(e_q0 + row) * p.heads + e_h) * D;
    if (n && !fail && __all_sync(0xffffffffu, mbar_wait(&o_full[s], 0))) {
      tc_fence_after();
      // The rows go through shared memory (the tile's queries have been
      // used), so that a store instruction writes whole rows: one row per lane
      // is one line per lane, and the stores took 2 us per CTA.
      constexpr int kPieces = D / 8;
      uint4* stage = reinterpret_cast<uint4*>(smem + s * C::kTileBytes) + quarter * 32 * kPieces;
      // a split leaves its sums as they are, to be joined
      const bool whole = p.splits == 1;
      const float inv = !whole ? 1.f : see > 0 ? 1.f / sum : 0.f;
      if (!whole && live) p.part_ml[at] = make_float2(sum == 0.f ? -INFINITY : m * scale, sum);
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < 4 * kPfMasked; ++i) any |= poison[i];
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(t_o + c * 32, o);
        tmem_wait_ld();
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = see > 0 ? __uint_as_float(o[i]) * inv : 0.f;
        if (any) {
          for (int i = 0; i < 4 * kPfMasked; ++i) {
            uint32_t bits = poison[i];
            while (bits) {
              const int key = e_jm * kPfRows + i * 32 + __ffs(bits) - 1;
              bits &= bits - 1;
              if (key >= see) continue;
              const T* vr = static_cast<const T*>(p.v) + (int64_t)(e_k0 + key) * p.sv_t + (int64_t)(e_h / p.group) * p.sv_h + c * 32;
#pragma unroll
              for (int d = 0; d < 32; ++d) {
                const float v = to_f32(vr[d]);
                if (!isfinite(v)) f[d] += v;
              }
            }
          }
        }
        if (live && !whole) {
          float* po = p.part_o + at * D + c * 32;
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(po + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        } else if (whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            stage[lane * kPieces + ((c * 4 + i) ^ (lane & 7))] =
                make_uint4(pack16<T>(f[8 * i], f[8 * i + 1]), pack16<T>(f[8 * i + 2], f[8 * i + 3]),
                           pack16<T>(f[8 * i + 4], f[8 * i + 5]), pack16<T>(f[8 * i + 6], f[8 * i + 7]));
        }
      }
      if (whole) {
        __syncwarp();
        const int rows = min(32, e_lq - first);
#pragma unroll 4
        for (int i = lane; i < rows * kPieces; i += 32) {
          const int r = i / kPieces, c = i - r * kPieces;
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + ((int64_t)(e_q0 + first + r) * p.heads + e_h) * D + c * 8) =
              stage[r * kPieces + (c ^ (r & 7))];
        }
      }
    } else if (!n && live && p.splits > 1) {                     // this tile's rows see nothing here
      p.part_ml[at] = make_float2(-INFINITY, 0.f);
    } else if (!n && live) {
#pragma unroll 1
      for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
}

// Joins the splits' partial results: one thread per four columns.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_prefill_join_kernel(const __grid_constant__ PrefillParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t n = (int64_t)p.rows * p.heads, e = (int64_t)blockIdx.x * 256 + threadIdx.x, at = e / (D / 4);
  if (at >= n) return;
  const int d = (int)(e - at * (D / 4)) * 4;
  float2 ml[kPfSplits];
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPfSplits; ++i) {
    ml[i] = i < p.splits ? p.part_ml[i * n + at] : make_float2(-INFINITY, 0.f);
    mx = fmaxf(mx, ml[i].x);
  }
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPfSplits; ++i) {
    if (ml[i].y == 0.f) continue;                          // this split saw nothing (its values are not set)
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + (i * n + at) * D + d);
    const float f = exp2f(ml[i].x - mx);
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
    sum = fmaf(ml[i].y, f, sum);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const T o[4] = {from_f32<T>(acc.x * inv), from_f32<T>(acc.y * inv), from_f32<T>(acc.z * inv), from_f32<T>(acc.w * inv)};
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * D + d) = *reinterpret_cast<const uint2*>(o);
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------
// [tokens][heads][dim] with the given element strides; boxes of 128 tokens
// by 64 columns of one head.
static bool encode_rows(CUtensorMap* map, const void* base, int dtype, int64_t rows, int heads, int dim, int64_t st_t,
                        int64_t st_h) {
  auto encode = get_encode();
  if (!encode) return false;
  // the stride of a dimension of one element is not used, but has to be valid
  if (heads == 1) st_h = dim;
  if (rows == 1) st_t = dim;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)st_h * 2, (cuuint64_t)st_t * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)kPfRows}, estr[3] = {1, 1, 1};
  return encode(map, dtype == PARO_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
static cudaError_t launch_prefill(const CUtensorMap* maps, const PrefillParams& p, int64_t slots, cudaStream_t st) {
  using C = PrefillTile<D>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(attn_prefill_kernel<T, D>), C::kSmem);
  if (e != cudaSuccess) return e;
  attn_prefill_kernel<T, D><<<(unsigned)(slots * p.heads * p.splits), kPfThreads, C::kSmem, st>>>(maps[0], maps[1],
                                                                                                  maps[2], p);
  if ((e = cudaGetLastError()) != cudaSuccess || p.splits == 1) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((int64_t)p.rows * p.heads * (D / 4) + 255) / 256));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_prefill_join_kernel<T, D>, p);
}

// Into how many CTAs an item's keys are split.  An item (256 rows of one
// head) takes as long as its keys whatever the number of rows, so where the
// items do not fill the SMs and the sequences are long, sharing the keys out
// shortens the call; the number of items is estimated as one per 256 rows and
// half a one more per sequence.  Two calls at 16 heads of 64: 901 queries
// behind 6596 keys 66 us unsplit, 39 us in two.
static int prefill_splits(int B, int64_t rows, int64_t k_rows, int heads) {
  const int64_t items = (rows / (2 * kPfRows) + (B + 1) / 2) * heads;
  const int64_t by_sms = items > 0 ? (sm_count() + sm_count() / 4) / items : 1;
  const int64_t by_keys = B > 0 ? k_rows / B / (4 * kPfRows) : 1;      // at least four key tiles each
  const int64_t n = by_sms < by_keys ? by_sms : by_keys;
  return n < 1 ? 1 : n > kPfSplits ? kPfSplits : (int)n;
}

size_t attn_prefill_workspace(int B, int64_t rows, int64_t k_rows, int heads, int dim) {
  const int n = prefill_splits(B, rows, k_rows, heads);
  return n == 1 ? 0 : (size_t)n * rows * heads * (dim * 4 + 8);
}

cudaError_t launch_attn_prefill(const void* q, const void* k, const void* v, int dtype, const int64_t* s,
                                const int32_t* cu_q, const int32_t* cu_k, int B, int64_t rows, int64_t k_rows,
                                int heads, int kv_heads, int dim, float scale, void* out, void* workspace, cudaStream_t st) {
  if (k_rows == 0) return cudaMemsetAsync(out, 0, (size_t)rows * heads * dim * 2, st);
  CUtensorMap maps[3];
  if (!encode_rows(&maps[0], q, dtype, rows, heads, dim, s[0], s[1]) ||
      !encode_rows(&maps[1], k, dtype, k_rows, kv_heads, dim, s[2], s[3]) ||
      !encode_rows(&maps[2], v, dtype, k_rows, kv_heads, dim, s[4], s[5]))
    return cudaErrorInvalidValue;
  // a scale of zero still has to leave -infinity where a key is not seen
  const float scale_log2 = fmaxf(scale * 1.4426950408889634f, 1e-37f);
  const int splits = workspace ? prefill_splits(B, rows, k_rows, heads) : 1;
  float* po = static_cast<float*>(workspace);
  const PrefillParams p{cu_q, cu_k, B, heads, heads / kv_heads, (int)rows, (int)k_rows, scale_log2, out, v, s[4], s[5],
                        splits, po, reinterpret_cast<float2*>(po + (size_t)splits * rows * heads * dim)};
  // at most one item more than whole ones per sequence (and for the rows behind the last)
  int64_t slots = rows / (2 * kPfRows) + B + 1;
  if (slots > rows) slots = rows;
  if (slots * heads * splits > 0x7FFFFFFF || rows * heads * (dim / 4) / 256 >= 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (dtype == PARO_BF16)
    return dim == 128 ? launch_prefill<__nv_bfloat16, 128>(maps, p, slots, st)
                      : launch_prefill<__nv_bfloat16, 64>(maps, p, slots, st);
  return dim == 128 ? launch_prefill<__half, 128>(maps, p, slots, st) : launch_prefill<__half, 64>(maps, p, slots, st);
}

}  // namespace paro
