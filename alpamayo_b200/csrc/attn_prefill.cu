// attn_prefill.cu — causal attention over packed prompts with grouped heads,
// on the 5th-generation tensor cores (sm_100a).
//
//   o_i = sum_{j <= i + Lk - Lq} softmax_j(scale * q_i . k_j) v_j
//
// An item is 256 query rows of one sequence and head: two tiles of 128 rows
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
//  * warp 8: finds the items and loads their tiles with TMA, K_0 V_0 K_1 V_1
//    ... through one ring that runs on from item to item.  The launch has a
//    CTA per item; one that is running takes over the items of those that
//    have not started (the hardware's cancel request), so the next item's
//    queries, first keys and first scores are under way while the softmax
//    warps store the last one's output.  28 heads, 8 prompts of 1 to 1500
//    tokens (560 items of 1 to 12 tiles): 61 us with an item per CTA, 58 with
//    the items shared out evenly beforehand, 53 like this; one prompt of 8192
//    gains 1 %; one of 37, whose items have a CTA each either way, takes 8.6
//    us for 7.5 (the hand-over of its description).
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
#include <cfloat>

#include "umma.cuh"

namespace paro {

PARO_DEFINE_ERROR_ACCESSOR(attn)

constexpr int kPfRows = 128;       // query rows per tile, keys per tile
constexpr int kPfThreads = 384;
constexpr int kPfSplits = 8;       // splits of an item's keys, at most
constexpr int kPfMasked = 3;       // key tiles that a CTA's rows see in part, at most
constexpr float kInPlace = -1.f;

// Division of 0 .. 2^31 - 1 by a divisor that the host knows: the rounded-up
// reciprocal gives the quotient or one more.
struct Divisor {
  int d;
  uint64_t inv;                    // ceil(2^32 / d)
  explicit Divisor(int d) : d(d), inv(((1ull << 32) + d - 1) / d) {}
  __device__ __forceinline__ int operator()(int n) const {
    const int q = (int)(((uint64_t)n * inv) >> 32);
    return q - ((int64_t)q * d > n);
  }
};

struct PrefillParams {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, heads, group;
  int rows, k_rows;
  float scale_log2;
  void* out;
  const void* v;                   // for the values that are not finite
  int64_t sv_t, sv_h;
  Divisor by_heads, by_group;
  int sms;
  int splits;                      // parts that an item's keys may be cut into; > 1: partial results, joined
  float* part_o;                   // [splits][rows][heads][dim] sums of terms times values
  float2* part_ml;                 // [splits][rows][heads] (reference maximum, sum of terms), in log2 units; a
                                   // sum of kInPlace, which no sum of terms is: one part, the row is in `out`
};

template <int D>
struct PrefillTile {
  static constexpr int kAtoms = D / 64;                    // 128-byte wide columns of a tile
  static constexpr int kTileBytes = kPfRows * D * 2;       // one Q, K or V tile
  static constexpr int kSlots = D == 128 ? 4 : 6;
  static constexpr int kOffKv = 2 * kTileBytes;
  static constexpr int kOffStage = kOffKv + kSlots * kTileBytes;   // [8 warps][32 rows][64 columns] output on its way
  static constexpr int kOffBar = kOffStage + 8 * 32 * 128;
  static constexpr int kSmem = kOffBar + 768 + 1024;
  static constexpr int kTmemO = 256;                       // S_0, S_1: columns 0 and 128; O_0, O_1: from 256
};

// An item as the loader hands it to the other warps.
enum { kCtxStop, kCtxQ0, kCtxLq, kCtxR0, kCtxH, kCtxOff, kCtxLk, kCtxJm, kCtxK0, kCtxNk, kCtxSplit = kCtxNk + 2, kCtxParts, kCtxLead, kCtxWords };

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

// 256-row items of sequence i (i = B: the rows behind the last sequence).
// The rows before the first sequence are in front of its own in its items; they
// give zeros.
__device__ __forceinline__ int prefill_tiles(const PrefillParams& p, int i) {
  if (i > p.B) return 0;
  const int lo = i == 0 ? 0 : min(max(p.cu_q[i], 0), p.rows), hi = i < p.B ? min(max(p.cu_q[i + 1], lo), p.rows) : p.rows;
  return (hi - lo + 2 * kPfRows - 1) / (2 * kPfRows);
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
  uint4* next = reinterpret_cast<uint4*>(smem + C::kOffBar);          // [1] answer to a request for the next item
  uint64_t* next_full = reinterpret_cast<uint64_t*>(next + 1);        // [1] it has come
  uint64_t* ctx_full = next_full + 1;                                 // [2] an item's description is written
  uint64_t* ctx_empty = ctx_full + 2;                                 // [2] every warp is done with the item
  uint64_t* q_full = ctx_empty + 2;                                   // [2] queries have landed
  uint64_t* q_empty = q_full + 2;                                     // [2] their last scores are done
  uint64_t* full = q_empty + 2;                                       // [slots] a K or V tile has landed
  uint64_t* empty = full + C::kSlots;                                 // [slots] its MMAs are done
  uint64_t* s_full = empty + C::kSlots;                               // [2] scores ready (and O up to date)
  uint64_t* p_ready = s_full + 2;                                     // [2][2] half a tile's probabilities written
  uint64_t* o_full = p_ready + 4;                                     // [2] output complete
  uint64_t* v_full = o_full + 2;                                      // [2][3] partly seen value tile has landed
  uint64_t* v_ok = v_full + 2 * kPfMasked;                            // [2][3] ... and is cleaned
  uint64_t* done = v_ok + 2 * kPfMasked;                              // [1] every MMA is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  uint32_t* poisons = tmem_slot + 1;                                  // [2][3][4] keys with values that are not finite
  // The items' descriptions, two deep; the softmax warps read them where they
  // use them, so that they take no registers in their loop (a few spilled
  // ones there cost 4 %).
  volatile int* ctxs = reinterpret_cast<volatile int*>(poisons + 2 * 4 * kPfMasked);   // [2][kCtxWords]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the loader's lanes keep sequences 0 .. 31: offsets of queries and keys, items
  const int cu_q0 = warp == 8 && lane <= p.B ? p.cu_q[lane] : 0, cu_k0 = warp == 8 && lane <= p.B ? p.cu_k[lane] : 0;
  const int mine0 = warp == 8 ? prefill_tiles(p, lane) : 0;
  if (threadIdx.x == 352) {
    // the tensor maps' descriptors, fetched while the first item is found
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  if (threadIdx.x == 320) {
    mbar_init(next_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctx_full[s], 1);
      mbar_init(&ctx_empty[s], 11);     // 8 softmax warps, the MMA warp, 2 cleaning warps
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[2 * s], 4);
      mbar_init(&p_ready[2 * s + 1], 4);
      mbar_init(&o_full[s], 1);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2 * kPfMasked; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ok[i], 2);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 10) {                            // the loader goes on as soon as the barriers are there
    __syncwarp();
    asm volatile("bar.arrive 1, 64;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // 256 x 176 + 128 x 152 = 384 x 168 registers.  The softmax warps need no
  // more than 176; with 184 to 200 of them the same code took up to 3 % longer
  // or the other warps' spilled.
  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 152;");
  // Every warp meets here but the loader's, which needs nothing of the others
  // and has begun by now.
  if (warp == 8) {
    asm volatile("bar.arrive 2, 384;" ::: "memory");
    asm volatile("bar.sync 1, 64;" ::: "memory");
  } else {
    tc_fence_before();
    asm volatile("bar.sync 2, 384;" ::: "memory");
    tc_fence_after();
  }
  const uint32_t tmem = warp == 8 ? 0u : *tmem_slot;
  auto all_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };

  if (warp >= 8) {
    if (warp == 8) {
      // Loader.  The whole warp finds the next item; one lane loads.
      auto left = [&](int t) {                             // items of one head at place t or later
        int n = max(0, mine0 - t);
        for (int b0 = 32; b0 <= p.B; b0 += 32) n += max(0, prefill_tiles(p, b0 + lane) - t);
        return __reduce_add_sync(0xffffffffu, n);
      };
      const int items = left(0) * p.heads;
      // Where keys may be shared out, an item of more than `part` key tiles is
      // cut into parts.  A part is an SM's share of the work (an item costs
      // about three tiles besides its own), four tiles at least, or up to half
      // as much more if that leaves no more parts than SMs.
      int part = 0x7FFFFFFF, parts = 1;
      if (p.splits > 1) {
        auto key_tiles = [&](int b) {
          const int lo = min(max(p.cu_k[b], 0), p.k_rows);
          return (min(max(p.cu_k[b + 1], lo), p.k_rows) - lo + kPfRows - 1) / kPfRows;
        };
        float work = 0.f;
        int longest = 0;
        for (int b = lane; b < p.B; b += 32) {
          const int n = prefill_tiles(p, b), tiles = n ? key_tiles(b) : 0;
          longest = max(longest, tiles);
          // a place of a sequence sees two key tiles fewer than the next one
          work += fmaxf((float)n * (float)(tiles - n + 1), (float)tiles) + 3.f * n;
        }
#pragma unroll
        for (int i = 16; i; i >>= 1) work += __shfl_xor_sync(0xffffffffu, work, i);
        longest = __reduce_max_sync(0xffffffffu, longest);
        const int share = max(max(4, (longest + p.splits - 1) / p.splits),
                              (int)fminf(ceilf(work * (float)p.heads / (float)p.sms), (float)longest));
        part = share;
#pragma unroll 1
        for (int i = 0; i <= 4 && items <= p.sms; ++i) {
          part = share + share * i / 8;
          int n = 0;
          for (int b = lane; b < p.B; b += 32) {
            const int tiles = key_tiles(b);
            for (int k = prefill_tiles(p, b) - 1, t = tiles; k >= 0; --k, t -= 2) n += max(1, (t + part - 1) / part);
          }
          if (__reduce_add_sync(0xffffffffu, n) * p.heads <= p.sms) break;
        }
        parts = max(1, (longest + part - 1) / part);
      }
      const int total = items * parts;
      auto load = [&](const CUtensorMap* map, uint8_t* dst, int head, int row, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, C::kTileBytes);
#pragma unroll
        for (int a = 0; a < C::kAtoms; ++a) tma_load_3d(dst + a * kPfRows * 128, map, a * 64, head, row, bar);
      };
      uint32_t slot = 0, phase = 1;                        // ring: a fresh `empty` passes for the first round
      uint32_t q_phase[2] = {1u, 1u}, v_phase = 0, asked = 0;
      bool ok = true, open = false;              // open: a request has no answer yet
      int it = blockIdx.x;
      bool first = true;
      for (int n = 0; ok;) {
        const int c = n & 1;
        if (n >= 2 && !all_wait(&ctx_empty[c], ((n >> 1) - 1) & 1)) break;
        // Items in order of their place in their sequence, the last places of
        // all sequences first (they see the most keys).  A CTA takes over the
        // items of CTAs that have not started, one while it works on the last.
        // (With no more items than SMs each has a CTA already; a CTA without
        // one clears away the others without one, which is quicker than
        // starting them.)
        // Parts beyond the launch's CTAs go to them in turn.
        const bool turn = !first && it + (int)gridDim.x < total;
        const bool claim = !turn && (first ? it >= total : total > p.sms);
        it = turn ? it + (int)gridDim.x : first && !claim ? it : -1;
        while (claim) {
          if (lane == 0) {
            mbar_arrive_expect_tx(next_full, 16);
            asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                         ::"r"(smem_u32(next)), "r"(smem_u32(next_full)) : "memory");
          }
          open = true;
          if (!all_wait(next_full, asked & 1)) break;
          open = false;
          ++asked;
          uint4 w;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(smem_u32(next)) : "memory");
          uint32_t taken = 0, x = 0;
          asm volatile(
              "{\n.reg .pred p;\n.reg .b128 a;\n.reg .b64 lo, hi;\n"
              "mov.b64 lo, {%2, %3};\nmov.b64 hi, {%4, %5};\nmov.b128 a, {lo, hi};\n"
              "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n"
              "selp.u32 %0, 1, 0, p;\n"
              "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n}"
              : "=r"(taken), "+r"(x)
              : "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w));
          if (!taken) break;
          fence_proxy_async_smem();                        // this read comes before the next answer
          __syncwarp();
          if ((int)x < total) {
            it = (int)x;
            break;
          }
        }
        first = false;
        volatile int* ctx = ctxs + c * kCtxWords;
        if (it < 0 || it >= total) {
          if (lane == 0) {
            ctx[kCtxStop] = 1;
            mbar_arrive(&ctx_full[c]);
          }
          break;
        }
        int item = it, split = 0;
        for (; item >= items; item -= items) ++split;
        int place = 0, hi = p.rows / (2 * kPfRows) + 1, above = 0, b = -1;
        while (hi - place > 1) {                           // the largest place with left(place) * heads > item
          const int mid = (place + hi) >> 1, n_mid = left(mid) * p.heads;
          if (n_mid > item) {
            place = mid;
          } else {
            hi = mid;
            above = n_mid;                                 // items of later places
          }
        }
        const int rest = item - above;
        int nth = p.by_heads(rest);                          // of the sequences that have such a place
        const int h = rest - nth * p.heads, hk = p.by_group(h);
        for (int b0 = 0; b0 <= p.B && b < 0; b0 += 32) {
          unsigned has = __ballot_sync(0xffffffffu, (b0 ? prefill_tiles(p, b0 + lane) : mine0) > place);
          if (nth >= __popc(has)) {
            nth -= __popc(has);
            continue;
          }
          for (; nth > 0; --nth) has &= has - 1;
          b = b0 + __ffs(has) - 1;                         // b = B: the rows behind the last sequence
        }
        // b < 31: from the lanes that keep them
        const bool kept = b < 31, last = b == p.B;
        const int cq0 = __shfl_sync(0xffffffffu, cu_q0, b & 31), cq1 = __shfl_sync(0xffffffffu, cu_q0, (b + 1) & 31);
        const int ck0 = __shfl_sync(0xffffffffu, cu_k0, b & 31), ck1 = __shfl_sync(0xffffffffu, cu_k0, (b + 1) & 31);
        const int bq0 = kept ? cq0 : p.cu_q[b], bq1 = last ? p.rows : kept ? cq1 : p.cu_q[b + 1];
        const int bk0 = last ? 0 : kept ? ck0 : p.cu_k[b], bk1 = last ? 0 : kept ? ck1 : p.cu_k[b + 1];
        const int qb = min(max(bq0, 0), p.rows), q0 = b == 0 ? 0 : qb, lq = min(max(bq1, qb), p.rows) - q0;
        const int lead = qb - q0;                          // rows before the first sequence, in front of its own
        int k0 = min(max(bk0, 0), p.k_rows), lk = min(max(bk1, k0), p.k_rows) - k0;
        if (lane == 0 && !last && (qb != bq0 || lq - lead != bq1 - qb || k0 != bk0 || lk != bk1 - k0)) report_error(kErrBadPage);
        const int r0 = place * 2 * kPfRows;
        int off = lk - lq;                                 // row i sees keys j <= i + off (lead rows: none)
        // key tiles of each row tile (0: no rows, or none that sees a key)
        int nk[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int begin = r0 + s * kPfRows, end = min(lq, begin + kPfRows);
          nk[s] = begin < lq && end + off > 0 ? (end + off + kPfRows - 1) / kPfRows : 0;
        }
        // this part's key tiles are j0 .. : from here on keys are counted from there
        int cut = 1;
        if (parts > 1) {
          const int all = max(nk[0], nk[1]);
          cut = max(1, (all + part - 1) / part);
          if (split >= cut) continue;                      // the item has fewer parts
          const int share = (all + cut - 1) / cut, j0 = min(all, split * share);
#pragma unroll
          for (int s = 0; s < 2; ++s) nk[s] = max(0, min(nk[s], j0 + share) - j0);
          k0 += j0 * kPfRows;
          lk -= j0 * kPfRows;
          off -= j0 * kPfRows;
        }
        const int nmax = max(nk[0], nk[1]);
        const int jm = min(nmax, max(0, (r0 + off + 1) / kPfRows));   // tiles from jm on are seen in part by some row
        if (lane < 4 * kPfMasked) poisons[c * 4 * kPfMasked + lane] = 0u;
        __syncwarp();
        if (lane == 0) {
          ctx[kCtxStop] = 0;
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
          ctx[kCtxSplit] = split;
          ctx[kCtxParts] = cut;
          ctx[kCtxLead] = lead;
          mbar_arrive(&ctx_full[c]);
          // position 2 j of the item is K_j, 2 j + 1 is V_j; the queries come behind K_0
#pragma unroll 1
          for (int i = 0; i < 2 * nmax; ++i) {
            if (i == 1) {
#pragma unroll
              for (int s = 0; s < 2; ++s)
                if (nk[s] && ok) {
                  ok = mbar_wait(&q_empty[s], q_phase[s]);
                  q_phase[s] ^= 1;
                  if (ok) load(&qmap, smem + s * C::kTileBytes, h, q0 + r0 + s * kPfRows, &q_full[s]);
                }
            }
            if (!(ok = ok && mbar_wait(&empty[slot], phase))) break;
            // a partly seen value tile goes to the cleaning warps: it has a
            // barrier of its own, and the slot's passes on to the next phase
            const int k = (i >> 1) - jm;
            const bool part = (i & 1) && k >= 0;
            if (part) mbar_arrive(&full[slot]);
            load((i & 1) ? &vmap : &kmap, smem + C::kOffKv + slot * C::kTileBytes, hk, k0 + (i >> 1) * kPfRows,
                 part ? &v_full[c * kPfMasked + k] : &full[slot]);
            if (part) v_phase ^= 1u << (c * kPfMasked + k);
            if (++slot == (uint32_t)C::kSlots) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        ++n;
      }
      // No copy is left in flight, whatever became of its readers: everything
      // that was issued has landed when each barrier's last phase is over.
      if (lane == 0) {
        if (open) mbar_wait(next_full, asked & 1);
        for (int i = 0; i < C::kSlots; ++i) {
          const uint32_t last = (uint32_t)i < slot ? phase : phase ^ 1;   // the slot's last round, as `empty` counted it
          mbar_wait(&full[i], last ^ 1);
        }
        for (int s = 0; s < 2; ++s) mbar_wait(&q_full[s], q_phase[s]);
        for (int i = 0; i < 2 * kPfMasked; ++i) mbar_wait(&v_full[i], ((v_phase >> i) & 1) ^ 1);
      }
    } else if (warp == 9) {
      constexpr uint32_t kFmt = (1u << 4) | (Type16<T>::kFmt << 7) | (Type16<T>::kFmt << 10) |
                                ((uint32_t)(kPfRows >> 4) << 24);
      constexpr uint32_t kIdS = kFmt | ((uint32_t)(kPfRows >> 3) << 17);
      constexpr uint32_t kIdO = kFmt | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // B is MN-major
      const uint32_t leader = elect_one();
      // warp-uniform copies of what the loop depends on
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const uint64_t dq = umma_desc_sw128(base), dk = umma_desc_sw128(base + C::kOffKv), dv = umma_desc_mn_sw128(base + C::kOffKv);
      constexpr uint32_t kStep = C::kTileBytes >> 4;
      // S_s = Q_s K^T, K in ring slot `slot`; after the item's last ones the
      // queries' place is free
      auto scores = [&](int s, uint32_t slot, bool last) {
        const uint64_t da = dq + s * kStep, db = dk + slot * kStep;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = ((k >> 2) * (kPfRows * 128) + (k & 3) * 32) >> 4;
          mma_f16_ss(tm + s * kPfRows, da + o, db + o, kIdS, k > 0, leader);
        }
        umma_commit(&s_full[s], leader);
        if (last) umma_commit(&q_empty[s], leader);
      };
      auto values = [&](int s, uint32_t slot, int half, uint32_t acc) {   // O_s += P_s V, one half of the keys
        const uint64_t db = dv + slot * kStep;
#pragma unroll
        for (int i = 0; i < kPfRows / 32; ++i) {
          const int k = half * (kPfRows / 32) + i;
          mma_f16_ts(tm + C::kTmemO + s * 128, tm + s * kPfRows + k * 8, db + k * (2048 >> 4), kIdO, acc | (k > 0), leader);
        }
      };
      // ring slot and phase of the tile that is waited for next; phases of
      // the other barriers
      uint32_t slot = 0, phase = 0, p_phase[2] = {0u, 0u}, q_phase[2] = {0u, 0u}, v_phase = 0;
      auto advance = [&]() {
        if (++slot == (uint32_t)C::kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int c = n & 1;
        if (!all_wait(&ctx_full[c], (n >> 1) & 1)) break;
        volatile int* ctx = ctxs + c * kCtxWords;
        if (__shfl_sync(0xffffffffu, ctx[kCtxStop], 0)) break;
        const int un[2] = {__shfl_sync(0xffffffffu, ctx[kCtxNk], 0), __shfl_sync(0xffffffffu, ctx[kCtxNk + 1], 0)};
        const int umax = max(un[0], un[1]), um = __shfl_sync(0xffffffffu, ctx[kCtxJm], 0);
        if (umax) {
          // V_j and, unless it is the last, K_(j + 1) are in their slots
          uint32_t vslot = 0, kslot = 0;
          auto landed = [&](int j, uint32_t& v, uint32_t& k) {
            v = slot;
            const int i = c * kPfMasked + j - um;
            bool r = j < um ? mbar_wait(&full[slot], phase) : mbar_wait(&v_ok[i], (v_phase >> i) & 1);
            if (j >= um) v_phase ^= 1u << i;
            advance();
            if (j + 1 < umax) {
              k = slot;
              if (r) r = mbar_wait(&full[slot], phase);
              advance();
            }
            return r;
          };
          const uint32_t first = slot;
          ok = mbar_wait(&full[slot], phase);
          advance();
#pragma unroll
          for (int s = 0; s < 2; ++s)
            if (ok && un[s]) {
              ok = mbar_wait(&q_full[s], q_phase[s]);
              q_phase[s] ^= 1;
              if (ok) scores(s, first, un[s] == 1);
            }
          if (ok) umma_commit(&empty[first], leader);
          ok = ok && landed(0, vslot, kslot);
          for (int j = 0; j < umax && ok; ++j) {
            uint32_t vnext = 0, knext = 0;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (j < un[s] && ok) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  ok = ok && mbar_wait(&p_ready[2 * s + half], p_phase[s]);
                  tc_fence_after();
                  if (ok) values(s, vslot, half, j > 0);
                }
                p_phase[s] ^= 1;
                if (ok) {
                  if (j + 1 < un[s]) scores(s, kslot, j + 2 == un[s]);
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
        }
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (ok && lane == 0) mbar_arrive(&ctx_empty[c]);
      }
      __syncwarp();
      umma_commit(done, leader);               // the tensor memory is not freed under an MMA
      mbar_wait(done, 0);
    } else {
      uint32_t at_item = 0, v_phase = 0;       // ring position of the item's K_0
      for (int n = 0;; ++n) {
        const int c = n & 1;
        if (!all_wait(&ctx_full[c], (n >> 1) & 1)) break;
        volatile int* ctx = ctxs + c * kCtxWords;
        if (ctx[kCtxStop]) break;
        const int nmax = max(ctx[kCtxNk], ctx[kCtxNk + 1]), jm = ctx[kCtxJm], lk = ctx[kCtxLk];
        uint32_t* poison = poisons + c * 4 * kPfMasked;
        bool ok = true;
        for (int j = jm; j < nmax && ok; ++j) {
          const int v = c * kPfMasked + j - jm;
          ok = all_wait(&v_full[v], (v_phase >> v) & 1);
          v_phase ^= 1u << v;
          if (!ok) break;
          uint8_t* tile = smem + C::kOffKv + ((at_item + 2 * j + 1) % C::kSlots) * C::kTileBytes;
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
                uint4 x4 = at[i * 64];
                if (key >= keys || !(not_finite<T>(x4.x) | not_finite<T>(x4.y) | not_finite<T>(x4.z) | not_finite<T>(x4.w)))
                  continue;
                atomicOr(&poison[(j - jm) * 4 + (key >> 5)], 1u << (key & 31));
                uint32_t* x = &x4.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint32_t b = not_finite<T>(x[k]);
                  if (b & 0x8000u) x[k] &= 0xffff0000u;
                  if (b & 0x80000000u) x[k] &= 0x0000ffffu;
                }
                at[i * 64] = x4;
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ok[v]);
        }
        if (!ok) break;
        at_item += 2 * nmax;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctx_empty[c]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int s = warp >> 2, quarter = warp & 3;
    const uint32_t t_s = tmem + s * kPfRows + ((uint32_t)(quarter * 32) << 16);
    static_assert(kPfRows == 128);
    const uint32_t t_o = t_s + C::kTmemO;
    uint32_t phases = 0;                                         // bit 0: s_full, bit 1: o_full
    for (int item = 0;; ++item) {
      volatile int* ctx = ctxs + (item & 1) * kCtxWords;
      if (!all_wait(&ctx_full[item & 1], (item >> 1) & 1) || ctx[kCtxStop]) break;
      // keys that the tile's first row sees, and this row
      const int seen_by_all = ctx[kCtxR0] + ctx[kCtxOff] + s * kPfRows + 1;
      const int reach = min(ctx[kCtxLk], seen_by_all + quarter * 32 + lane), n = ctx[kCtxNk + s];
      float m = -INFINITY, sum = 0.f;                            // reference maximum of the raw scores, sum of terms
      const float scale = p.scale_log2;
      bool fail = false;
      for (int j = 0; j < n; ++j) {
        if (!all_wait(&s_full[s], phases & 1)) {
          fail = true;
          break;
        }
        phases ^= 1;
        tc_fence_after();
        uint32_t x[4][32];
        const bool masked = (j + 1) * kPfRows > seen_by_all;
        const int here = reach - j * kPfRows;
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
      if (fail || (n && !all_wait(&o_full[s], phases >> 1))) break;
      if (n) phases ^= 2;
      tc_fence_after();
      const int e_q0 = ctx[kCtxQ0], e_lq = ctx[kCtxLq], e_h = ctx[kCtxH], e_k0 = ctx[kCtxK0], e_jm = ctx[kCtxJm];
      const int first = ctx[kCtxR0] + s * kPfRows + quarter * 32, row = first + lane;   // within the sequence
      const bool live = row < e_lq;
      const int see = row < ctx[kCtxLead] ? 0 : reach;
      const int64_t at = ((int64_t)ctx[kCtxSplit] * p.rows + e_q0 + row) * p.heads + e_h;   // splits: partial row
      // one of several parts leaves its sums as they are, to be joined; an
      // item of one part says that there is nothing to join
      const bool whole = ctx[kCtxParts] == 1;
      if (p.splits > 1 && live) {
        // a row that sees nothing: -infinity and 0; one whose scores are all
        // minus infinity: a finite maximum and 0
        const float top = sum != 0.f ? m * scale : -FLT_MAX;
        p.part_ml[at] = whole ? make_float2(0.f, kInPlace) : see > 0 ? make_float2(top, sum) : make_float2(-INFINITY, 0.f);
        if (!whole && ctx[kCtxSplit] == 0)
          for (int i = ctx[kCtxParts]; i < p.splits; ++i)
            p.part_ml[at + (int64_t)i * p.rows * p.heads] = make_float2(-INFINITY, 0.f);
      }
      if (n || whole) {
        // The rows go through shared memory, 64 columns at a time, so that a
        // store instruction writes whole lines: with one row per lane it
        // touches 32 of them, and the stores took 2 us per item.
        uint4* stage = reinterpret_cast<uint4*>(smem + C::kOffStage) + warp * 32 * 8;
        const float inv = !whole ? 1.f : see > 0 && n ? 1.f / sum : 0.f;
        const uint32_t* poison = poisons + (item & 1) * 4 * kPfMasked;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4 * kPfMasked; ++i) any |= poison[i];
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
          uint32_t o[2][32];
          tmem_ld32(t_o + c, o[0]);
          tmem_ld32(t_o + c + 32, o[1]);
          tmem_wait_ld();
          float f[64];
          // a row that sees nothing gives zeros, whatever the accumulator holds
#pragma unroll
          for (int i = 0; i < 64; ++i) f[i] = see > 0 && n ? __uint_as_float(o[i / 32][i % 32]) * inv : 0.f;
          if (any && n) {
            for (int i = 0; i < 4 * kPfMasked; ++i) {
              uint32_t bits = poison[i];
              while (bits) {
                const int key = e_jm * kPfRows + i * 32 + __ffs(bits) - 1;
                bits &= bits - 1;
                if (key >= see) continue;
                const T* vr = static_cast<const T*>(p.v) + (int64_t)(e_k0 + key) * p.sv_t + (int64_t)p.by_group(e_h) * p.sv_h + c;
#pragma unroll
                for (int d = 0; d < 64; ++d) {
                  const float v = to_f32(vr[d]);
                  if (!isfinite(v)) f[d] += v;
                }
              }
            }
          }
          if (!whole) {
            if (live) {
              float* po = p.part_o + at * D + c;
#pragma unroll
              for (int i = 0; i < 64; i += 4) *reinterpret_cast<float4*>(po + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            stage[lane * 8 + (i ^ (lane & 7))] =
                make_uint4(pack16<T>(f[8 * i], f[8 * i + 1]), pack16<T>(f[8 * i + 2], f[8 * i + 3]),
                           pack16<T>(f[8 * i + 4], f[8 * i + 5]), pack16<T>(f[8 * i + 6], f[8 * i + 7]));
          __syncwarp();
          const int rows = min(32, e_lq - first);
          T* to = static_cast<T*>(p.out) + ((int64_t)(e_q0 + first) * p.heads + e_h) * D + c;
#pragma unroll 4
          for (int i = lane; i < rows * 8; i += 32)
            *reinterpret_cast<uint4*>(to + (int64_t)(i >> 3) * p.heads * D + (i & 7) * 8) = stage[(i & ~7) + ((i ^ (i >> 3)) & 7)];
          __syncwarp();
        }
      }
      // this warp's reads of the output come before the next item's MMAs
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctx_empty[item & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*(volatile uint32_t*)tmem_slot), "n"(512));
}

// Joins the parts of the items that have several: one thread per four columns.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_prefill_join_kernel(const __grid_constant__ PrefillParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t n = (int64_t)p.rows * p.heads, e = (int64_t)blockIdx.x * 256 + threadIdx.x, at = e / (D / 4);
  if (at >= n) return;
  const int d = (int)(e - at * (D / 4)) * 4;
  float2 ml[kPfSplits];
  ml[0] = p.part_ml[at];
  if (ml[0].y == kInPlace) return;                         // one part, already in place
  float mx = ml[0].x;
#pragma unroll
  for (int i = 1; i < kPfSplits; ++i) {
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
  // nothing seen: zeros; scores of minus infinity alone: 0 / 0
  const float inv = sum != 0.f ? 1.f / sum : mx == -INFINITY ? 0.f : __uint_as_float(0x7fffffffu);
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
  // Parts of items: nearly all of them make no more than a CTA per SM on top
  // of the items; CTAs that find nothing to do cost time.
  const int64_t more = slots * p.heads * (p.splits - 1);
  const int64_t ctas = slots * p.heads + (more < sm_count() ? more : sm_count());
  attn_prefill_kernel<T, D><<<(unsigned)ctas, kPfThreads, C::kSmem, st>>>(maps[0], maps[1], maps[2], p);
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

// Into how many parts an item's keys may be cut (the device chooses, by the
// lengths).  An item (256 rows of one head) takes as long as its keys whatever
// the number of rows, so one long history among short ones, or few items on
// many SMs, shorten when keys are shared out; the price is the second launch,
// 2 to 3 us.  So only where an item may be of 8 key tiles or more, and
//  * some sequences have keys before their queries, and the longest of them
//    may be twice an SM's share of the work (key tiles, and three more per
//    item; one item per 256 rows, half a one more per sequence), or
//  * there are none, and the items leave half of the SMs without work.
// 16 heads of 64, 901 queries behind 6596 keys: 58 us unsplit, 41 in two parts;
// 2 heads of 128, 14 prompts of which one lies behind 5676 keys: 86 and 32 us;
// 14 heads, 10 prompts of which one lies behind 1118 keys: 35 and 39 us.
// Partial results take at most 256 MB.
static int prefill_splits(int B, int64_t rows, int64_t k_rows, int heads, int dim) {
  if (B < 1 || rows < 1) return 1;
  const int64_t sms = sm_count(), before = k_rows - rows;
  const int64_t longest = (before > 0 ? before + (rows + B - 1) / B : k_rows) / kPfRows;
  if (longest < 8) return 1;
  const double items = (double)(rows / (2 * kPfRows) + (B + 1) / 2) * heads;
  const double work = (double)rows * rows / (4.0 * B * kPfRows * kPfRows) * heads + 3.0 * items;   // at least
  if (before > 0 ? (double)longest * sms < 2 * work : 2 * items > sms) return 1;
  const int64_t fit = (256LL << 20) / (rows * heads * (dim * 4 + 8));
  const int64_t n = fit < longest / 4 ? fit : longest / 4;
  return n < 1 ? 1 : n > kPfSplits ? kPfSplits : (int)n;
}

size_t attn_prefill_workspace(int B, int64_t rows, int64_t k_rows, int heads, int dim) {
  const int n = prefill_splits(B, rows, k_rows, heads, dim);
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
  const int splits = workspace ? prefill_splits(B, rows, k_rows, heads, dim) : 1;
  float* po = static_cast<float*>(workspace);
  const PrefillParams p{cu_q, cu_k, B, heads, heads / kv_heads, (int)rows, (int)k_rows, scale_log2, out, v, s[4], s[5],
                        Divisor(heads), Divisor(heads / kv_heads), sm_count(),
                        splits, po, reinterpret_cast<float2*>(po + (size_t)splits * rows * heads * dim)};
  // at most one item more than whole ones per sequence (and for the rows behind the last)
  int64_t slots = rows / (2 * kPfRows) + B + 1;
  if (slots > rows) slots = rows;
  if (slots * heads * splits > 0x3FFFFFFF || rows * heads * (dim / 4) / 256 >= 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (dtype == PARO_BF16)
    return dim == 128 ? launch_prefill<__nv_bfloat16, 128>(maps, p, slots, st)
                      : launch_prefill<__nv_bfloat16, 64>(maps, p, slots, st);
  return dim == 128 ? launch_prefill<__half, 128>(maps, p, slots, st) : launch_prefill<__half, 64>(maps, p, slots, st);
}

}  // namespace paro
