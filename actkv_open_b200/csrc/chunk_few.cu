// Chunk attention of sessions with few new tokens (a single token, a drafted run: at most 16 query rows,
// token x head of the GQA group, per KV head; 8 over the 8-bit cache) over the paged cache: the formulas of
// chunk_umma.cu.
//
// Such a call reads each key and value once for a handful of products, so memory bounds it: 4 (2 over
// the 8-bit cache) bytes per key-value pair of values against 4 operations per query row.  What matters is
// bytes in flight and no hand-overs between them and the sums.  So there are none: a warp copies 16 tokens
// of keys and values (cp.async, a private ring of three steps), reads them as operands of the warp-wide
// m16n8k16 product straight from there, keeps its own running maximum, sum and output in registers, and the
// results leave from registers.  The 128-row tensor-core tile of chunk_umma.cu would be at most an eighth
// full here, and over the 8-bit cache would need the widened values in shared memory; here they are
// widened in registers on their way into the product.
//
// Operands.  The first product sums over dims in any order, as long as both operands agree, so a lane's four
// dims of a k-step are consecutive ones of a 16-byte piece of its token's row.  The outputs' dims come in any
// order, so lane group n takes dims (D / 8) n .. of the values, again consecutive bytes of a row; the
// pairs of tokens that an operand register holds are put together by byte permutes.
//   16-bit rows: S = Q K^T and O = P V, 16 query rows as the products' rows; p goes from the layout of S to
//     that of the second product without a move.  8 warps of 244 registers.
//   8-bit rows: S^T = K Q^T and O^T = V^T P^T, tokens and dims as the products' rows and 8 query rows as
//     their columns: half the products, and O^T takes half the registers, so that 16 warps of 127 hide
//     the widening's latencies (the batch below: 8 warps 344 us, 16 warps 304 us, the other way round 379 us, all before
//     the widening was made shorter); p^T is an
//     8 x 8 transpose per 8 tokens.
//
// Work is shared out as in chunk_umma.cu, in equal shares per CTA.  A unit is a session and a group of 8 (4, 2, 1:
// what divides them) KV heads, a warp per head: a token's row is read whole by one CTA at one time.  With a
// head per CTA the 8-bit rows' scale bytes, 4 per head and row, were fetched from memory once per head, 64 bytes
// each time: 1.7 times the bytes of the rows, against 1.03 times now.  Further warps of a head take its tokens in
// turn and join through shared memory.
//
// Measured: 32 single-token sessions of 4096 to 32768 tokens, 32 query heads over 8 KV heads of 128: 16-bit
// rows (2.4 GB) 380 us, 6.3 TB/s, 0.97 of the measured copy rate, memory bound; 8-bit rows (1.25 GB) 292 to 300 us
// (the board's power limit), 4.2 TB/s, 0.64 of it, bound by issue and the logic pipe (five operations per pair of values to
// widen them to bf16 and one to find e4m3's NaN, of about 730 instructions per step; conversion to fp16 by one
// instruction per pair instead, with the ranges kept by powers of two, measured no faster).
#include <type_traits>

#include "chunk_common.cuh"

namespace actkv {
namespace chunk {
namespace few {

constexpr int kRoundCost = 6;               // a unit's fixed cost in rounds of its warps
constexpr int kMinRounds = 6;               // a CTA's share is at least so many: fewer partial results to join
constexpr int kStep = 16;                   // tokens per step
constexpr int kJoinRow = kMaxD + 8;         // a warp's O, m and l in shared memory: 16 of these floats

template <int D, bool QUANT>
struct Ring {
  static constexpr int kWarps = QUANT ? 16 : 8, kThreads = kWarps * 32;
  static constexpr int kEs = QUANT ? 1 : 2;
  static constexpr int kChunks = D * kEs / 16;              // 16-byte pieces of a row
  static constexpr uint32_t kPlane = kStep * D * kEs;       // keys, then values
  static constexpr uint32_t kStage = 2 * kPlane + (QUANT ? 128 : 0);     // and their scale words
  static constexpr int kStages = QUANT ? 3 : (D == 128 ? 3 : 6);
  static constexpr uint32_t kBytes = kWarps * kStages * kStage;
  static constexpr uint32_t kJoinBytes = kWarps * kFewRows * kJoinRow * 4;
  static constexpr uint32_t kSmemBytes = (kBytes > kJoinBytes ? kBytes : kJoinBytes) + 512;
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
};

// Where piece c of token row r is kept: the eight lanes that read together (two rows of keys, four pairs
// of rows of values) find their pieces in different banks.
template <int CH>
__device__ __forceinline__ int key_piece(int r, int c) { return CH >= 8 ? c ^ ((r & 1) << 2) : c; }
template <int CH>
__device__ __forceinline__ int value_piece(int r, int c) {
  return CH == 16 ? c ^ (((r >> 1) & 1) | (r & 4)) : (CH == 8 ? c ^ (r & 6) : c ^ ((r >> 1) & 2));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Lane (r, c) has elements (r, 2 c) and (r, 2 c + 1) of an 8 x 8 matrix; of its transpose after.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Two e4m3 bytes, at the bottom of x's halves, times f.  (Two of four operations on the logic pipe: 260 us for 32
// single tokens of 18432; with the bytes' order and mask of widen16 269, with a shift, two masks and an or 278, all
// before NaN bytes were looked for.)
template <bool BF16>
__device__ __forceinline__ uint32_t widen2(uint32_t x, uint32_t f) {
  return mul16x2<BF16>(under_exponent<BF16>(x * 256u, x & 0x007f007fu), f);
}
// ... for any scale bytes of the two halves.
template <bool BF16>
__device__ __forceinline__ uint32_t widen2_any(uint32_t x, uint32_t b_lo, uint32_t b_hi) {
  uint32_t lo[3], hi[3];
  any_factors<BF16>(b_lo, lo);
  any_factors<BF16>(b_hi, hi);
  return put_nan(mul_rest<BF16>(widen2<BF16>(x, __byte_perm(lo[0], hi[0], 0x5410)), __byte_perm(lo[1], hi[1], 0x5410),
                                __byte_perm(lo[2], hi[2], 0x5410)), x & 0x007f007fu);
}
struct Sched {
  Share share;
  int64_t scan[32], sums[2];
  int bad_v;                 // values that are not finite went in as 0: 1 among those some row does not see, 2 anywhere
};
static_assert(sizeof(Sched) <= 512, "the schedule's place in shared memory");

template <int D, bool BF16, bool QUANT>
__global__ void __launch_bounds__(Ring<D, QUANT>::kThreads, 1) chunk_few_kernel(const __grid_constant__ ChunkArgs a, bool vec_out) {
  using Rg = Ring<D, QUANT>;
  constexpr int kWarps = Rg::kWarps, kThreads = Rg::kThreads;
  constexpr int CH = Rg::kChunks, kRowsPerCopy = 32 / CH, kCopies = kStep / kRowsPerCopy;
  constexpr int kKSteps = D / 16, kTiles = D / 8;           // k-steps of S, dims of O per lane (group)
  constexpr int kOut = QUANT ? kTiles / 2 : kTiles;         // products of O
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r8 = lane >> 2, c4 = lane & 3;
  constexpr uint32_t kSchedOff = Rg::kSmemBytes - 512;
  Sched& sched = *reinterpret_cast<Sched*>(smem + kSchedOff);
  const int cta = blockIdx.x, n_cta = gridDim.x;
  const uint32_t ring = smem_u32(smem) + warp * Rg::kStages * Rg::kStage;
  const unsigned full = 0xffffffffu;
  const float ninf = -__int_as_float(0x7f800000);
  const Parts ps = few_parts(a.workspace, n_cta);
  pdl_trigger();
  if (threadIdx.x == 0) {
    sched.share = Share{0, 0, a.R};
    sched.bad_v = 0;
    ps.desc[cta].valid = 0;
  }
  __syncthreads();
  const int HG = a.Hkv % 8 == 0 ? 8 : (a.Hkv % 4 == 0 ? 4 : (a.Hkv % 2 == 0 ? 2 : 1));   // heads per unit
  const int wph = kWarps / HG, round = kStep * wph;         // warps per head, tokens of a round of theirs
  const int my_head = warp % HG, my_part = warp / HG;
  const int few_rows = few_rows_now<kThreads>(a, sched.sums);
  if (few_rows == 0) return;
  share_out<kThreads>(a.R, [&](int r) -> int64_t {
    const int A = new_tokens(a, r), S = a.seq_used[r];
    if (A == 0 || A * a.G > few_rows) return 0;
    flag_long(a, S);
    return int64_t(a.Hkv / HG) * (kRoundCost + (held_tokens(a, S) + round - 1) / round);
  }, sched.share, sched.scan, cta, n_cta, kMinRounds);
  const int64_t total = sched.share.total;
  const int n_used = used_ctas(total, n_cta, kMinRounds);
  const int64_t lo = total * cta / n_used, hi = total * (cta + 1) / n_used;
  if (cta >= n_used || lo >= hi) return;
  int r = sched.share.r0;
  int64_t at = sched.share.pre;              // start of (session r, head group hg) in the schedule
  int hg = 0;
  bool seek = true;
  const float c2 = a.scale * kLog2e;
  const char* kv = static_cast<const char*>(a.kv);
  const int64_t es = QUANT ? 1 : 2, stride_s = a.kv_stride_s * es, stride_b = a.kv_stride_b * es;
  const int64_t to_values = a.kv_stride_kv * es;
  const int shift = (a.BS & (a.BS - 1)) == 0 ? __ffs(a.BS) - 1 : -1;
  auto block_of = [&](int tok) { return shift >= 0 ? tok >> shift : tok / a.BS; };

  for (; r < a.R && at < hi; ++r, hg = 0) {
    const int a0 = a.q_off[r], A = new_tokens(a, r), S = a.seq_used[r];
    if (A == 0 || A * a.G > few_rows) continue;
    const int rows = A * a.G;
    const int nt = (held_tokens(a, S) + round - 1) / round;
    const int64_t weight = kRoundCost + nt;
    if (seek) {                               // the group that holds lo
      hg = int((lo - at) / weight);
      at += hg * weight;
      seek = false;
    }
    const int32_t* table = a.block_table + r * a.bt_stride_r;
    for (; hg < a.Hkv / HG && at < hi; ++hg, at += weight) {
      const int64_t first = at + kRoundCost;
      const int t0 = int(lo > first ? lo - first : 0), t1 = nt == 0 ? 0 : int(min(int64_t(nt), hi - first));
      if (nt == 0 ? at < lo : t0 >= t1) continue;
      const int h = hg * HG + my_head;
      const int begin = t0 * round, end = min(t1 * round, held_tokens(a, S));
      const int start = begin + my_part * kStep;              // this warp's steps: start, start + round, ...
      const int mine = start < end ? (end - start + round - 1) / round : 0;
      // the lane's two query rows, and the last tokens they see
      const int row0 = QUANT ? 2 * c4 : r8, row1 = QUANT ? row0 + 1 : r8 + 8;
      const int lim0 = S - A + row0 / a.G, lim1 = S - A + row1 / a.G;
      const bool wide = rows > 8;
      // ---- queries, dims as the keys come: 16-bit rows as the first operand, rows r8 and r8 + 8 for each k-step;
      // 8-bit rows as the second, row r8
      constexpr int kQ = QUANT ? 1 : 2;
      uint32_t q[kKSteps][2 * kQ];
      {
        const uint16_t* qp = static_cast<const uint16_t*>(a.q);
#pragma unroll
        for (int hf = 0; hf < kQ; ++hf) {
          const int row = r8 + hf * 8, jq = row / a.G;
          const uint16_t* p = qp + (int64_t(a0) + jq) * a.q_stride_t + int64_t(h * a.G + row - jq * a.G) * a.q_stride_h;
#pragma unroll
          for (int k = 0; k < kKSteps; ++k) {
            // the dims of k-step k: 4 consecutive ones of piece c4 + 4 i
            const int per = QUANT ? 4 : 2;    // k-steps per piece
            const int d = (c4 + 4 * (k / per)) * (per * 4) + (k % per) * 4;
            const uint2 u = row < rows ? *reinterpret_cast<const uint2*>(p + d) : make_uint2(0u, 0u);
            q[k][hf] = u.x;
            q[k][kQ + hf] = u.y;
          }
        }
      }
      float o[kOut][4];
#pragma unroll
      for (int j = 0; j < kOut; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
      float m0 = ninf, m1 = ninf, l0 = 0.0f, l1 = 0.0f;

      // ---- copies of step i of this warp: lane l (and l - 16) looks up token l's block a step ahead (and looks at
      // what it got only then: 32 single tokens over 18432 in 8 bits 314 us where the id was used at once, 271 here)
      auto look_up = [&](int i) -> int {
        const int tok = start + i * round + (lane & 15);
        if (i >= mine || tok >= end) return -1;
        const int lb = block_of(tok);
        return lb < a.MB ? table[lb] : -1;
      };
      int phys = look_up(0);
      const char* head = kv + (QUANT ? int64_t(h) * D : int64_t(h) * a.kv_stride_h * 2);
      const int at_word = a.Hkv * D + (D == 128 ? h * 4 : (h * 2) & ~3);
      bool gaps = false;                      // this lane met a block outside the cache: from there on every step looks
      auto issue = [&](int i, int slot) {
        if (i < mine) {
          const int tok = start + i * round + (lane & 15);
          const bool none = uint32_t(phys) >= uint32_t(a.NB); // past the end, or an id outside the cache: zeros
          if (none && tok < end) {
            flag(a.status, ACTKV_DEV_BAD_INDEX);
            gaps = true;
          }
          const int in_block = shift >= 0 ? tok & (a.BS - 1) : tok % a.BS;
          const int64_t off = none ? -1 : int64_t(phys) * stride_b + int64_t(in_block) * stride_s;
          const uint32_t dst = ring + slot * Rg::kStage;
#pragma unroll
          for (int e = 0; e < kCopies; ++e) {
            const int row = e * kRowsPerCopy + lane / CH, c = lane % CH;
            const int64_t from = __shfl_sync(full, off, row);
            const char* p = (from < 0 ? kv : head + from) + c * 16;
            copy16(dst + row * (CH * 16) + key_piece<CH>(row, c) * 16, p, from >= 0);
            copy16(dst + Rg::kPlane + row * (CH * 16) + value_piece<CH>(row, c) * 16, p + to_values, from >= 0);
          }
          if constexpr (QUANT)                // words: lanes 0-15 the keys', 16-31 the values'
            copy4(dst + 2 * Rg::kPlane + lane * 4, kv + (off < 0 ? 0 : off + at_word) + (lane >> 4) * to_values, off >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        phys = look_up(i + 1);
      };

      // the rows' references go up to the maxima given (the same in all lanes of a row)
      auto raise = [&](float top0, float top1) {
        const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
        const float e0 = m0 == n0 ? 1.0f : ex2(m0 - n0), e1 = m1 == n1 ? 1.0f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= e0;
        l1 *= e1;
#pragma unroll
        for (int j = 0; j < kOut; ++j) {
          o[j][0] *= e0;
          o[j][1] *= QUANT ? e1 : e0;
          o[j][2] *= QUANT ? e0 : e1;
          o[j][3] *= e1;
        }
      };
      // 8-bit rows: e4m3 NaN among the keys and among the values of the steps whose every token every row sees
      [[maybe_unused]] uint32_t odd_k = 0, odd_v = 0;
      auto step = [&](int i, int slot, auto edge_) {
        constexpr bool EDGE = decltype(edge_)::value;        // hidden tokens, or scale bytes out of the ordinary
        const int t = start + i * round;
        const uint32_t kb = ring + slot * Rg::kStage, vb = kb + Rg::kPlane;
        [[maybe_unused]] const uint32_t sb = kb + 2 * Rg::kPlane;
        [[maybe_unused]] const int sh = QUANT && D == 64 && (h & 1) ? 16 : 0; // the head's bytes within the word
        bool found = false;
        // the step's tokens that are there: neither past the end nor in a block outside the cache
        [[maybe_unused]] uint32_t there = 0xffffu;
        if constexpr (EDGE) {
          bool here = lane < kStep && t + lane < end;
          if (__any_sync(full, gaps) && here) {
            const int lb = block_of(t + lane);
            here = lb < a.MB && uint32_t(table[lb]) < uint32_t(a.NB);
          }
          there = __ballot_sync(full, here);
        }
        // the lane's tokens of the values, and those that some row does not see: what is not finite goes in as 0
        const int row[4] = {2 * c4, 2 * c4 + 1, 2 * c4 + 8, 2 * c4 + 9};
        [[maybe_unused]] uint32_t hide[2] = {0u, 0u};
        if constexpr (EDGE) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
            hide[n] = (t + row[2 * n] > S - A ? 0xffffu : 0u) | (t + row[2 * n + 1] > S - A ? 0xffff0000u : 0u);
        }
        if constexpr (QUANT) {
          // ---- S^T = K Q^T, tokens as the product's rows: s[0..1] token t + r8, s[2..3] token t + r8 + 8, query
          // rows 2 c4 and 2 c4 + 1.  Eight query rows fill the product's columns, O^T takes half the registers
          // that O would, and twice the warps fit.
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const uint32_t word0 = lds4(sb + r8 * 4) >> sh, word1 = lds4(sb + 32 + r8 * 4) >> sh;
#pragma unroll
          for (int p = 0; p < CH / 4; ++p) {
            const uint4 u = lds16(kb + r8 * (CH * 16) + key_piece<CH>(r8, c4 + 4 * p) * 16);
            const uint4 v = lds16(kb + (r8 + 8) * (CH * 16) + key_piece<CH>(r8 + 8, c4 + 4 * p) * 16);
            const uint32_t w0[4] = {u.x, u.y, u.z, u.w}, w1[4] = {v.x, v.y, v.z, v.w};
            if constexpr (!EDGE) {
#pragma unroll
              for (int k = 0; k < 4; ++k) odd_k = nan_bytes(nan_bytes(odd_k, w0[k]), w1[k]);
            }
            const int g8 = (c4 + 4 * p) / 2 * 8;             // 16 dims: four k-steps of one scale group
            const uint32_t b0 = word0 >> g8 & 255u, b1 = word1 >> g8 & 255u;
            const uint32_t f0 = plain_factor<BF16>(b0), f1 = plain_factor<BF16>(b1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t x[4] = {__byte_perm(w0[k], 0u, 0x4140), __byte_perm(w1[k], 0u, 0x4140),
                                     __byte_perm(w0[k], 0u, 0x4342), __byte_perm(w1[k], 0u, 0x4342)};
              uint32_t m[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                m[e] = EDGE ? widen2_any<BF16>(x[e], e & 1 ? b1 : b0, e & 1 ? b1 : b0)
                            : widen2<BF16>(x[e], e & 1 ? f1 : f0);
              mma16816<BF16>(s, m, q[p * 4 + k][0], q[p * 4 + k][1]);
            }
          }
          if constexpr (EDGE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = r8 + (e >> 1) * 8;
              s[e] = t + at <= (e & 1 ? lim1 : lim0) && (there >> at & 1u) ? s[e] : ninf;
            }
          }
          float top0 = fmaxf(s[0], s[2]) * c2, top1 = fmaxf(s[1], s[3]) * c2;
          if (__any_sync(full, top0 > m0 + kSlack || top1 > m1 + kSlack)) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
              top0 = fmaxf(top0, __shfl_xor_sync(full, top0, x));
              top1 = fmaxf(top1, __shfl_xor_sync(full, top1, x));
            }
            raise(top0, top1);
          }
          const float o0 = m0 == ninf ? 0.0f : m0, o1 = m1 == ninf ? 0.0f : m1;
          const float x = ex2(fmaf(s[0], c2, -o0)), y = ex2(fmaf(s[1], c2, -o1)), z = ex2(fmaf(s[2], c2, -o0)),
                      w = ex2(fmaf(s[3], c2, -o1));
          l0 += x + z;
          l1 += y + w;
          // p^T as the second operand: row r8, tokens 2 c4, 2 c4 + 1 and those + 8
          const uint32_t p0 = transpose8x8(pack_p<BF16>(x, y)), p1 = transpose8x8(pack_p<BF16>(z, w));
          // ---- O^T += V^T p^T: values of tokens 2 c4, 2 c4 + 1 and those + 8, dims kTiles r8 ..
          uint32_t vw[4][kTiles / 4], b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t base = vb + row[e] * (CH * 16);
            if constexpr (D == 128) {
              const uint4 u = lds16(base + value_piece<CH>(row[e], r8) * 16);
              vw[e][0] = u.x;
              vw[e][1] = u.y;
              vw[e][kTiles / 4 - 2] = u.z;
              vw[e][kTiles / 4 - 1] = u.w;
            } else {
              const uint2 u = lds8(base + value_piece<CH>(row[e], r8 >> 1) * 16 + (r8 & 1) * 8);
              vw[e][0] = u.x;
              vw[e][1] = u.y;
            }
            if constexpr (!EDGE) {
#pragma unroll
              for (int k = 0; k < kTiles / 4; ++k) odd_v = nan_bytes(odd_v, vw[e][k]);
            }
            b[e] = (lds4(sb + 64 + row[e] * 4) >> (sh + kTiles * r8 / 32 * 8)) & 255u;
          }
          const uint32_t f0 = __byte_perm(plain_factor<BF16>(b[0]), plain_factor<BF16>(b[1]), 0x5410);
          const uint32_t f1 = __byte_perm(plain_factor<BF16>(b[2]), plain_factor<BF16>(b[3]), 0x5410);
#pragma unroll
          for (int k = 0; k < kTiles / 4; ++k) {
            // dims 4 k .. 4 k + 3 of two tokens each, a dim's two bytes next to one another
            const uint32_t pair[2][2] = {{__byte_perm(vw[0][k], vw[1][k], 0x5140), __byte_perm(vw[2][k], vw[3][k], 0x5140)},
                                         {__byte_perm(vw[0][k], vw[1][k], 0x7362), __byte_perm(vw[2][k], vw[3][k], 0x7362)}};
#pragma unroll
            for (int e = 0; e < 2; ++e) {     // dims 4 k + 2 e and + 1: rows r8 and r8 + 8 of the product
              uint32_t m[4];
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                const uint32_t x = __byte_perm(pair[e][n >> 1], 0u, n & 1 ? 0x4342 : 0x4140);
                if constexpr (EDGE) m[n] = drop_bad<BF16>(widen2_any<BF16>(x, b[n >> 1 << 1], b[(n >> 1 << 1) + 1]), hide[n >> 1], found);
                else m[n] = widen2<BF16>(x, n >> 1 ? f1 : f0);
              }
              mma16816<BF16>(o[k * 2 + e], m, p0, p1);
            }
          }
        } else {
          float s[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int tok = n * 8 + r8;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
            for (int p = 0; p < (CH + 3) / 4; ++p) {
              const uint4 u = lds16(kb + tok * (CH * 16) + key_piece<CH>(tok, c4 + 4 * p) * 16);
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
              mma16816<BF16>(s[n], q[p * 2], w[0], w[1]);           // 8 dims: two k-steps
              mma16816<BF16>(s[n], q[p * 2 + 1], w[2], w[3]);
            }
          }
          // s[n][0..1]: row r8, tokens t + 8 n + 2 c4, + 1; s[n][2..3]: row r8 + 8
          float top0 = ninf, top1 = ninf;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if constexpr (EDGE) {
                const int at = 8 * n + 2 * c4 + e;
                const bool is = there >> at & 1u;
                s[n][e] = t + at <= lim0 && is ? s[n][e] : ninf;
                s[n][2 + e] = t + at <= lim1 && is ? s[n][2 + e] : ninf;
              }
              top0 = fmaxf(top0, s[n][e]);
              top1 = fmaxf(top1, s[n][2 + e]);
            }
          top0 *= c2;
          top1 *= c2;
          if (__any_sync(full, top0 > m0 + kSlack || top1 > m1 + kSlack)) {
            top0 = fmaxf(top0, __shfl_xor_sync(full, top0, 1));
            top0 = fmaxf(top0, __shfl_xor_sync(full, top0, 2));
            top1 = fmaxf(top1, __shfl_xor_sync(full, top1, 1));
            top1 = fmaxf(top1, __shfl_xor_sync(full, top1, 2));
            raise(top0, top1);
          }
          const float b0 = m0 == ninf ? 0.0f : m0, b1 = m1 == ninf ? 0.0f : m1;
          uint32_t p[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float x = ex2(fmaf(s[n][0], c2, -b0)), y = ex2(fmaf(s[n][1], c2, -b0));
            l0 += x + y;
            p[2 * n] = pack_p<BF16>(x, y);
            if (wide) {
              const float z = ex2(fmaf(s[n][2], c2, -b1)), w = ex2(fmaf(s[n][3], c2, -b1));
              l1 += z + w;
              p[2 * n + 1] = pack_p<BF16>(z, w);
            }
          }
          // ---- values: tokens 2 c4, 2 c4 + 1 and those + 8, dims kTiles r8 ..
#pragma unroll
            for (int c = 0; c < kTiles / 8; ++c) {
              uint32_t w[4][4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint4 u = lds16(vb + row[e] * (CH * 16) + value_piece<CH>(row[e], r8 * (kTiles / 8) + c) * 16);
                w[e][0] = u.x;
                w[e][1] = u.y;
                w[e][2] = u.z;
                w[e][3] = u.w;
              }
#pragma unroll
              for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  uint32_t x0 = __byte_perm(w[0][k], w[1][k], e ? 0x7632 : 0x5410);
                  uint32_t x1 = __byte_perm(w[2][k], w[3][k], e ? 0x7632 : 0x5410);
                  if constexpr (EDGE) {
                    x0 = drop_bad<BF16>(x0, hide[0], found);
                    x1 = drop_bad<BF16>(x1, hide[1], found);
                  }
                  mma16816<BF16>(o[c * 8 + k * 2 + e], p, x0, x1);
                }
            }
        }
        if (EDGE && found) atomicOr(&sched.bad_v, 1);
      };

      // ---- the steps
      constexpr int kAhead = Rg::kStages - 1;
#pragma unroll 1
      for (int i = 0; i < kAhead; ++i) issue(i, i);
      int slot = 0, fill = kAhead;
#pragma unroll 1
      for (int i = 0; i < mine; ++i) {
        issue(i + kAhead, fill);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
        __syncwarp();
        const int t = start + i * round;
        bool edge = t + kStep - 1 > S - A || t + kStep > end;
        if constexpr (QUANT) {
          const uint32_t word = lds4(ring + slot * Rg::kStage + 2 * Rg::kPlane + lane * 4);
          edge = edge || !__all_sync(full, plain_scales<BF16>(word) && !gaps);
        } else {
          edge = edge || __any_sync(full, gaps);
        }
        if (edge) step(i, slot, std::true_type());
        else step(i, slot, std::false_type());
        __syncwarp();                         // every lane has read the slot that the next copies fill
        slot = slot + 1 == Rg::kStages ? 0 : slot + 1;
        fill = fill + 1 == Rg::kStages ? 0 : fill + 1;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if constexpr (QUANT) {                  // such a key makes every row NaN, such a value a dim of every row
        if (__any_sync(full, any_nan_byte(odd_k))) l0 = l1 = __int_as_float(0x7fffffff);
        if (any_nan_byte(odd_v)) atomicOr(&sched.bad_v, 2);
        __syncwarp();
      }
      // ---- results: l of a row over the lanes that share it
#pragma unroll
      for (int x = QUANT ? 4 : 1; x < (QUANT ? 32 : 4); x *= 2) {
        l0 += __shfl_xor_sync(full, l0, x);
        l1 += __shfl_xor_sync(full, l1, x);
      }
      const bool whole = t0 == 0 && t1 == nt;
      const int ps_slot = t0 > 0 ? 0 : 1;
      if (wph > 1) {                          // the warps of a head meet through shared memory, the first goes on
        __syncthreads();                      // the rings are free
        float* jo = reinterpret_cast<float*>(smem) + warp * (kFewRows * kJoinRow);
        if (my_part > 0) {
#pragma unroll
          for (int j = 0; j < kOut; ++j)
            *reinterpret_cast<float4*>(jo + (j * 32 + lane) * 4) = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
          *reinterpret_cast<float4*>(jo + (kOut * 32 + lane) * 4) = make_float4(m0, l0, m1, l1);
        }
        __syncthreads();
        if (my_part == 0)
#pragma unroll 1
          for (int w = warp + HG; w < kWarps; w += HG) {
            const float4* po = reinterpret_cast<const float4*>(smem) + w * (kFewRows * kJoinRow / 4);
            const float4 y = po[kOut * 32 + lane];
            const float M0 = fmaxf(m0, y.x), M1 = fmaxf(m1, y.z);
            // an empty side (sum 0) counts for nothing; a NaN sum stays
            const float p0 = l0 == 0.0f ? 0.0f : (m0 == M0 ? 1.0f : ex2(m0 - M0)), q0 = y.y == 0.0f ? 0.0f : (y.x == M0 ? 1.0f : ex2(y.x - M0));
            const float p1 = l1 == 0.0f ? 0.0f : (m1 == M1 ? 1.0f : ex2(m1 - M1)), q1 = y.w == 0.0f ? 0.0f : (y.z == M1 ? 1.0f : ex2(y.z - M1));
            m0 = M0;
            m1 = M1;
            l0 = fmaf(l0, p0, y.y * q0);
            l1 = fmaf(l1, p1, y.w * q1);
#pragma unroll
            for (int j = 0; j < kOut; ++j) {
              const float4 x = po[j * 32 + lane];
              o[j][0] = fmaf(o[j][0], p0, x.x * q0);
              o[j][1] = QUANT ? fmaf(o[j][1], p1, x.y * q1) : fmaf(o[j][1], p0, x.y * q0);
              o[j][2] = QUANT ? fmaf(o[j][2], p0, x.z * q0) : fmaf(o[j][2], p1, x.z * q1);
              o[j][3] = fmaf(o[j][3], p1, x.w * q1);
            }
          }
      }
      // The lane's dims come in runs of kTiles: over the 8-bit cache one run, kTiles r8 on, of both its rows; else
      // two, of columns 2 c4 and 2 c4 + 1 of the products.
      if (my_part == 0) {
        const int fix = *reinterpret_cast<volatile int*>(&sched.bad_v);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = hf ? row1 : row0;
          if (row >= rows) continue;
          const float L = hf ? l1 : l0, M = hf ? m1 : m0, inv = over<BF16>(L);
          const int jq = row / a.G, hq = h * a.G + row - jq * a.G, hr = my_head * rows + row;
          const int64_t qt = int64_t(a0) + jq;
          uint16_t* dst = static_cast<uint16_t*>(a.out) + qt * a.out_stride_t + int64_t(hq) * a.out_stride_h;
          float* part = ps.out(cta, ps_slot) + int64_t(hr) * D;
#pragma unroll
          for (int cc = 0; cc < (QUANT ? 1 : 2); ++cc) {
            const int d0 = kTiles * (QUANT ? r8 : 2 * c4 + cc);
            auto val = [&](int j) { return QUANT ? o[j >> 1][(j & 1) * 2 + hf] : o[QUANT ? 0 : j][2 * hf + cc]; };
            if (whole) {
#pragma unroll
              for (int j = 0; j < kTiles; j += 8) {
                uint32_t u[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  u[k] = pack2<BF16>(val(j + 2 * k) * inv, val(j + 2 * k + 1) * inv);
                if (vec_out) {
                  *reinterpret_cast<uint4*>(dst + d0 + j) = make_uint4(u[0], u[1], u[2], u[3]);
                } else {
#pragma unroll
                  for (int k = 0; k < 8; ++k) dst[d0 + j + k] = uint16_t(u[k >> 1] >> (k & 1) * 16);
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < kTiles; j += 4)
                *reinterpret_cast<float4*>(part + d0 + j) = make_float4(val(j), val(j + 1), val(j + 2), val(j + 3));
            }
            if (fix) {                        // values that are not finite and that this row does see
#pragma unroll 1
              for (int t = (fix & 2) ? begin : max(S - A + 1, begin); t <= min(S - A + jq, end - 1); ++t) {
                const int lb = block_of(t), ph = lb < a.MB ? table[lb] : -1;
                if (ph < 0 || ph >= a.NB) continue;
                const char* p = kv + to_values + int64_t(ph) * stride_b + int64_t(t - lb * a.BS) * stride_s;
#pragma unroll 1
                for (int d = d0; d < d0 + kTiles; ++d) {
                  float f;
                  if constexpr (QUANT) {
                    f = quant_value<BF16>(reinterpret_cast<const uint8_t*>(p), a.Hkv, D, h * D + d);
                  } else {
                    const uint16_t u = reinterpret_cast<const uint16_t*>(p)[int64_t(h) * a.kv_stride_h + d];
                    f = BF16 ? __uint_as_float(uint32_t(u) << 16) : __half2float(__ushort_as_half(u));
                  }
                  if (isfinite(f)) continue;
                  if (whole) {
                    const float y = BF16 ? __uint_as_float(uint32_t(dst[d]) << 16) : __half2float(__ushort_as_half(dst[d]));
                    dst[d] = uint16_t(pack2<BF16>(y + f, 0.0f));
                  } else {
                    part[d] += f;
                  }
                }
              }
            }
          }
          if ((QUANT ? r8 : c4) == 0) {
            if (whole)
              a.lse[qt * a.lse_stride_t + hq] = L == 0.0f ? ninf : (M == ninf ? L : (M + log2f(L)) * 0.69314718055994531f);
            else
              *reinterpret_cast<float2*>(ps.ml(cta, ps_slot, D) + 2 * hr) = make_float2(M, L);
          }
        }
      }
      if (!whole && t0 == 0 && threadIdx.x == 0) {
        Desc ds = {};
        ds.valid = 1;
        ds.r = r;
        ds.h = hg * HG;
        ds.heads = HG;
        ds.n_used = n_used;
        ds.ntok = A;
        ds.S = S;
        ds.A = A;
        ds.a0 = a0;
        ds.end = first + nt;
        ds.total = total;
        ps.desc[cta] = ds;
      }
      if (wph > 1) __syncthreads();           // the rings are written again
    }
  }
}

}  // namespace few
}  // namespace chunk

namespace {

template <int D, bool BF16, bool QUANT>
cudaError_t launch_few_t(const ChunkArgs& a, int grid, cudaStream_t st) {
  auto k = chunk::few::chunk_few_kernel<D, BF16, QUANT>;
  constexpr int bytes = int(chunk::few::Ring<D, QUANT>::kSmemBytes);
  static SmemLimit limit;
  const cudaError_t e = limit.set(reinterpret_cast<const void*>(k), bytes);
  if (e != cudaSuccess) return e;
  const bool vec_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride_t % 8 == 0 && a.out_stride_h % 8 == 0;
  k<<<grid, chunk::few::Ring<D, QUANT>::kThreads, bytes, st>>>(a, vec_out);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk_few(const ChunkArgs& a, int dtype, int grid, cudaStream_t st) {
  const bool bf = dtype == ACTKV_BF16;
  if (a.quant) {
    if (a.D == 128) return bf ? launch_few_t<128, true, true>(a, grid, st) : launch_few_t<128, false, true>(a, grid, st);
    return bf ? launch_few_t<64, true, true>(a, grid, st) : launch_few_t<64, false, true>(a, grid, st);
  }
  if (a.D == 128) return bf ? launch_few_t<128, true, false>(a, grid, st) : launch_few_t<128, false, false>(a, grid, st);
  return bf ? launch_few_t<64, true, false>(a, grid, st) : launch_few_t<64, false, false>(a, grid, st);
}

}  // namespace actkv
