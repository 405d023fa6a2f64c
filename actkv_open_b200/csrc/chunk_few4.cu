// Chunk attention of sessions with few new tokens over the 4-bit cache (quant_row.cuh): the formulas of
// chunk_umma.cu, the plan of chunk_few.cu (a warp per KV head and run of tokens, a private ring of cp.async
// copies, running sums in registers, no hand-overs), with products laid out so that no value is scaled by itself.
//
// e2m1 values are exact in fp16 and one instruction widens two of them, so both products take them as they are, in fp16
// whatever the queries' type, and the scales enter elsewhere:
//   S^T = K Q^T    the 16 dims of a product are of one group of 32, so a group's two products give a 32-bit partial sum
//                  per (token, row), which is multiplied by the token's scale as it is added: 4 multiply-adds per
//                  512 values.
//   O^T = V^T p^T  the 16 dims that a product gives are of one group, so p is multiplied by the token's scale of
//                  that group, in fp16, once per group: 2 multiplications per 512 values.  The scale is taken
//                  relative to a reference of the warp and group, 2^(b - E), with b in E - 7 .. E.
// Queries of 16-bit types go in as fp16: bf16 rows times the power of two that brings their largest value to 2^14 .. 2^15, so
// that what is 2^-28 of it is still exact; rows with a group whose largest value is 2^-12 of that (its keys may be as much larger)
// have a power of two per group, which the steps of the uncommon kind undo.  p is rounded to fp16's 11 bits, times 2^7 and the scale.
//
// Scales of any size.  A value's size says nothing of its weight, and fp16 loses what is 2^-32 of the largest p.  So the
// tokens of the products, those whose bytes are within the window of all groups' E, are a class of their own: m is the
// maximum of THEIR logits, so one of them has p = 1 at 2^(E - 10) at least, and what another loses is below 2^-32 2^E.
// The rest of a step's tokens are added in 32 bits one by one, p above 1 if need be.  Where a step does not fit E, E goes to
// its largest byte, or to the largest of its lower ones if they are more, O is rescaled exactly, and, but for a rise of up
// to 3, m goes, down or up, to the step's tokens.  (With E the largest byte met and m every token's maximum, a token of no weight
// with values 2^25 times the others' took their share of the output away.)  Ordinary steps look at one difference of bytes for it.
//
// A session of more than 8 rows per KV head goes in groups of 8, each reading the cache again (most of it from L2): up to
// 32 rows that is faster than the wide kernel.
//
// Tokens that some of a group's rows do not see are the newest ones, 7 at most: their values are added in 32 bits one
// token at a time, each row with an E of its own from there on, so that a hidden value of any size changes nothing in the
// rows that do not see it.
//
// What bounds it: issue and latency, 581 instructions of a warp per 32 tokens and head, a quarter of them the conversions of e2m1 (one
// per pair of values, at half rate), against 17 / 32 bytes per value.  Measured: 32 single tokens over 4096 to 32768 (32 query heads
// over 8 of 128, 644 MB) 173 us, 3.7 TB/s, 0.57 of the measured copy rate (8-bit cache 290 us, 16-bit 392); one token over 2000 20.5,
// over 32768 36; 16 sessions of 3 to 7 drafted tokens over 1000 to 9000 (4 query heads per KV head) 85 (the wide kernel: 131).
// (Before the window of scales 164, 18.5, 34 and 81, with other tokens' shares lost beside values 2^20 times theirs.)
// One tile of 16 tokens at a time instead of two: 193 us for the first; queries in registers spill (185).
#include <type_traits>

#include "few_common.cuh"

namespace actkv {
namespace chunk {
namespace few {
namespace four {

constexpr int kStep = 32;                   // tokens per step of a warp
constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kRoundCost = 3;               // a unit's fixed cost in rounds of its warps
constexpr int kMinRounds = 1;               // the least share of a CTA (one token over 2000: 27.6 us with 3, 25.3 with 2, 23.0 with 1)
constexpr int kRowsMax = 8;                 // query rows of a group: the products' columns
constexpr float kLowest = -3.0e38f;         // m of a row before its first token: below any logit, and finite
constexpr float kPBits = 7.0f;              // p, and l with it, is held times 2^7 (kPScale, here by way of the exponent)
constexpr int kQuerySpread = 12;            // groups of a query row whose largest values differ by more in their exponents are scaled apart
constexpr int kWindow = 7;                  // a product's tokens have scale bytes E - kWindow .. E
constexpr uint32_t kWindows = kWindow * 0x01010101u;
constexpr int kRise = 3;                    // E may rise by this before m is set anew
constexpr int kAbove = 90;                  // tokens added in 32 bits: at most this far above E,
constexpr float kOver = 100.0f;             // ... and p times the scale over 2^E at most 2^kOver

template <int D>
struct Ring4 {
  static constexpr int G = D / 32;
  static constexpr int kChunks = D / 32;                    // 16-byte pieces of a row
  static constexpr uint32_t kPlane = kStep * D / 2;         // keys, then values
  static constexpr uint32_t kStage = 2 * kPlane + 2 * kStep * 4;        // and their scale words
  static constexpr int kStages = D == 128 ? 2 : 4;          // (a step takes a warp 3 us: one ahead is enough)
  // a step's scales as its products take them: of keys in 32 bits, of values in fp16 relative to E
  static constexpr uint32_t kKeyScale = kStep * G * 4, kTable = kKeyScale + kStep * G * 2;
  static constexpr uint32_t kWarpBytes = kStages * kStage + kTable;
  static constexpr int kJoin = (D / 16 * 4 + 4) * 32;       // a warp's O, m, l as floats
  static constexpr uint32_t kBytes = kWarps * kWarpBytes, kJoinBytes = kWarps * kJoin * 4;
  static constexpr uint32_t kQ = kBytes > kJoinBytes ? kBytes : kJoinBytes, kQBytes = 8 * G * 512;   // 8 heads' queries
  static constexpr uint32_t kBack = kQ + kQBytes, kWords = kBack + 8 * 8 * G * 4;     // ... what undoes their powers of two, a word per warp
  static constexpr uint32_t kSmemBytes = kWords + kWarps * 4 + 512;
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
};

// Token of the 16 (of the 8) that row i of a product is: pairs (2 c, 2 c + 1) of rows are the pairs of tokens that a lane takes
// of the values, and with these the eight lanes that read together find their pieces in different banks.
__device__ __forceinline__ int token_of(int i) { return i ^ (i >> 1 & 1); }
// Where piece c of 16 bytes of token row r is kept.
template <int D>
__device__ __forceinline__ int piece(int r, int c) { return D == 128 ? c ^ ((r >> 2 & 1) << 1) : c; }

// 2^(b - 127), and 2^d (0 from -127 down).
__device__ __forceinline__ float pow2_of(uint32_t b) { return __uint_as_float(max(b << 23, 0x00400000u)); }
__device__ __forceinline__ float pow2(int d) { return __uint_as_float(uint32_t(min(max(127 + d, 0), 254)) << 23); }

// fp16 reads: what the value pair h of scale byte b stands for as fp16 has it (subnormals rounded, past the range the
// largest), divided by the scale of byte `held(b)`.
__device__ __forceinline__ uint32_t held(uint32_t b) { return min(max(b, 104u), 140u); }
__device__ __forceinline__ uint32_t as_fp16(uint32_t h, uint32_t b_lo, uint32_t b_hi) {
  auto one = [](__half x, uint32_t b) {
    const int by = int(b) - int(held(b));
    if (by > 0) return __hmin(__hmax(__hmul(x, __float2half_rn(pow2(min(by, 15)))),
                                     __ushort_as_half(0xc7ffu)), __ushort_as_half(0x47ffu));        // 65504 / 2^13
    if (by < 0) {                             // to multiples of a half: fp16's smallest number over 2^-23
      const __half y = __hmul(x, __float2half_rn(pow2(max(by, -24))));
      return __hsub(__hadd(y, __ushort_as_half(0x6200u)), __ushort_as_half(0x6200u));
    }
    return x;
  };
  const __half2 x = reinterpret_cast<const __half2&>(h);
  const __half2 y = __halves2half2(one(__low2half(x), b_lo), one(__high2half(x), b_hi));
  return reinterpret_cast<const uint32_t&>(y);
}

// Keeps a value in a register that the compiler would work out again at every use (of the 630 instructions of a step 70
// were such).
template <typename T>
__device__ __forceinline__ void keep(T& x) { asm volatile("" : "+r"(x)); }
// The low half bytes of u with the high ones of v.
__device__ __forceinline__ uint32_t low_halves(uint32_t u, uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, 0x0f0f0f0f, 0xe4;" : "=r"(r) : "r"(u), "r"(v));
  return r;
}
// The first product of a sum.
__device__ __forceinline__ void mma16816_new(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) chunk_few4_kernel(const __grid_constant__ ChunkArgs a, bool vec_out) {
  using Rg = Ring4<D>;
  constexpr int G = Rg::G, CH = Rg::kChunks, kRowsPerCopy = 32 / CH, kCopies = kStep / kRowsPerCopy;
  constexpr int kOut = D / 16;                // products of O: two per group
  constexpr int kTiles = kStep / 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5;
  int lane = threadIdx.x & 31;
  keep(lane);
  const int r8 = lane >> 2, c4 = lane & 3;
  auto value_piece = [&](int t) -> uint32_t { return t * (D / 2) + (D == 128 ? piece<D>(t, r8 >> 1) * 16 + (r8 & 1) * 8 : r8 * 4); };
  Sched& sched = *reinterpret_cast<Sched*>(smem + Rg::kSmemBytes - 512);
  const int cta = blockIdx.x, n_cta = gridDim.x;
  const uint32_t ring = smem_u32(smem) + warp * Rg::kWarpBytes, table_at = ring + Rg::kStages * Rg::kStage;
  const unsigned full = 0xffffffffu;
  const float ninf = -__int_as_float(0x7f800000);
  // where the lane reads within a stage and the tables; tiles of 16 tokens, and 8 tokens within one, are constant steps on
  const int row_tok = token_of(r8);
  uint32_t key_at = row_tok * (D / 2) + (D == 128 ? piece<D>(row_tok, c4) * 16 : c4 * 8);
  uint32_t value_at = value_piece(token_of(2 * c4));  // ... and the other token's of the pair: the bit of token 1 turned
  uint32_t key_scale = table_at + row_tok * (G * 4), value_scale = table_at + Rg::kKeyScale + c4 * (G * 4);
  // ... and where it puts its token's: the second of a pair of tokens takes the second half of the groups
  const int odd = token_of(lane & 7) & 1;
  uint32_t pair_at = table_at + Rg::kKeyScale + ((lane >> 3) * 4 + (token_of(lane & 7) >> 1)) * (G * 4) + odd * (G * 2);
  uint32_t copy_at = lane / CH * (CH * 16) + piece<D>(lane / CH, lane % CH) * 16;
  keep(key_at);
  keep(value_at);
  keep(key_scale);
  keep(value_scale);
  keep(pair_at);
  keep(copy_at);
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
  // A session's rows go in groups of up to 8 (whole tokens), each reading the tokens that some row of it sees.
  const int per_group = kRowsMax / a.G;
  auto rounds = [&](int sees) { return (held_tokens(a, sees) + round - 1) / round; };
  auto rounds_of = [&](int A, int S) {        // of one group of heads, with the groups' fixed costs
    int n = 0;
    for (int j = 0; j < A; j += per_group) n += kRoundCost + rounds(S - A + min(A, j + per_group));
    return n;
  };
  share_out<kThreads>(a.R, [&](int r) -> int64_t {
    const int A = new_tokens(a, r), S = a.seq_used[r];
    if (A == 0 || A * a.G > few_rows) return 0;
    flag_long(a, S);
    return int64_t(a.Hkv / HG) * rounds_of(A, S);
  }, sched.share, sched.scan, cta, n_cta, kMinRounds);
  // The share is [lo, lo + span) of the schedule; places in it are kept relative to lo, in 32 bits (registers are short).
  auto n_used = [&] { return used_ctas(sched.share.total, n_cta, kMinRounds); };
  auto low = [&] { return sched.share.total * cta / n_used(); };
  if (cta >= n_used()) return;
  const int span = int(sched.share.total * (cta + 1) / n_used() - low());
  if (span <= 0) return;
  int r = sched.share.r0;
  int at = int(sched.share.pre - low());     // start of (session r, head group hg) in the schedule
  int hg = 0;
  bool seek = true;
  const float c2 = a.scale * kLog2e;
  const int shift = (a.BS & (a.BS - 1)) == 0 ? __ffs(a.BS) - 1 : -1;
  auto block_of = [&](int tok) { return shift >= 0 ? tok >> shift : tok / a.BS; };
  auto bytes_at = [&](int64_t off) { return static_cast<const char*>(a.kv) + off; };

  for (; r < a.R && at < span; ++r, hg = 0) {
    int A = new_tokens(a, r);
    const int S = a.seq_used[r];
    if (A == 0 || A * a.G > few_rows) continue;
    if (seek) {                               // the group of heads that holds lo
      const int each = rounds_of(A, S);
      hg = -at / each;
      at += hg * each;
      seek = false;
    }
    for (int j0 = 0; hg < a.Hkv / HG && at < span; j0 = j0 + per_group < A ? j0 + per_group : 0, hg += j0 == 0) {
      int ntok = min(per_group, A - j0), rows = ntok * a.G;
      const int all = a.seq_used[r] - A + j0; // tokens that all rows see: up to this one
      int nt = rounds(all + ntok), first = at + kRoundCost;
      at += kRoundCost + nt;
      int t0 = max(-first, 0), t1 = nt == 0 ? 0 : min(nt, span - first);
      if (nt == 0 ? first < kRoundCost : t0 >= t1) continue;
      int h = hg * HG + my_head;
      const int32_t* table = a.block_table + r * a.bt_stride_r;
      int begin = t0 * round;
      const int end = min(t1 * round, held_tokens(a, all + ntok));
      const int start = begin + my_part * kStep;              // this warp's steps: start, start + round, ...
      const int mine = start < end ? (end - start + round - 1) / round : 0;
      // the lane's two query rows; the first sees the tokens up to all + row0 / G, the second up to all + row1 / G
      const int row0 = 2 * c4, row1 = row0 + 1;
      // ---- queries as the second operand, row r8: of k-step (group g, i) dims 32 g + 8 c4 + 4 i .. + 3
      uint32_t q[2 * G][2];
      {
        const int jq = r8 / a.G;
        const uint16_t* p = static_cast<const uint16_t*>(a.q) + (int64_t(a.q_off[r]) + j0 + jq) * a.q_stride_t +
                            int64_t(h * a.G + r8 - jq * a.G) * a.q_stride_h;
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) {
          const uint2 u = r8 < rows ? *reinterpret_cast<const uint2*>(p + 32 * (k >> 1) + 8 * c4 + 4 * (k & 1)) : make_uint2(0u, 0u);
          q[k][0] = u.x;
          q[k][1] = u.y;
        }
      }
      // scale * log2 e, and what undoes the queries' power of two, for rows row0 and row1
      float cq0 = c2, cq1 = c2;
      uint32_t rare = 0;                      // what no ordinary step looks at:
      constexpr uint32_t kGaps = 1;           // this lane met a block outside the cache: from there on every step looks
      constexpr uint32_t kStale = 2;          // m is not of the products' tokens: the next of them set it
      constexpr uint32_t kUneven = 4;         // the rows' E differ (from there on no token is in all rows)
      constexpr uint32_t kSpread = 8;         // the queries' groups have powers of two of their own
      if constexpr (BF16) {
        uint32_t tops[G], top = 0, least = 0x7f80u;           // the groups' largest finite values, by their bits
#pragma unroll
        for (int g = 0; g < G; ++g) {
          tops[g] = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t u = q[2 * g + (e >> 1)][e & 1], x = u & 0x7fffu, y = u >> 16 & 0x7fffu;
            tops[g] = max(tops[g], max(x < 0x7f80u ? x : 0u, y < 0x7f80u ? y : 0u));
          }
          tops[g] = max(tops[g], __shfl_xor_sync(full, tops[g], 1));
          tops[g] = max(tops[g], __shfl_xor_sync(full, tops[g], 2));
          top = max(top, tops[g]);
          if (tops[g] > 0) least = min(least, tops[g]);
        }
        const bool spread = __any_sync(full, top > 0 && (least >> 7) + kQuerySpread < (top >> 7));
        if (spread) rare = kSpread;
        float back = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int by = min(141 - int((spread && tops[g] > 0 ? tops[g] : top) >> 7), 126);
          const float f = pow2(by);
          back = pow2(-by);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t& u = q[2 * g + (e >> 1)][e & 1];
            u = pack2<false>(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f);
          }
          if (my_part == 0 && c4 == 0) reinterpret_cast<float*>(smem + Rg::kBack)[(my_head * 8 + r8) * G + g] = back;
        }
        cq0 *= __shfl_sync(full, back, 4 * row0);             // (of use where the groups share it)
        cq1 *= __shfl_sync(full, back, 4 * row1);
      }
      // ... in shared memory, the head's first warp putting them there: they are read again for every tile
      if (my_part == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g)
          *reinterpret_cast<uint4*>(smem + Rg::kQ + (my_head * G + g) * 512 + lane * 16) =
              make_uint4(q[2 * g][0], q[2 * g][1], q[2 * g + 1][0], q[2 * g + 1][1]);
      }
      // What the steps have no use for waits in shared memory (as spilled registers they came back in every step: 185 us for
      // 32 single tokens of 4096 to 32768, 171 so).
      if (threadIdx.x == 0) {
        const int u[10] = {r, hg, j0, at, A, nt, first, t0, t1, ntok};
#pragma unroll
        for (int i = 0; i < 10; ++i) sched.unit[i] = u[i];
        sched.bad_v = 0;
      }
      __syncthreads();
      const uint32_t q_at = smem_u32(smem) + Rg::kQ + my_head * (G * 512) + lane * 16;
      float o[kOut][4];
#pragma unroll
      for (int j = 0; j < kOut; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
      float m0 = kLowest, m1 = kLowest, l0 = 0.0f, l1 = 0.0f;
      // by group (a byte each), what O is relative to, 2^(E - 127), for the two rows; equal until tokens are added one by one
      uint32_t E0 = 0, E1 = 0;
      auto byte_of = [](uint32_t w, int g) { return int(w >> (8 * g) & 255u); };

      // ---- copies of step i of this warp: a lane looks up its token's block a step ahead
      auto look_up = [&](int i) -> int {
        const int tok = start + i * round + lane;
        if (i >= mine || tok >= end) return -1;
        const int lb = block_of(tok);
        return lb < a.MB ? table[lb] : -1;
      };
      int phys = look_up(0);
      const char* const head = static_cast<const char*>(a.kv) + (h * (D / 2) + lane % CH * 16);
      const int at_word = a.Hkv * (D / 2) + (D == 128 ? h * 4 : (h * 2) & ~3);
      const int sh = D == 64 && (h & 1) ? 16 : 0;             // the head's bytes within the word
      auto issue = [&](int i, int slot) {
        if (i < mine) {
          const int tok = start + i * round + lane;
          const bool none = uint32_t(phys) >= uint32_t(a.NB); // past the end, or an id outside the cache
          if (none && tok < end) {
            flag(a.status, ACTKV_DEV_BAD_INDEX);
            rare |= kGaps;
          }
          // The token's place, in tokens (blocks are whole and in order, and all of them fewer than 2^31, a token's bytes too).
          // One that is not there takes the cache's first: it is hidden, and nothing of a hidden token counts.
          const uint32_t place = none ? 0u : uint32_t(phys * a.BS + (shift >= 0 ? tok & (a.BS - 1) : tok % a.BS));
          const uint32_t stride = uint32_t(a.kv_stride_s), dst = ring + slot * Rg::kStage;
#pragma unroll
          for (int e = 0; e < kCopies; ++e) {
            const int row = e * kRowsPerCopy + lane / CH;
            const char* p = head + uint64_t(__shfl_sync(full, place, row)) * stride;
            const uint32_t to = dst + copy_at + e * 512;
            copy16(to, p, true);
            copy16(to + Rg::kPlane, p + a.kv_stride_kv, true);
          }
          const char* w = static_cast<const char*>(a.kv) + at_word + uint64_t(place) * stride;
          copy4(dst + 2 * Rg::kPlane + lane * 4, w, true);
          copy4(dst + 2 * Rg::kPlane + kStep * 4 + lane * 4, w + a.kv_stride_kv, true);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        phys = look_up(i + 1);
      };

      // the rows' references go to those given (the same in all lanes of a row; each row by its own tokens alone, so
      // that what others see does not show in its digits)
      auto move = [&](float n0, float n1) {
        const float e0 = m0 == n0 ? 1.0f : ex2(m0 - n0), e1 = m1 == n1 ? 1.0f : ex2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= e0;
        l1 *= e1;
#pragma unroll
        for (int j = 0; j < kOut; ++j) {
          o[j][0] *= e0;
          o[j][1] *= e1;
          o[j][2] *= e0;
          o[j][3] *= e1;
        }
      };
      // ... and the scales' references
      auto move_scale = [&](uint32_t n0, uint32_t n1) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float e0 = pow2(byte_of(E0, g) - byte_of(n0, g)), e1 = pow2(byte_of(E1, g) - byte_of(n1, g));
#pragma unroll
          for (int j = 2 * g; j < 2 * g + 2; ++j) {
            o[j][0] *= e0;
            o[j][1] *= e1;
            o[j][2] *= e0;
            o[j][3] *= e1;
          }
        }
        E0 = n0;
        E1 = n1;
      };
      // the value bytes of a scale word as they are held, 0 for NaN
      auto counted = [&](uint32_t w) -> uint32_t {
        uint32_t x = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t b = byte_of(w, g);
          if (b < kNan4) x |= (BF16 ? b : held(b)) << (8 * g);
        }
        return x;
      };
      // The next E where a step's bytes (top: 0 for what does not count, low: 255) do not fit the present one.
      auto fit = [&](uint32_t top, uint32_t low) -> uint32_t {
        uint32_t next = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t b = byte_of(top, g), now = byte_of(E0, g);
          const bool in = byte_of(low, g) < 255;
          const uint32_t hi = __reduce_max_sync(full, b), lo = __reduce_min_sync(full, in ? b : 255u);
          uint32_t n = now;
          if (lo <= hi && (hi > now || lo + kWindow < now)) {
            n = hi;
            if (hi - lo > kWindow) {
              const int high = __popc(__ballot_sync(full, in && b + kWindow >= hi)), small = __popc(__ballot_sync(full, in && b <= lo + kWindow));
              const uint32_t most = __reduce_max_sync(full, in && b <= lo + kWindow ? b : 0u);
              if (small > high) n = max(most, hi > kAbove ? hi - kAbove : 0u);
            }
            if (n < now) {                    // O stays finite
              uint32_t o_top = 0;
#pragma unroll
              for (int j = 2 * g; j < 2 * g + 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t y = __float_as_uint(o[j][e]) & 0x7fffffffu;
                  o_top = max(o_top, y < 0x7f800000u ? y : 0u);
                }
              const int room = max(247 - int(__reduce_max_sync(full, o_top) >> 23), 0);
              n = uint32_t(max(int(n), int(now) - room));
            }
          }
          next |= n << (8 * g);
        }
        return next;
      };
      // how far E may rise before m is set anew
      volatile uint32_t* const E_set = reinterpret_cast<uint32_t*>(smem + Rg::kWords) + warp;
      *E_set = kRise * 0x01010101u;           // (a unit may begin with bytes that fit E = 0)
      __syncwarp();
      // there: the step's tokens that are there (neither past the end nor in a block outside the cache); fast: those of them
      // that every row sees and whose bytes vs fit E; restart: they set m
      auto step = [&](int i, int slot, uint32_t wk, uint32_t wv, uint32_t there, uint32_t fast, uint32_t vs, bool restart, auto edge_) {
        constexpr bool EDGE = decltype(edge_)::value;        // other tokens too, or scale bytes out of the ordinary
        const int t = start + i * round;
        const uint32_t kb = ring + slot * Rg::kStage, vb = kb + Rg::kPlane, sb = kb + 2 * Rg::kPlane;
        [[maybe_unused]] int lim0 = 0, lim1 = 0;             // the last tokens that the lane's rows see
        if constexpr (EDGE) {
          lim0 = all + row0 / a.G;
          lim1 = all + row1 / a.G;
        }
        // (its address worked out here and read where it is used: kept over the loops below it spilled 128 bytes)
        uint32_t back_at = 0;
        if constexpr (EDGE && BF16) {
          back_at = smem_u32(smem) + Rg::kBack + (my_head * 8 + row0) * (G * 4);
          keep(back_at);
        }
        [[maybe_unused]] const volatile float* const backs = reinterpret_cast<const float*>(smem + (back_at - smem_u32(smem)));
        // ---- the lane's token: its scales into the tables
        {
          float ks[G];
          if constexpr (EDGE) {
#pragma unroll
            for (int g = 0; g < G; ++g)
              if (byte_of(wv, g) >= int(kNan4) && (there >> lane & 1u)) atomicOr(&sched.bad_v, 2);   // it comes back when the unit ends
          }
#pragma unroll
          for (int g = 0; g < G; ++g) {
            uint32_t b = byte_of(wk, g);
            if constexpr (EDGE && !BF16)
              if (b < kNan4) b = held(b);
            ks[g] = EDGE && b >= kNan4 ? __int_as_float(0x7fffffff) : pow2_of(b);
          }
          uint8_t* const tables = smem + (table_at - smem_u32(smem));
          if constexpr (G == 4) *reinterpret_cast<float4*>(tables + lane * 16) = make_float4(ks[0], ks[1], ks[G - 2], ks[G - 1]);
          else *reinterpret_cast<float2*>(tables + lane * 8) = make_float2(ks[0], ks[1]);
          // 2^(b - E) in fp16 (of equal E0 and E1), two groups' next to one another; 0 for other tokens' and NaN
          uint32_t f[G / 2];
          // (by byte: none of vs is above E0's or more than kWindow below, but for those that do not count)
          const uint32_t up = 0x0f0f0f0fu - (EDGE ? (E0 - vs) & kWindows : E0 - vs);
#pragma unroll
          for (int g = 0; g < G; g += 2) {
            f[g / 2] = (up >> (8 * g) & 0xffu) << 10 | (up >> (8 * g) & 0xff00u) << 18;
            if constexpr (EDGE) {
              const bool in = fast >> lane & 1u;
              if (!in || byte_of(wv, g) >= int(kNan4)) f[g / 2] &= 0xffff0000u;
              if (!in || byte_of(wv, g + 1) >= int(kNan4)) f[g / 2] &= 0x0000ffffu;
            }
          }
          // by pair of tokens and group, the pair's factors: each of the two lanes puts half of the groups
          if constexpr (G == 4) {
            const uint32_t got = __shfl_xor_sync(full, odd ? f[0] : f[G / 2 - 1], 1);
            const uint32_t lo = odd ? got : f[0], hi = odd ? f[G / 2 - 1] : got;
            *reinterpret_cast<uint2*>(smem + (pair_at - smem_u32(smem))) =
                make_uint2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
          } else {
            const uint32_t got = __shfl_xor_sync(full, f[0], 1);
            *reinterpret_cast<uint32_t*>(smem + (pair_at - smem_u32(smem))) =
                odd ? __byte_perm(got, f[0], 0x7632) : __byte_perm(f[0], got, 0x5410);
          }
        }
        __syncwarp();
        // ---- S^T = K Q^T: s[n][0..1] token 16 n + token_of(r8), s[n][2..3] the one 8 on, query rows 2 c4 and 2 c4 + 1
        float s[kTiles][4];
        uint32_t w[kTiles][2][2 * (G / 2)];   // by tile and token: words of pieces 2 c4 and 2 c4 + 1
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int on = 16 * n + 8 * e;
            if constexpr (D == 128) {
              const uint4 u = lds16(kb + key_at + on * 64);
              w[n][e][0] = u.x;
              w[n][e][1] = u.y;
              w[n][e][G - 2] = u.z;
              w[n][e][G - 1] = u.w;
            } else {
              const uint2 u = lds8(kb + key_at + on * 32);
              w[n][e][0] = u.x;
              w[n][e][1] = u.y;
            }
          }
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
        for (int g2 = 0; g2 < G / 2; ++g2) {
          const uint4 q0 = lds16(q_at + 2 * g2 * 512), q1 = lds16(q_at + (2 * g2 + 1) * 512);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            // of two groups: x[token][piece][byte]
            uint32_t x[2][2][4];
            uint2 ks[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              ks[e] = lds8(key_scale + (16 * n + 8 * e) * (G * 4) + g2 * 8);
#pragma unroll
              for (int pc = 0; pc < 2; ++pc)
                e2m1x8_f16(w[n][e][pc * (G / 2) + g2], x[e][pc][0], x[e][pc][1], x[e][pc][2], x[e][pc][3]);
            }
#pragma unroll
            for (int gg = 0; gg < 2; ++gg) {
              if constexpr (EDGE && !BF16) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t b = lds4(sb + (16 * n + 8 * e + row_tok) * 4) >> (sh + 8 * (2 * g2 + gg)) & 255u;
#pragma unroll
                  for (int pc = 0; pc < 2; ++pc)
#pragma unroll
                    for (int k = 0; k < 2; ++k) x[e][pc][2 * gg + k] = as_fp16(x[e][pc][2 * gg + k], b, b);
                }
              }
              float c[4], qs0 = 1.0f, qs1 = 1.0f;             // (and what undoes the queries' power of two)
              if constexpr (EDGE && BF16) {
                qs0 = backs[2 * g2 + gg];
                qs1 = backs[G + 2 * g2 + gg];
              }
              const uint4 qg = gg ? q1 : q0;
#pragma unroll
              for (int pc = 0; pc < 2; ++pc) {
                const uint32_t m[4] = {x[0][pc][2 * gg], x[1][pc][2 * gg], x[0][pc][2 * gg + 1], x[1][pc][2 * gg + 1]};
                if (pc == 0) mma16816_new(c, m, qg.x, qg.y);
                else mma16816<false>(c, m, qg.z, qg.w);
              }
              // (powers of two, the same digits with the queries' or without; the smaller one first, so that scales of any size
              // stay in range, beside sums of 0 too)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float k = __uint_as_float(gg ? ks[e >> 1].y : ks[e >> 1].x), qs = e & 1 ? qs1 : qs0;
                if constexpr (EDGE) s[n][e] = k < qs ? fmaf(c[e] * k, qs, s[n][e]) : fmaf(c[e] * qs, k, s[n][e]);
                else s[n][e] = fmaf(c[e], k, s[n][e]);
              }
            }
          }
        }
        if constexpr (EDGE) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int tk = 16 * n + 8 * (e >> 1) + row_tok;
              s[n][e] = t + tk <= (e & 1 ? lim1 : lim0) && (there >> tk & 1u) ? s[n][e] : ninf;
            }
        }
        // (the product rounded before the difference, not in one step with it: the largest logit's is then 0 whatever its size)
        const float f0 = EDGE ? a.scale * kLog2e : cq0, f1 = EDGE ? a.scale * kLog2e : cq1;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = __fmul_rn(s[n][e], e & 1 ? f1 : f0);
        // the largest of the products' tokens
        auto of_products = [&](int n, int e) { return !EDGE || (fast >> row_tok >> (16 * n + 8 * (e >> 1)) & 1u) ? s[n][e] : ninf; };
        float top0 = fmaxf(of_products(0, 0), of_products(0, 2)), top1 = fmaxf(of_products(0, 1), of_products(0, 3));
#pragma unroll
        for (int n = 1; n < kTiles; ++n) {
          top0 = fmaxf(top0, fmaxf(of_products(n, 0), of_products(n, 2)));
          top1 = fmaxf(top1, fmaxf(of_products(n, 1), of_products(n, 3)));
        }
        bool moves = top0 > m0 + kSlack || top1 > m1 + kSlack;
        // ... and of the others: logits with the scales, which p times the scale must not outgrow; those that some row does not see
        [[maybe_unused]] float far0 = ninf, far1 = ninf, last0 = ninf, last1 = ninf;
        if constexpr (EDGE) {
          const uint32_t others = there & ~fast;
          if (others) {
            // (in ordinary steps none is near: the largest logit, the largest scale above E)
            auto above = [&](uint32_t bytes, uint32_t E) {
              const uint32_t y = __vsubus4(bytes, E);
              return min(max(max(byte_of(y, 0), byte_of(y, 1)), max(byte_of(y, 2), byte_of(y, 3))), kAbove);
            };
            const uint32_t bytes = counted(wv);
            const float most = float(__reduce_max_sync(full, others >> lane & 1u ? above(bytes, E0) : 0)) - kOver;
            float all0 = fmaxf(s[0][0], s[0][2]), all1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
            for (int n = 1; n < kTiles; ++n) {
              all0 = fmaxf(all0, fmaxf(s[n][0], s[n][2]));
              all1 = fmaxf(all1, fmaxf(s[n][1], s[n][3]));
            }
            if (__any_sync(full, (rare & kUneven) || moves || restart || all0 + most > m0 || all1 + most > m1)) {
#pragma unroll
              for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int tk = 16 * n + 8 * (e >> 1) + row_tok;
                  const int lift = above(__shfl_sync(full, bytes, tk), e & 1 ? E1 : E0);
                  if (fast >> tk & 1u) continue;
                  (e & 1 ? far1 : far0) = fmaxf(e & 1 ? far1 : far0, s[n][e] + float(lift));
                  if (t + tk > all) (e & 1 ? last1 : last0) = fmaxf(e & 1 ? last1 : last0, s[n][e]);
                }
              moves = true;
            }
          }
          moves |= restart;
        }
        if (__any_sync(full, moves)) {
#pragma unroll
          for (int x = 4; x < 32; x *= 2) {
            top0 = fmaxf(top0, __shfl_xor_sync(full, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(full, top1, x));
          }
          if constexpr (EDGE) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
              far0 = fmaxf(far0, __shfl_xor_sync(full, far0, x));
              far1 = fmaxf(far1, __shfl_xor_sync(full, far1, x));
              last0 = fmaxf(last0, __shfl_xor_sync(full, last0, x));
              last1 = fmaxf(last1, __shfl_xor_sync(full, last1, x));
            }
            float room0 = 0.0f, room1 = 0.0f;                // what m may go down by: as long as O and l stay finite
            if (restart) {
              uint32_t y0 = __float_as_uint(l0), y1 = __float_as_uint(l1);
              y0 = y0 < 0x7f800000u ? y0 : 0u;
              y1 = y1 < 0x7f800000u ? y1 : 0u;
#pragma unroll
              for (int j = 0; j < kOut; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t y = __float_as_uint(o[j][e]) & 0x7fffffffu;
                  (e & 1 ? y1 : y0) = max(e & 1 ? y1 : y0, y < 0x7f800000u ? y : 0u);
                }
#pragma unroll
              for (int x = 4; x < 32; x *= 2) {
                y0 = max(y0, __shfl_xor_sync(full, y0, x));
                y1 = max(y1, __shfl_xor_sync(full, y1, x));
              }
              room0 = float(min(max(237 - int(y0 >> 23), 0), 120));
              room1 = float(min(max(237 - int(y1 >> 23), 0), 120));
            }
            auto next = [&](float m, float top, float far, float last, float room) {
              float n = m;
              if (top > m + kSlack || (restart && top > kLowest)) n = fmaxf(top, m - room);
              // nothing before: p of at most 1, where that costs the products' tokens little
              if (m == kLowest) n = fmaxf(n, n == kLowest ? last : fminf(last, n + 4.0f));
              return fmaxf(n, far - kOver);
            };
            move(next(m0, top0, far0, last0, room0), next(m1, top1, far1, last1, room1));
          } else {
            move(top0 > m0 + kSlack ? top0 : m0, top1 > m1 + kSlack ? top1 : m1);
          }
        }
        const float base0 = m0 - kPBits, base1 = m1 - kPBits;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = ex2(__fsub_rn(s[n][e], e & 1 ? base1 : base0));
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          l0 += s[n][0] + s[n][2];
          l1 += s[n][1] + s[n][3];
        }
        // ---- O^T += V^T p^T: the lane's tokens are those of rows 2 c4, 2 c4 + 1 and 8 on, its dims 4 r8 .. + 3 of each group
        if (!EDGE || fast) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            uint32_t p0 = pack2<false>(s[n][0], s[n][1]), p1 = pack2<false>(s[n][2], s[n][3]);
            if constexpr (EDGE) {             // (the others' may be infinite in fp16)
              if (!(fast >> row_tok >> (16 * n) & 1u)) p0 = 0;
              if (!(fast >> row_tok >> (16 * n + 8) & 1u)) p1 = 0;
            }
            p0 = transpose8x8(p0);
            p1 = transpose8x8(p1);
            uint32_t vw[4][G / 2], ft[2][G];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int on = 16 * n + 8 * (e >> 1);
              if constexpr (D == 128) {
                const uint2 u = lds8(vb + (e & 1 ? value_at ^ 64u : value_at) + on * 64);
                vw[e][0] = u.x;
                vw[e][G / 2 - 1] = u.y;
              } else {
                vw[e][0] = lds4(vb + (e & 1 ? value_at ^ 32u : value_at) + on * 32);
              }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if constexpr (G == 4) {
                const uint4 f = lds16(value_scale + (2 * n + e) * 4 * (G * 4));
                ft[e][0] = f.x;
                ft[e][1] = f.y;
                ft[e][G - 2] = f.z;
                ft[e][G - 1] = f.w;
              } else {
                const uint2 f = lds8(value_scale + (2 * n + e) * 4 * (G * 4));
                ft[e][0] = f.x;
                ft[e][1] = f.y;
              }
            }
#pragma unroll
            for (int g2 = 0; g2 < G / 2; ++g2) {
              // two tokens' half bytes of a dim next to one another: even dims, odd dims; x[pair][odd][byte]
              uint32_t x[2][2][4];
#pragma unroll
              for (int pr = 0; pr < 2; ++pr) {
                const uint32_t u = vw[2 * pr][g2], v = vw[2 * pr + 1][g2];
                const uint32_t even = low_halves(u, v * 16u), odd = low_halves(u >> 4, v);
                e2m1x8_f16(even, x[pr][0][0], x[pr][0][1], x[pr][0][2], x[pr][0][3]);
                e2m1x8_f16(odd, x[pr][1][0], x[pr][1][1], x[pr][1][2], x[pr][1][3]);
              }
#pragma unroll
              for (int gg = 0; gg < 2; ++gg) {
                const int g = 2 * g2 + gg;
                if constexpr (EDGE && !BF16) {
#pragma unroll
                  for (int pr = 0; pr < 2; ++pr) {
                    const uint32_t at = sb + (kStep + 16 * n + 8 * pr) * 4;
                    const uint32_t b_lo = lds4(at + token_of(2 * c4) * 4) >> (sh + 8 * g) & 255u;
                    const uint32_t b_hi = lds4(at + token_of(2 * c4 + 1) * 4) >> (sh + 8 * g) & 255u;
#pragma unroll
                    for (int od = 0; od < 2; ++od)
#pragma unroll
                      for (int k = 0; k < 2; ++k) x[pr][od][2 * gg + k] = as_fp16(x[pr][od][2 * gg + k], b_lo, b_hi);
                  }
                }
                const uint32_t pg0 = mul16x2<false>(p0, ft[0][g]), pg1 = mul16x2<false>(p1, ft[1][g]);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const uint32_t m[4] = {x[0][0][2 * gg + k], x[0][1][2 * gg + k], x[1][0][2 * gg + k], x[1][1][2 * gg + k]};
                  mma16816<false>(o[2 * g + k], m, pg0, pg1);
                }
              }
            }
          }
        }
        // ---- the other tokens, one by one: first those outside the window, then those that some row does not see
        if constexpr (EDGE) {
#pragma unroll 1
          for (uint32_t some = there & ~fast; some; some &= some - 1) {
            const int tk = __ffs(some) - 1, of = tk & 7;
            // p of the lane's two rows: from the lanes of the product's row that the token is
            float x0 = 0.0f, x1 = 0.0f;
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if ((tk >> 3) == 2 * n + e) {
                  x0 = s[n][2 * e];
                  x1 = s[n][2 * e + 1];
                }
            x0 = __shfl_sync(full, x0, token_of(of) * 4 + c4);
            x1 = __shfl_sync(full, x1, token_of(of) * 4 + c4);
            const bool see0 = t + tk <= lim0, see1 = t + tk <= lim1;
            const uint32_t word = lds4(sb + (kStep + tk) * 4) >> sh;
            const uint32_t seen = counted(word), least = __vsubus4(seen, kAbove * 0x01010101u);
            const uint32_t n0 = see0 ? __vmaxu4(E0, least) : E0, n1 = see1 ? __vmaxu4(E1, least) : E1;
            if (__any_sync(full, n0 != E0 || n1 != E1)) {
              move_scale(n0, n1);
              rare |= kUneven;
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const uint32_t b = byte_of(word, g);
              if (b >= kNan4) continue;
              const int by0 = byte_of(seen, g) - byte_of(E0, g), by1 = byte_of(seen, g) - byte_of(E1, g);
              const float g0 = see0 ? x0 * pow2(by0) : 0.0f, g1 = see1 ? x1 * pow2(by1) : 0.0f;
              // the lane's four dims of the group: two bytes of piece r8
              const uint32_t byte_at = D == 128 ? tk * 64 + piece<D>(tk, r8 >> 1) * 16 + (r8 & 1) * 8 : tk * 32 + r8 * 4;
              const uint32_t two = lds4(vb + byte_at + (g >> 1) * 4) >> (16 * (g & 1));
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                uint32_t v = e2m1x2_f16(two >> (8 * k) & 255u);
                if constexpr (!BF16) v = as_fp16(v, b, b);
                const float2 y = f16x2_f32(v);
                o[2 * g + k][0] = fmaf(g0, y.x, o[2 * g + k][0]);
                o[2 * g + k][1] = fmaf(g1, y.x, o[2 * g + k][1]);
                o[2 * g + k][2] = fmaf(g0, y.y, o[2 * g + k][2]);
                o[2 * g + k][3] = fmaf(g1, y.y, o[2 * g + k][3]);
              }
            }
          }
          rare = fast == 0 ? rare | kStale : rare & ~kStale;
        }
      };

      // ---- the steps
      constexpr int kAhead = Rg::kStages - 1;
#pragma unroll 1
      for (int i = 0; i < kAhead; ++i) issue(i, i);
#pragma unroll 1
      for (int i = 0; i < mine; ++i) {
        const int slot = i % Rg::kStages;
        issue(i + kAhead, (i + kAhead) % Rg::kStages);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
        __syncwarp();
        const int t = start + i * round;
        const uint32_t sb = ring + slot * Rg::kStage + 2 * Rg::kPlane;
        uint32_t wk = lds4(sb + lane * 4) >> sh, wv = lds4(sb + (kStep + lane) * 4) >> sh;
        if constexpr (D == 64) {
          wk &= 0xffffu;
          wv &= 0xffffu;
        }
        // bits of what is out of the ordinary: scale bytes, values' outside the window, and what the steps so far left behind
        uint32_t odd = rare;
        if constexpr (BF16) odd |= ((wk & (wk << 1)) | (wv & (wv << 1))) & 0x80808080u;
        else odd |= __vcmpgtu4(wk, 0x8c8c8c8cu) | __vcmpgtu4(wv, 0x8c8c8c8cu) |
                    ((__vcmpgtu4(0x68686868u, wk) | __vcmpgtu4(0x68686868u, wv)) & (D == 64 ? 0xffffu : 0xffffffffu));
        const uint32_t off = (E0 - wv) & ~kWindows;
        const bool ends = t + kStep - 1 > all || t + kStep > end;
        uint32_t there = 0, fast = 0, vs = 0;
        bool edge = false, restart = false;
        if (ends || __any_sync(full, (odd | off) != 0)) {
          edge = ends || __any_sync(full, odd != 0);
          restart = rare & kStale;
          bool here = t + lane < end;
          if (__any_sync(full, rare & kGaps) && here) {
            const int lb = block_of(t + lane);
            here = lb < a.MB && uint32_t(table[lb]) < uint32_t(a.NB);
          }
          there = __ballot_sync(full, here);
          fast = there & __ballot_sync(full, t + lane <= all);
          // the lane's bytes that count, and with 255 in place of the others
          vs = fast >> lane & 1u ? counted(wv) : 0u;
          uint32_t low = vs;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (!(fast >> lane & 1u) || g >= G || byte_of(wv, g) >= int(kNan4)) low |= 255u << (8 * g);
          auto outside = [&] { return (__vcmpgtu4(vs, E0) | __vcmpgtu4(__vsubus4(E0, kWindows), low)) != 0; };
          if (__any_sync(full, outside())) {
            uint32_t n = __vmaxu4(vs, E0);    // the larger E, where that will do
#pragma unroll
            for (int x = 1; x < 32; x *= 2) n = __vmaxu4(n, __shfl_xor_sync(full, n, x));
            if (__any_sync(full, __vcmpgtu4(__vsubus4(n, kWindows), low) != 0)) n = fit(vs, low);
            const bool begun = __any_sync(full, m0 > kLowest || m1 > kLowest);
            restart |= begun && (__vcmpgtu4(E0, n) | __vcmpgtu4(n, *E_set)) != 0;
            __syncwarp();
            if (restart || !begun) *E_set = n + kRise * 0x01010101u;
            if (n != E0) move_scale(n, n);
            const bool out = outside();
            fast &= ~__ballot_sync(full, out);
            if (out) vs = 0;
            edge |= restart || __any_sync(full, out);
          }
        }
        if (edge) step(i, slot, wk, wv, there, fast, vs, restart, std::true_type());
        else step(i, slot, wk, wv, full, full, wv, false, std::false_type());
        __syncwarp();                         // every lane has read the slot that the next copies fill, and the tables
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      {
        const volatile int* u = sched.unit;
        r = u[0];
        hg = u[1];
        j0 = u[2];
        at = u[3];
        A = u[4];
        nt = u[5];
        first = u[6];
        t0 = u[7];
        t1 = u[8];
        ntok = u[9];
        rows = ntok * a.G;
        h = hg * HG + my_head;
        begin = t0 * round;
        table = a.block_table + r * a.bt_stride_r;
      }
      // ---- results: l of a row over the lanes that share it; O as the sums of p v (of 2^7 p v in fp16) that the join takes
#pragma unroll
      for (int x = 4; x < 32; x *= 2) {
        l0 += __shfl_xor_sync(full, l0, x);
        l1 += __shfl_xor_sync(full, l1, x);
      }
      l0 *= 1.0f / kPScale<false>;
      l1 *= 1.0f / kPScale<false>;
      {
        // A row whose m is far from the maximum of its logits goes on with m + k and 2^-k of O and l, so that l is of the order of 1:
        // what the warps and CTAs have is added up in 32 bits.
        auto shift_of = [](float l) -> int {
          const int e = int(__float_as_uint(l) >> 23) - 127;
          return e > -127 && e < 128 && (e < -8 || e > 40) ? e : 0;
        };
        const int k0 = shift_of(l0), k1 = shift_of(l1);
        l0 = l0 * pow2(-k0 / 2) * pow2(-k0 - -k0 / 2);
        l1 = l1 * pow2(-k1 / 2) * pow2(-k1 - -k1 / 2);
        m0 += float(k0);
        m1 += float(k1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          constexpr int kBack = BF16 ? int(kPBits) : 0;
          const int e0 = byte_of(E0, g) - 127 - kBack - k0, e1 = byte_of(E1, g) - 127 - kBack - k1;
          const float y0 = pow2(e0 / 2), z0 = pow2(e0 - e0 / 2), y1 = pow2(e1 / 2), z1 = pow2(e1 - e1 / 2);
#pragma unroll
          for (int j = 2 * g; j < 2 * g + 2; ++j) {
            o[j][0] = o[j][0] * y0 * z0;
            o[j][1] = o[j][1] * y1 * z1;
            o[j][2] = o[j][2] * y0 * z0;
            o[j][3] = o[j][3] * y1 * z1;
          }
        }
      }
      const bool whole = t0 == 0 && t1 == nt;
      const int ps_slot = t0 > 0 ? 0 : 1;
      __syncthreads();                        // the rings are free, and every warp's NaN groups are known
      {                                       // the warps of a head, two at least, meet through shared memory, the first goes on
        float* jo = reinterpret_cast<float*>(smem) + warp * Rg::kJoin;
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
            const float4* po = reinterpret_cast<const float4*>(smem) + w * (Rg::kJoin / 4);
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
              o[j][1] = fmaf(o[j][1], p1, x.y * q1);
              o[j][2] = fmaf(o[j][2], p0, x.z * q0);
              o[j][3] = fmaf(o[j][3], p1, x.w * q1);
            }
          }
      }
      if (my_part == 0) {
        const int fix = *reinterpret_cast<volatile int*>(&sched.bad_v);
        // the head's NaN groups of token t; of the tokens that every row sees, each lane looking at every 32nd
        auto nan_groups = [&](int t) -> uint32_t {
          const int lb = block_of(t), ph = lb < a.MB ? table[lb] : -1;
          uint32_t nan = 0;
          if (ph >= 0 && ph < a.NB) {
            const uint8_t* p = reinterpret_cast<const uint8_t*>(
                bytes_at(a.kv_stride_kv + (int64_t(ph) * a.BS + (t - lb * a.BS)) * a.kv_stride_s)) + a.Hkv * (D / 2) + h * G;
#pragma unroll
            for (int g = 0; g < G; ++g) nan |= p[g] >= kNan4 ? 1u << g : 0u;
          }
          return nan;
        };
        uint32_t nan_all = 0;
        if (fix) {
#pragma unroll 1
          for (int t = begin + lane; t < min(all + 1, end); t += 32) nan_all |= nan_groups(t);
          nan_all = __reduce_or_sync(full, nan_all);
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = hf ? row1 : row0;
          if (row >= rows) continue;
          const float L = hf ? l1 : l0, M = hf ? m1 : m0, inv = over<BF16>(L);
          const int jq = row / a.G, hq = h * a.G + row - jq * a.G, hr = my_head * rows + row;
          const int64_t qt = int64_t(a.q_off[r]) + j0 + jq;
          uint16_t* dst = static_cast<uint16_t*>(a.out) + qt * a.out_stride_t + int64_t(hq) * a.out_stride_h;
          float* part = ps.out(cta, ps_slot) + int64_t(hr) * D;
          uint32_t nan = nan_all;             // ... and of those that this row sees beside
          if (fix) {
#pragma unroll 1
            for (int t = max(all + 1, begin); t <= min(all + jq, end - 1); ++t) nan |= nan_groups(t);
          }
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const int d0 = 32 * g + 4 * r8;
            float y[4] = {o[2 * g][hf], o[2 * g][2 + hf], o[2 * g + 1][hf], o[2 * g + 1][2 + hf]};
            if (nan >> g & 1u) y[0] = y[1] = y[2] = y[3] = __int_as_float(0x7fffffff);
            if (whole) {
              const uint32_t u0 = pack2<BF16>(y[0] * inv, y[1] * inv), u1 = pack2<BF16>(y[2] * inv, y[3] * inv);
              if (vec_out) {
                *reinterpret_cast<uint2*>(dst + d0) = make_uint2(u0, u1);
              } else {
                dst[d0] = uint16_t(u0);
                dst[d0 + 1] = uint16_t(u0 >> 16);
                dst[d0 + 2] = uint16_t(u1);
                dst[d0 + 3] = uint16_t(u1 >> 16);
              }
            } else {
              *reinterpret_cast<float4*>(part + d0) = make_float4(y[0], y[1], y[2], y[3]);
            }
          }
          if (r8 == 0) {
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
        ds.n_used = n_used();
        ds.ntok = ds.A = ntok;
        ds.S = all + ntok;
        ds.a0 = a.q_off[r] + j0;
        ds.end = low() + first + nt;
        ds.total = sched.share.total;
        ps.desc[cta] = ds;
      }
      __syncthreads();                        // the rings are written again
    }
  }
}

}  // namespace four
}  // namespace few
}  // namespace chunk

namespace {

template <int D, bool BF16>
cudaError_t launch_few4_t(const ChunkArgs& a, int grid, cudaStream_t st) {
  auto k = chunk::few::four::chunk_few4_kernel<D, BF16>;
  constexpr int bytes = int(chunk::few::four::Ring4<D>::kSmemBytes);
  static SmemLimit limit;
  const cudaError_t e = limit.set(reinterpret_cast<const void*>(k), bytes);
  if (e != cudaSuccess) return e;
  const bool vec_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride_t % 8 == 0 && a.out_stride_h % 8 == 0;
  k<<<grid, chunk::few::four::kThreads, bytes, st>>>(a, vec_out);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk_few4(const ChunkArgs& a, int dtype, int grid, cudaStream_t st) {
  const bool bf = dtype == ACTKV_BF16;
  if (a.D == 128) return bf ? launch_few4_t<128, true>(a, grid, st) : launch_few4_t<128, false>(a, grid, st);
  return bf ? launch_few4_t<64, true>(a, grid, st) : launch_few4_t<64, false>(a, grid, st);
}

}  // namespace actkv
