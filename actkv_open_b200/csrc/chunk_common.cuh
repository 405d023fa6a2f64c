// What the two tensor-core kernels of chunk attention share (chunk_umma.cu, chunk_few.cu): the shares of
// work, the partial results that a cut unit leaves, and 16-bit values from 8-bit rows.
#pragma once

#include "common.cuh"
#include "kernels.cuh"
#include "quant_row.cuh"
#include "umma_common.cuh"

namespace actkv {
namespace chunk {

using namespace umma;

constexpr int kRows = 128;                  // query rows per row tile (MMA M)
constexpr int kTile = 128;                  // tokens per key tile, the grain of the schedule
constexpr int kFewRows = 16;                // query rows of a session and KV head that chunk_few_kernel takes
constexpr int few_limit(bool quant) { return quant ? 8 : kFewRows; }      // ... of which over the 8-bit cache
constexpr int kFewParts = 8 * kFewRows;     // rows of its units: up to 8 heads
// (6 sessions of 2000 to 10000 tokens with 1088 new: 749 us with a cost of 2, 713 with 4, 708 with 6; prompts and
// single tokens of head size 64: 157, 153, 157)
constexpr int kUnitCost = 4;                // a unit's fixed cost (queries in, results out) in key tiles
constexpr float kSlack = 8.0f;              // log2 units the maximum may outgrow m by
// p is multiplied by this, exactly, before it is rounded to 16 bits, and O / l divided by it: p is at most 2^8, and fp16
// then holds what is 2^-32 of the maximum's (of 2^-24 at least, it lost the tail of a dominant token: thousands of
// others of 2^-25 each).  bf16 has the range of 32 bits.
template <bool BF16> constexpr float kPScale = BF16 ? 1.0f : 128.0f;
constexpr int kMaxD = 128;

// ------------------------------------------------------------------------------------ shares of work
struct Share {
  int64_t total, pre;        // all weight, weight before session r0
  int r0;                    // the session that holds the CTA's first unit of weight
};

// New tokens of session r; 0, and flagged, when its offsets leave the call's T rows (negative, or past the end), so
// that no row outside q, out and lse is touched.
__device__ __forceinline__ int new_tokens(const ChunkArgs& a, int r) {
  const int a0 = a.q_off[r], a1 = a.q_off[r + 1];
  if (a1 <= a0) return 0;
  if (a0 >= 0 && a1 <= a.T) return a1 - a0;
  flag(a.status, ACTKV_DEV_BAD_INDEX);
  return 0;
}

// Tokens that a table has a place for (short of where 32-bit token arithmetic would end): what the kernels walk of a
// session.  A longer one is flagged, and the rest of it hidden like any token of a block outside the cache.
__device__ __forceinline__ int table_room(const ChunkArgs& a) { return int(min(int64_t(a.MB) * a.BS, int64_t(0x7fffff00))); }
__device__ __forceinline__ int held_tokens(const ChunkArgs& a, int S) { return min(max(S, 0), table_room(a)); }
__device__ __forceinline__ void flag_long(const ChunkArgs& a, int S) {
  if (S > table_room(a)) flag(a.status, ACTKV_DEV_BAD_INDEX);
}

// Query rows per KV head up to which chunk_few_kernel takes a session in this call, 0 when chunk_umma_kernel takes
// all.  The two kernels run one after the other, so short work is not split between them: where the other kernel
// has sessions too, those of few rows go to their own only when they hold bytes enough to win back a
// kernel's start and end (about 15 us) by its higher rate: 512 MB of 16-bit rows, 64 MB of 8-bit ones.  Single tokens
// over 8192 (32 query heads over 8 of 128) beside one chunk, together and split, us:
//                                   16-bit rows: 128 MB   256 MB    512 MB    1 GB      8-bit rows: 32 MB    64 MB     128 MB
//   beside 512 new over 8192               139, 142  171, 160  226, 203  347, 283              142, 141  162, 149  198, 161
//   beside 64 new over 2048                 79, 101  110, 122  158, 169  272, 246               61, 89    83, 94   123, 110
// The more the chunk has to do the sooner splitting pays; the limits lie between the two.  (16 sessions of 1000 to 9000
// tokens with 3 to 7 new ones each, 4 query heads per KV head, 330 MB: 120 us split, 82 us together.)
// Every thread of the block calls it; `sums` is shared.
template <int kThreads>
__device__ __forceinline__ int few_rows_now(const ChunkArgs& a, int64_t (&sums)[2]) {
  if (a.few_rows == 0 || int64_t(a.T) * a.G <= a.few_rows) return a.few_rows;      // none, or all of them
  if (threadIdx.x < 2) sums[threadIdx.x] = 0;
  __syncthreads();
  int64_t few = 0, all = 0;
  for (int r = threadIdx.x; r < a.R; r += kThreads) {
    const int A = new_tokens(a, r);
    if (A == 0) continue;
    const int s = max(a.seq_used[r], 1);
    all += s;
    if (A * a.G <= a.few_rows) few += s;
  }
  few = warp_sum(few);
  all = warp_sum(all);
  if ((threadIdx.x & 31) == 0 && all > 0) {
    atomicAdd(reinterpret_cast<unsigned long long*>(&sums[0]), static_cast<unsigned long long>(few));
    atomicAdd(reinterpret_cast<unsigned long long*>(&sums[1]), static_cast<unsigned long long>(all));
  }
  __syncthreads();
  const int64_t bytes = sums[0] * a.Hkv * a.D * 2 * (a.quant ? 1 : 2);
  return sums[0] == sums[1] || bytes >= (int64_t(a.quant ? 64 : 512) << 20) ? a.few_rows : 0;
}

// CTAs that get work when a share is at least `least`.
__device__ __forceinline__ int used_ctas(int64_t total, int n, int least) {
  return int(max(int64_t(1), min(int64_t(n), total / least)));
}

// CTA `cta` of the n used takes the weight [total * cta / n, total * (cta + 1) / n), sessions in order.
// Every thread of the block calls it; `s` starts as {0, 0, R}.
template <int kThreads, typename Weight>
__device__ __forceinline__ void share_out(int R, Weight weight, Share& s, int64_t* scan, int cta, int n,
                                          int least) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // pass 0 adds the weights up, pass 1 finds the session (only when a pass over all does not fit)
  int64_t lo = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int64_t carry = 0;
#pragma unroll 1
    for (int base = 0; base < R; base += kThreads) {
      const int r = base + int(threadIdx.x);
      const int64_t w = r < R ? weight(r) : 0;
      int64_t incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      int64_t before = carry, all = carry;
      for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) before += scan[i];
        all += scan[i];
      }
      __syncthreads();
      if (pass == 0 && base + kThreads >= R) {              // the last step: the total is known
        if (threadIdx.x == 0) s.total = all;
        lo = all * cta / used_ctas(all, n, least);
      }
      const int64_t excl = before + incl - w;
      if ((pass == 1 || R <= kThreads) && w > 0 && lo >= excl && lo < excl + w) {
        s.r0 = r;
        s.pre = excl;
      }
      carry = all;
    }
    if (R <= kThreads) break;
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------ partial results
struct Desc {                // the unit that a CTA began and left to the next ones
  int32_t valid, r, h, j0, ntok, S, A, a0;
  int64_t end, total;
  int32_t two, heads;        // two row tiles; KV heads from h on
  int32_t n_used, pad;       // CTAs that the work was shared out to
};
static_assert(sizeof(Desc) == 64, "the partial results after the descriptors are 16-byte aligned");


// The workspace of one kernel: a descriptor per CTA, then two partial results per CTA (slot 0: of a unit begun
// by an earlier CTA, 1: of one left to the next), each `rows` rows of D values and (m, l) per row.
struct Parts {
  Desc* desc;
  float* base;
  int rows;
  __device__ __forceinline__ float* out(int cta, int slot) const {
    return base + (int64_t(cta) * 2 + slot) * rows * (kMaxD + 2);
  }
  __device__ __forceinline__ float* ml(int cta, int slot, int D) const { return out(cta, slot) + int64_t(rows) * D; }
};
__host__ __device__ inline size_t parts_bytes(int n_cta, int rows) {
  return size_t(n_cta) * (sizeof(Desc) + size_t(2) * rows * (kMaxD + 2) * sizeof(float));
}
__host__ __device__ inline size_t few_offset(int n_cta) { return (parts_bytes(n_cta, 2 * kRows) + 255) & ~size_t(255); }
__device__ __forceinline__ Parts parts_at(void* ws, size_t off, int n_cta, int rows) {
  char* p = static_cast<char*>(ws) + off;
  return Parts{reinterpret_cast<Desc*>(p), reinterpret_cast<float*>(p + int64_t(n_cta) * sizeof(Desc)), rows};
}
__device__ __forceinline__ Parts wide_parts(void* ws, int n_cta) { return parts_at(ws, 0, n_cta, 2 * kRows); }
__device__ __forceinline__ Parts few_parts(void* ws, int n_cta) { return parts_at(ws, few_offset(n_cta), n_cta, kFewParts); }

// ------------------------------------------------------------------------------------ 16-bit values
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two probabilities.
template <bool BF16>
__device__ __forceinline__ uint32_t pack_p(float lo, float hi) {
  if constexpr (BF16) return pack2<true>(lo, hi);
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(lo), "+f"(hi)
      : "f"(kPScale<BF16>));
  return pack2<BF16>(lo, hi);
}
// What O is multiplied by for the output, from l.
template <bool BF16>
__device__ __forceinline__ float over(float l) { return l == 0.0f ? 0.0f : 1.0f / (l * kPScale<BF16>); }

// 16 e4m3 values with scale byte b as 16-bit values.  The four exponent and three mantissa bits of a
// byte, moved under the wider type's exponent, read as the value times 2^-120 (bf16) or 2^-8 (fp16),
// subnormals included, so one multiplication by a power of two, 2^(b - 127) with that put right, gives
// the value exactly; a power of two outside the type takes a second one.  fp16 values past its range
// become its largest.
template <bool BF16>
__device__ __forceinline__ uint32_t mul16x2(uint32_t x, uint32_t f) {
  uint32_t r;
  if constexpr (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(f));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(f));
  return r;
}
// Whether one multiplication does for every byte of a word of scale bytes.
template <bool BF16>
__device__ __forceinline__ bool plain_scales(uint32_t w) {
  return __vcmpgtu4(w, 0x86868686u) == 0 && (BF16 || __vcmpgtu4(0x69696969u, w) == 0);   // <= 134 (fp16: >= 105)
}
// Those bits of two values: x has their bytes atop its halves and zeros below, m has them without their signs at the
// bottom of its halves.  With s the sign and v the rest, x is 2^15 s + 2^8 v and the result 2^15 s + 2^4 v (bf16;
// 2^7 v for fp16): a multiplication and addition, off the logic pipe, which is the busiest here.
template <bool BF16>
__device__ __forceinline__ uint32_t under_exponent(uint32_t x, uint32_t m) {
  return x - m * (BF16 ? 0xf0u : 0x80u);
}
// e4m3's NaN (all seven bits below the sign set) reads as 480 under these: who widens finds such bytes in the words as
// they come and leaves the fast way.  Adding 1 to each byte flips its sign bit for them and, when there is none to
// carry out of a byte, for no other.  It costs the few-row kernel 4 to 5 per cent (32 single tokens over 18432: 278 to
// 291 us; the largest of three 16-bit halves at a time instead: 288 with spills, and 8 per cent at head size 64) and
// the wide one 2.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t seen, uint32_t w) { return seen | ((w + 0x01010101u) ^ w); }
__device__ __forceinline__ bool any_nan_byte(uint32_t seen) { return (seen & 0x80808080u) != 0; }
// ... and the slow way puts NaN where m, two bytes without their signs at the bottom of its halves, has one.
__device__ __forceinline__ uint32_t put_nan(uint32_t r, uint32_t m) { return r | (__vcmpeq2(m, 0x007f007fu) & 0x7fff7fffu); }
template <bool BF16>
__device__ __forceinline__ void widen16(const uint4& raw, uint32_t f, uint32_t (&r)[8], uint32_t& seen) {
  const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
  // nan_bytes of the words without their signs, which are needed anyway (4 chunks of 512 over 10240: 418 us, 426 so)
  seen |= ((in[0] & 0x7f7f7f7fu) + 0x01010101u) | ((in[1] & 0x7f7f7f7fu) + 0x01010101u);
  seen |= ((in[2] & 0x7f7f7f7fu) + 0x01010101u) | ((in[3] & 0x7f7f7f7fu) + 0x01010101u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t x = __byte_perm(in[i >> 1], 0u, (i & 1) ? 0x3424 : 0x1404);
    const uint32_t m = __byte_perm(in[i >> 1] & 0x7f7f7f7fu, 0u, (i & 1) ? 0x4342 : 0x4140);
    r[i] = mul16x2<BF16>(under_exponent<BF16>(x, m), f);
  }
}
// The multiplier of scale byte b, in both halves, where plain_scales holds.
template <bool BF16>
__device__ __forceinline__ uint32_t plain_factor(uint32_t b) {
  return BF16 ? b * 0x00800080u + 0x3c003c00u : (b - 104u) * 0x04000400u;
}
// For any scale byte: multipliers whose product is the power of two, each a value of the type, in an order in which
// only the last one that is not 1 rounds.  fp16: 2^(b - 119) is 2^-7, exact for what comes first, and the rest, down to
// its subnormals (0 below: such values round to 0); or up to three factors of at most 2^15, past which everything but 0
// is past the range.
template <bool BF16>
__device__ __forceinline__ void any_factors(uint32_t b, uint32_t (&f)[3]) {
  const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
  f[1] = f[2] = one;
  if constexpr (BF16) {
    const int e = int(b) + 120, e1 = min(e, 254);
    f[0] = e1 * 0x00800080u;
    f[1] = (e - e1 + 127) * 0x00800080u;
  } else if (b < 105u) {
    f[0] = 0x20002000u;                        // 2^-7
    f[1] = (b >= 98u ? b - 97u << 10 : (b >= 88u ? 1u << b - 88u : 0u)) * 0x00010001u;
  } else {
    const uint32_t e = min(b, 164u) - 104u;    // the exponent field of one factor, 30 of which it can hold
    const uint32_t e1 = min(e, 30u), e2 = min(e - e1, 15u), e3 = e - e1 - e2;
    f[0] = e1 * 0x04000400u;
    f[1] = (e2 + 15u) * 0x04000400u;
    f[2] = (e3 + 15u) * 0x04000400u;
  }
  if (b == 255u) f[0] = 0x7fff7fffu;           // NaN
}
// x, already under the exponent and times the first factor, times the others; past fp16's range: its largest.
template <bool BF16>
__device__ __forceinline__ uint32_t mul_rest(uint32_t x, uint32_t f1, uint32_t f2) {
  x = mul16x2<BF16>(x, f1);
  if constexpr (!BF16) {
    x = mul16x2<BF16>(x, f2);
    asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7bff7bffu));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xfbfffbffu));
  }
  return x;
}
// What is not finite among two 16-bit values, in the halves `hide` (0xffff per half), becomes 0.
template <bool BF16>
__device__ __forceinline__ uint32_t drop_bad(uint32_t u, uint32_t hide, bool& found) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  uint32_t bad = ((u & kExp) == kExp ? 0xffffu : 0u) | (((u >> 16) & kExp) == kExp ? 0xffff0000u : 0u);
  bad &= hide;
  found |= bad != 0;
  return u & ~bad;
}
// Value e of an 8-bit row, inf and NaN as in the 16-bit type (whose finite values it may exceed in digits).
template <bool BF16>
__device__ __forceinline__ float quant_value(const uint8_t* row, int Hkv, int D, int e) {
  const float x = e4m3x2_f32(row[e]).x * scale_of(row[Hkv * D + e / kQuantGroup]);
  return BF16 || x != x ? x : fminf(fmaxf(x, -65504.0f), 65504.0f);
}

}  // namespace chunk
}  // namespace actkv
