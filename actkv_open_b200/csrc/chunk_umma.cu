// Chunk attention over the paged cache on the sm_100a tensor cores (tcgen05 + TMA + TMEM): the newest
// A of a session's S tokens are the queries, query j sees tokens t <= S - A + j, and the call gives
// out = softmax(scale q.k) v and lse = log sum exp(scale q.k) of every (query, head) row.
//
// With c = scale * log2 e and a reference exponent m per row, p_t = 2^(c q.k_t - m), l = sum p_t,
// O = sum p_t v_t, out = O / l, lse = (m + log2 l) ln 2.  m need not be the running maximum, only
// near it: it is raised (and O and l rescaled) when the maximum has grown by more than 2^8, so p
// stays below 2^8 and the rescaling, a pass over O, is rare.  S = Q K^T and O are accumulated in 32
// bits in TMEM, m and l are 32-bit registers; p is rounded to the cache's 16-bit type for the second
// product only (l sums the unrounded values), the same half unit that the output is rounded by.
//
// Work.  A unit is (session, KV head, group of up to 256 query rows): rows are (token, head of the
// GQA group), two tiles of 128.  The units' key tiles of 128 tokens, laid end to end with a fixed
// cost per unit, are cut into one equal share per CTA (one CTA per SM), so ragged batches, one long
// session and many short ones balance alike; a unit that a cut divides leaves 32-bit partial
// results (m, l, O) in the workspace, at most two per CTA, which chunk_combine_kernel joins in a
// fixed order.
//
// Two streams of (S, p, O) run in a CTA, each with its own softmax warpgroup and 256 TMEM columns:
//   two row tiles   both streams take every key tile (one copy of K and V serves 256 rows)
//   one row tile    (few new tokens) stream w takes every second key tile with the same queries,
//                   and the first warpgroup joins the two at the end
// While one stream's softmax runs, the tensor core works on the other's products.
//
// Warp roles (384 threads): warp 0 TMA (a paged block per lane and tile: one 5-D box of 8-token
// groups x both D-halves; 4 KB boxes, since the copy engine spends ~60 cycles per box whatever its
// size), warp 1 MMA issue (p from TMEM as the A operand, V as an MN-major B operand straight from
// the tile), warps 4-7 and 8-11 softmax (a thread per row).  Every wait is bounded
// (umma_common.cuh).
#include <cuda.h>

#include "common.cuh"
#include "kernels.cuh"
#include "umma_common.cuh"

namespace actkv {
namespace chunk {

using namespace umma;

constexpr int kMaxThreads = 512;
constexpr int threads(bool quant) { return quant ? 512 : 384; }
constexpr int kUnitSlots = 4;               // units announced ahead of their results
constexpr int kRows = 128;                  // query rows per tile (MMA M)
constexpr int kTile = 128;                  // tokens per key tile
constexpr int kUnitCost = 2;                // a unit's fixed cost (queries in, results out) in key tiles
constexpr float kSlack = 8.0f;              // log2 units the maximum may outgrow m by
constexpr int kMaxD = 128;

constexpr uint32_t kSchedBytes = 512;

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kTileBytes = kTile * D * 2;      // a K, V or Q tile
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr uint32_t kGroupBytes = kHalves * 1024;    // 8 tokens of a K / V tile
  static constexpr uint32_t kKvOff = 2 * kTileBytes;
  static constexpr uint32_t kMlOff = kKvOff + kSlots * kTileBytes;       // stream 1's (m, l) per row
  static constexpr uint32_t kBarOff = kMlOff + kRows * 8;
  // kv_full[slots] kv_empty[slots] q_full q_empty s_full[2] p_full[2][2] o_full[2] o_empty[2]
  // x_full unit_full[4] unit_empty[4]
  static constexpr int kNumBars = 2 * kSlots + 13 + 2 * kUnitSlots;
  static constexpr uint32_t kSchedOff = kBarOff + kNumBars * 8;
  static constexpr uint32_t kSmemBytes = kSchedOff + kSchedBytes;
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
};

// TMEM columns: S (and p over it) of stream w at 128 w, O of stream w at 256 + 128 w.
constexpr uint32_t kSCol = 0, kOCol = 256;

// ------------------------------------------------------------------------------------ the schedule
struct Unit {
  int r, h, j0, ntok;        // session, KV head, first query token of the group, tokens in it
  int S, A, a0;
  int nt, t0, t1;            // key tiles of the unit, and this CTA's part of them
  int two;                   // two row tiles
  int64_t end;               // the unit's end in the schedule
};

struct Desc {                // the unit that a CTA began and left to the next ones
  int32_t valid, r, h, j0, ntok, S, A, a0;
  int64_t end, total;
  int32_t two, pad[3];
};
static_assert(sizeof(Desc) == 64, "the partial results after the descriptors are 16-byte aligned");

struct Sched {               // in shared memory
  int64_t total, pre;        // all weight, weight before session r0
  int r0;
  uint32_t tmem;
  int abort_flag;
  int bad_v;                 // a value that some row of the unit does not see is not finite
  int64_t scan[kMaxThreads / 32];
  Unit units[kUnitSlots];    // from the TMA warp, which alone walks the schedule; r < 0 ends it
};
static_assert(sizeof(Sched) <= kSchedBytes, "the schedule's place in shared memory");

struct Geometry {
  int tpb;                   // tokens per row tile
  __device__ explicit Geometry(const ChunkArgs& a) : tpb(kRows / a.G) {}
  __device__ int groups(int A) const { return (A + 2 * tpb - 1) / (2 * tpb); }
  // key tiles that some query of tokens [j0, j0 + n) sees
  __device__ int tiles(int S, int A, int j_end) const {
    const int last = S - A + j_end - 1;
    return last >= 0 ? last / kTile + 1 : 0;
  }
  __device__ int64_t head_weight(int S, int A) const {
    int64_t w = 0;
    for (int j = 0; j < A; j += 2 * tpb) w += kUnitCost + tiles(S, A, min(A, j + 2 * tpb));
    return w;
  }
};

// Walks the units that overlap this CTA's share [lo, hi) of the schedule: sessions in order, KV heads,
// then row groups.  Every thread walks the same sequence.
struct Walker {
  const ChunkArgs* a;
  Geometry geo;
  int64_t lo, hi, at;
  int r, h, j, S, A, a0;

  __device__ void load() {
    while (r < a->R) {
      a0 = a->q_off[r];
      A = a->q_off[r + 1] - a0;
      S = a->seq_used[r];
      if (A > 0) return;
      ++r;
    }
  }
  __device__ Walker(const ChunkArgs* args, const Sched& s, int cta, int n) : a(args), geo(*args) {
    lo = s.total * cta / n;
    hi = s.total * (cta + 1) / n;
    r = s.r0;
    h = j = S = A = a0 = 0;
    at = s.pre;
    if (lo >= hi) {
      at = hi;
      return;
    }
    load();
    const int64_t w = geo.head_weight(S, A);
    h = int((lo - at) / w);
    at += h * w;
    while (true) {                            // the group that holds lo
      const int64_t x = kUnitCost + geo.tiles(S, A, min(A, j + 2 * geo.tpb));
      if (lo < at + x) break;
      at += x;
      j += 2 * geo.tpb;
    }
  }
  __device__ bool next(Unit& x) {
    while (at < hi && r < a->R) {
      x.r = r;
      x.h = h;
      x.j0 = j;
      x.ntok = min(2 * geo.tpb, A - j);
      x.S = S;
      x.A = A;
      x.a0 = a0;
      x.nt = geo.tiles(S, A, j + x.ntok);
      x.two = x.ntok > geo.tpb;
      const int64_t start = at, first = at + kUnitCost;
      at = x.end = first + x.nt;
      j += 2 * geo.tpb;
      if (j >= A) {
        j = 0;
        if (++h == a->Hkv) {
          h = 0;
          ++r;
          load();
        }
      }
      x.t0 = int(lo > first ? lo - first : 0);
      x.t1 = x.nt == 0 ? 0 : int(min(int64_t(x.nt), hi - first));
      if (x.nt == 0 ? start >= lo : x.t0 < x.t1) return true;
    }
    return false;
  }
};

// Total weight, and the session that holds this CTA's first unit of weight.
template <int kThreads>
__device__ void make_schedule(const ChunkArgs& a, Sched& s, int cta, int n) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Geometry geo(a);
  // pass 0 adds the weights up, pass 1 finds the session (only when a pass over all does not fit)
  int64_t lo = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t carry = 0;
    for (int base = 0; base < a.R; base += kThreads) {
      const int r = base + int(threadIdx.x);
      int64_t w = 0;
      if (r < a.R) {
        const int A = a.q_off[r + 1] - a.q_off[r];
        if (A > 0) w = a.Hkv * geo.head_weight(a.seq_used[r], A);
      }
      int64_t incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) s.scan[warp] = incl;
      __syncthreads();
      int64_t before = carry, all = carry;
      for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) before += s.scan[i];
        all += s.scan[i];
      }
      __syncthreads();
      if (pass == 0 && base + kThreads >= a.R) {            // the last step: the total is known
        if (threadIdx.x == 0) s.total = all;
        lo = all * cta / n;
      }
      const int64_t excl = before + incl - w;
      if ((pass == 1 || a.R <= kThreads) && w > 0 && lo >= excl && lo < excl + w) {
        s.r0 = r;
        s.pre = excl;
      }
      carry = all;
    }
    if (a.R <= kThreads) break;
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------ operands
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = uint64_t((addr >> 4) & 0x3FFFu);
  d |= uint64_t(lbo >> 4) << 16;
  d |= uint64_t(sbo >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;                     // 128-byte swizzle
  return d;
}

__device__ __forceinline__ void mma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]),
      "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]),
      "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]),
      "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]),
      "r"(u[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
        "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]),
      "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]),
      "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(taddr)
      : "memory");
}
// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A slot of the K / V ring and the parity of its current use.
struct Ring {
  uint32_t slot = 0, par = 0;
  __device__ __forceinline__ void next(uint32_t n) {
    const bool wrap = slot + 1 == n;
    slot = wrap ? 0 : slot + 1;
    par ^= uint32_t(wrap);
  }
};

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// Ring position, within a unit of nt key tiles of which `lead` keys go ahead of the values, of the
// values of tile t: keys 0 .. lead - 1, then values t and keys t + lead in turn.
__device__ __forceinline__ int v_position(int t, int nt, int lead) {
  return min(lead, nt) + t + min(t, max(0, nt - lead));
}

// Part `slot` (0: a unit begun by an earlier CTA, 1: one left to the next) of CTA `cta`'s partial
// results: rows of D values, then (m, l) per row.
constexpr int64_t kPartFloats = int64_t(2 * kRows) * (kMaxD + 2);
__device__ __forceinline__ float* part_of(void* ws, int n_cta, int cta, int slot) {
  return reinterpret_cast<float*>(static_cast<char*>(ws) + int64_t(n_cta) * sizeof(Desc)) +
         (int64_t(cta) * 2 + slot) * kPartFloats;
}

template <int D, bool BF16>
__device__ __forceinline__ void store_row(uint16_t* dst, const float (&o)[32], float inv, bool vec) {
  uint32_t u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) u[i] = pack2<BF16>(o[2 * i] * inv, o[2 * i + 1] * inv);
  if (vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint4*>(dst)[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dst[2 * i] = uint16_t(u[i]);
      dst[2 * i + 1] = uint16_t(u[i] >> 16);
    }
  }
}

// 16 e4m3 values with scale byte b as 16-bit values.  The four exponent and three mantissa bits of a
// byte, moved under the wider type's exponent, read as the value times 2^-120 (bf16) or 2^-8 (fp16),
// subnormals included, so one multiplication by a power of two, 2^(b - 127) with that put right, gives
// the value exactly; a power of two outside the type takes a second one.  fp16 values past its range
// become its largest.
template <bool BF16>
__device__ __forceinline__ void widen16(const uint4& raw, uint32_t b, uint4 (&out)[2]) {
  const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t r[8];
  // bits of the multiplier in both halves
  const int e = BF16 ? int(b) + 120 : int(b) - 104;
  const int top = BF16 ? 254 : 30;
  const int e1 = min(max(e, 1), top);
  uint32_t f1 = uint32_t(e1) << (BF16 ? 7 : 10);
  if (b == 255u) f1 = 0x7fffu;               // NaN
  f1 |= f1 << 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t x = __byte_perm(in[i >> 1], 0u, (i & 1) ? 0x3424 : 0x1404);   // two bytes, each atop a half
    const uint32_t y = ((x >> (BF16 ? 4 : 1)) & (BF16 ? 0x07f007f0u : 0x3f803f80u)) | (x & 0x80008000u);
    if constexpr (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(y), "r"(f1));
    else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(y), "r"(f1));
  }
  if (e != e1 && b != 255u) {
    const int e2 = min(max(e - e1 + (BF16 ? 127 : 15), 1), top);
    uint32_t f2 = uint32_t(e2) << (BF16 ? 7 : 10);
    f2 |= f2 << 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (BF16) {
        asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(f2));
      } else {
        asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(f2));
      }
    }
  }
  if (!BF16 && b >= 134u && b != 255u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      asm("min.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(0x7bff7bffu));
      asm("max.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(0xfbfffbffu));
    }
  }
  out[0] = make_uint4(r[0], r[1], r[2], r[3]);
  out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// One token's values of a tile in shared memory: zeroed when the token is past the session's end; when
// `hidden` (some row does not see it), what is not finite is zeroed and *bad_v set.
template <int D, bool BF16>
__device__ __forceinline__ void clean_values(uint8_t* tile, bool past, bool hidden, volatile int* bad_v) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  if (!past && !hidden) return;
#pragma unroll
  for (int k = 0; k < D / 8; ++k) {
    uint4* p = reinterpret_cast<uint4*>(tile + (k >> 3) * 1024) + (k & 7);
    if (past) {
      *p = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    uint32_t u[4] = {p->x, p->y, p->z, p->w};
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((u[e] & kExp) == kExp) {
        u[e] &= 0xffff0000u;
        bad = true;
      }
      if (((u[e] >> 16) & kExp) == kExp) {
        u[e] &= 0xffffu;
        bad = true;
      }
    }
    if (bad) {
      *p = make_uint4(u[0], u[1], u[2], u[3]);
      *bad_v = 1;
    }
  }
}

// ------------------------------------------------------------------------------------ the kernel
template <int D, bool BF16, bool QUANT>
__global__ void __launch_bounds__(threads(QUANT), 1)
    chunk_umma_kernel(const __grid_constant__ CUtensorMap tmap_kv, const __grid_constant__ CUtensorMap tmap_q,
                      const __grid_constant__ ChunkArgs a, bool vec_out) {
  using Ly = Layout<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Ly::kBarOff);
  Sched& sched = *reinterpret_cast<Sched*>(smem + Ly::kSchedOff);
  volatile int* abort_flag = &sched.abort_flag;
  volatile int* bad_v = &sched.bad_v;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int kSlots = Ly::kSlots;
  constexpr int B_KVF = 0, B_KVE = kSlots, B_QF = 2 * kSlots, B_QE = B_QF + 1, B_SF = B_QE + 1, B_PF = B_SF + 2,
                B_OF = B_PF + 4, B_OE = B_OF + 2, B_XF = B_OE + 2, B_UF = B_XF + 1,
                B_UE = B_UF + kUnitSlots;
  const unsigned full = 0xffffffffu;
  const int cta = blockIdx.x, n_cta = gridDim.x;

  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) flag(a.status, ACTKV_DEV_MISALIGNED);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(bar(B_KVF + i), QUANT ? 4 : 1);
      mbar_init(bar(B_KVE + i), 1);
    }
    mbar_init(bar(B_QF), 1);
    mbar_init(bar(B_QE), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(B_SF + i), 1);
      mbar_init(bar(B_PF + 2 * i), 4);
      mbar_init(bar(B_PF + 2 * i + 1), 4);
      mbar_init(bar(B_OF + i), 1);
      mbar_init(bar(B_OE + i), 4);
    }
    mbar_init(bar(B_XF), 4);
    for (int i = 0; i < kUnitSlots; ++i) {
      mbar_init(bar(B_UF + i), 1);
      mbar_init(bar(B_UE + i), QUANT ? 13 : 9);   // the MMA warp, the softmax warps, the converting warps
    }
    sched.total = sched.pre = 0;
    sched.r0 = a.R;
    sched.abort_flag = 0;
    sched.bad_v = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    Desc* dsc = static_cast<Desc*>(a.workspace) + cta;
    dsc->valid = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sched.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  __syncthreads();
  make_schedule<threads(QUANT)>(a, sched, cta, n_cta);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sched.tmem;
  const int tpb = kRows / a.G;

  // 384 threads of 168 registers: the softmax warps take 208 each, the others keep 88.  With the
  // converting warps 512 threads of 128: 160, 64, and 128 for those.
  if (warp < 4) {
  if constexpr (QUANT) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (whole warp)
    if (lane == 0) {
      if constexpr (!QUANT) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_kv)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_q)) : "memory");
    }
    const int bs_box = min(a.BS, kTile);         // token rows of a box
    const int bpt = kTile / bs_box;              // boxes per tile (<= 16: one per lane)
    const uint32_t box_bytes = uint32_t(bs_box) * D * 2;
    Walker wk(&a, sched, cta, n_cta);
    Unit x;
    uint32_t ring = 0, q_uses = 0;
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
      const bool any = wk.next(x);
      ok = __all_sync(full, mbar_wait(bar(B_UE + n % kUnitSlots), ((n / kUnitSlots) & 1u) ^ 1u, abort_flag, a.status));
      if (!ok) break;
      if (lane == 0) {
        if (!any) x.r = -1;
        sched.units[n % kUnitSlots] = x;
        mbar_arrive(bar(B_UF + n % kUnitSlots));
      }
      if (!any) break;
      if (x.t0 >= x.t1) continue;
      const int lead = x.two ? 1 : 2, nt = x.t1 - x.t0;
      // first token slot, in units of 8, of lane b's box of key tile t; -2 past the session's end
      auto read_id = [&](int t) -> int {
        const int tok = t * kTile + lane * bs_box;
        if (lane >= bpt || t >= x.t1 || tok >= x.S) return -2;
        const int lb = tok / a.BS;
        const int phys = lb < a.MB ? a.block_table[x.r * a.bt_stride_r + lb] : -1;
        if (phys < 0 || phys >= a.NB) {
          flag(a.status, ACTKV_DEV_BAD_INDEX);
          return 0;
        }
        return int((int64_t(phys) * a.BS + (tok - lb * a.BS)) >> 3);
      };
      int id0 = -2, id1 = -2, id2 = -2;
      if constexpr (!QUANT) {
        id0 = read_id(x.t0);
        id1 = read_id(x.t0 + 1);
        id2 = read_id(x.t0 + 2);
      }
      ok = __all_sync(full, mbar_wait(bar(B_QE), (q_uses & 1u) ^ 1u, abort_flag, a.status));
      if (!ok) break;
      if (lane == 0) {
        const int blocks = x.two ? 2 : 1;
        mbar_expect_tx(bar(B_QF), uint32_t(blocks) * tpb * a.G * D * 2);
        for (int b = 0; b < blocks; ++b)
          for (int hf = 0; hf < Ly::kHalves; ++hf)
            tma_load_3d(base + b * Ly::kTileBytes + hf * (kRows * 128), &tmap_q, bar(B_QF), hf * 64, x.h * a.G,
                        x.a0 + x.j0 + b * tpb);
      }
      ++q_uses;
      if constexpr (QUANT) continue;             // keys and values come through the converting warps
      auto load = [&](int t, int id, int plane) -> bool {
        const int slot = ring % kSlots;
        const bool w2 = mbar_wait(bar(B_KVE + slot), ((ring / kSlots) & 1u) ^ 1u, abort_flag, a.status);
        if (!__all_sync(full, w2)) return false;
        const int n = __popc(__ballot_sync(full, id >= 0));
        if (lane == 0) mbar_expect_tx(bar(B_KVF + slot), uint32_t(n) * box_bytes);
        __syncwarp();
        if (id >= 0)
          tma_load_5d(base + Ly::kKvOff + slot * Ly::kTileBytes + lane * box_bytes, &tmap_kv, bar(B_KVF + slot), 0, 0,
                      x.h * Ly::kHalves, id, plane);
        ++ring;
        return true;
      };
      ok = load(x.t0, id0, 0);
      if (ok && lead == 2 && nt > 1) ok = load(x.t0 + 1, id1, 0);
      for (int t = 0; ok && t < nt; ++t) {
        const int id3 = read_id(x.t0 + t + 3);
        ok = load(x.t0 + t, id0, 1);
        if (ok && t + lead < nt) ok = load(x.t0 + t + lead, lead == 1 ? id1 : id2, 0);
        id0 = id1;
        id1 = id2;
        id2 = id3;
      }
      if (!ok) break;
    }
    if (*abort_flag && lane == 0) {
      for (uint32_t s = 0; s < kSlots; ++s) {
        const uint32_t uses = ring / kSlots + (s < ring % kSlots ? 1u : 0u);
        if (uses) mbar_drain(bar(B_KVF + s), (uses - 1) & 1u);
      }
      if (q_uses) mbar_drain(bar(B_QF), (q_uses - 1) & 1u);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp walks the loop, so that the operand descriptors are warp-uniform values, and one
    // elected lane issues: with a lone thread the descriptors went through vector registers and an MMA
    // took ~90 cycles to issue, more than the 64 it runs.
    const uint32_t idesc_s = instr_desc_mn(kRows, kTile, BF16);
    const uint32_t idesc_o = instr_desc_mn(kRows, D, BF16) | (1u << 16);       // B (V) MN-major
    const uint64_t q_desc = desc(base, 16, 1024), k_desc = desc(base + Ly::kKvOff, 16, Ly::kGroupBytes),
                   v_desc = desc(base + Ly::kKvOff, 1024, Ly::kGroupBytes);
    const uint32_t tm = __shfl_sync(full, tmem, 0);
    const bool leader = elect_one();
    Ring ring;
    uint32_t q_uses = 0, p_uses[2] = {0, 0}, o_uses[2] = {0, 0};   // p_uses: tiles
    int last_bar = -1;
    uint32_t last_par = 0;
    bool ok = true;
    auto wait = [&](int b, uint32_t par) -> bool {
      return __all_sync(full, mbar_wait(bar(b), par, abort_flag, a.status));
    };
    auto commit = [&](int b) {
      if (leader) mma_commit(bar(b));
    };
    auto issue_s = [&](int w, int q_tile, uint32_t slot) {
      if (leader) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_f16(tm + kSCol + w * 128, q_desc + (q_tile * Ly::kTileBytes + (k >> 2) * (kRows * 128) + (k & 3) * 32) / 16,
                  k_desc + (slot * Ly::kTileBytes + (k >> 2) * 1024 + (k & 3) * 32) / 16, idesc_s, k > 0);
        mma_commit(bar(B_SF + w));
      }
      last_bar = B_SF + w;
      last_par = p_uses[w] & 1u;
    };
    // p arrives in halves of 64 tokens
    auto issue_o = [&](int w, uint32_t slot, bool first) -> bool {
      const uint32_t par = p_uses[w] & 1u;
      ++p_uses[w];
      if (first) {
        if (!wait(B_OE + w, (o_uses[w] & 1u) ^ 1u)) return false;
        ++o_uses[w];
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (!wait(B_PF + 2 * w + b, par)) return false;
        fence_after();
        if (leader) {
#pragma unroll
          for (int k = b * (kTile / 32); k < (b + 1) * (kTile / 32); ++k)
            mma_f16_ta(tm + kOCol + w * 128, tm + kSCol + w * 128 + k * 8,
                       v_desc + (slot * Ly::kTileBytes + k * 2 * Ly::kGroupBytes) / 16, idesc_o, !first || k > 0);
        }
      }
      return true;
    };
    auto finish_o = [&](int w) {
      commit(B_OF + w);
      last_bar = B_OF + w;
      last_par = (o_uses[w] - 1) & 1u;
    };
    auto kv_wait = [&](const Ring& r) {
      const bool r_ok = wait(B_KVF + r.slot, r.par);
      fence_after();
      return r_ok;
    };
    for (uint32_t n = 0; ok; ++n) {
      const uint32_t slot = n % kUnitSlots;
      if (!wait(B_UF + slot, (n / kUnitSlots) & 1u)) break;
      const volatile Unit& x = sched.units[slot];
      const int nt = __shfl_sync(full, x.r < 0 ? -1 : x.t1 - x.t0, 0);
      const bool two = __shfl_sync(full, x.two, 0) != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_UE + slot));
      if (nt < 0) break;
      if (nt == 0) continue;
      ok = wait(B_QF, q_uses & 1u);
      if (!ok) break;
      ++q_uses;
      if (two) {
        ok = kv_wait(ring);
        if (!ok) break;
        issue_s(0, 0, ring.slot);
        issue_s(1, 1, ring.slot);
        commit(B_KVE + ring.slot);
        ring.next(kSlots);
        if (nt == 1) commit(B_QE);
        for (int i = 0; ok && i < nt; ++i) {
          const Ring v = ring;
          ring.next(kSlots);
          const Ring k = ring;
          const bool more = i + 1 < nt;
          if (more) ring.next(kSlots);
          ok = kv_wait(v) && issue_o(0, v.slot, i == 0);
          if (!ok) break;
          if (more) {
            ok = kv_wait(k);
            if (!ok) break;
            issue_s(0, 0, k.slot);
          } else {
            finish_o(0);
          }
          ok = issue_o(1, v.slot, i == 0);
          if (!ok) break;
          commit(B_KVE + v.slot);
          if (more) {
            issue_s(1, 1, k.slot);
            commit(B_KVE + k.slot);
            if (i + 2 == nt) commit(B_QE);
          } else {
            finish_o(1);
          }
        }
      } else {
        // ring order: keys 0, 1, then values t and keys t + 2 in turn
        auto key = [&](int t) -> bool {
          if (!kv_wait(ring)) return false;
          issue_s(t & 1, 0, ring.slot);
          commit(B_KVE + ring.slot);
          ring.next(kSlots);
          if (t + 1 == nt) commit(B_QE);
          return true;
        };
        ok = key(0) && (nt == 1 || key(1));
        for (int t = 0; ok && t < nt; ++t) {
          ok = kv_wait(ring) && issue_o(t & 1, ring.slot, t < 2);
          if (!ok) break;
          commit(B_KVE + ring.slot);
          ring.next(kSlots);
          if (t + 2 < nt) ok = key(t + 2);
          else finish_o(t & 1);
        }
      }
    }
    if (*abort_flag && last_bar >= 0 && lane == 0) mbar_drain(bar(last_bar), last_par);
  }
  } else if (warp < 12) {
    if constexpr (QUANT) asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------------ softmax and output
    // A thread per row; p goes to the second product in two halves of 64 tokens.
    const int w = (warp - 4) >> 2;               // stream
    const int quad = warp & 3;                   // TMEM lanes 32 quad .. + 31
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = tmem + (uint32_t(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + kSCol + w * 128, o_addr = lane_addr + kOCol + w * 128;
    const float c2 = a.scale * kLog2e;
    const float ninf = -__int_as_float(0x7f800000);
    float2* ml = reinterpret_cast<float2*>(smem + Ly::kMlOff);
    const int jr = row / a.G, g = row - jr * a.G;             // token of the tile, head of the group
    uint32_t it = 0, ring = 0, o_uses[2] = {0, 0}, x_uses = 0;
    auto wait = [&](int b, uint32_t par) -> bool {
      return __all_sync(full, mbar_wait(bar(b), par, abort_flag, a.status));
    };
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      const uint32_t slot = n % kUnitSlots;
      if (!wait(B_UF + slot, (n / kUnitSlots) & 1u)) break;
      const volatile Unit& x = sched.units[slot];
      if (x.r < 0) break;
      const int nt = max(0, x.t1 - x.t0);
      const bool two = x.two;
      const int lead = two ? 1 : 2;
      const int n_w = two ? nt : (nt + 1 - w) / 2;
      const int j = x.j0 + (two ? w * tpb : 0) + jr;          // query token of the chunk
      const int live = min(tpb, x.ntok - (two ? w * tpb : 0)) * a.G;   // rows of this tile
      const bool mine = row < live;
      const int lim = x.S - x.A + j;                          // last token this row sees
      const int lim_min = x.S - x.A + x.j0;                   // last token every row of the unit sees
      const bool busy = quad * 32 < live;                     // some row of this warp is live
      const int t_first = x.t0;
      float m = ninf, l = 0.0f;
      for (int i = 0; ok && i < n_w; ++i, ++it) {
        const int t = two ? i : 2 * i + w;                    // tile of this CTA's part
        const int tok0 = (t_first + t) * kTile;
        ok = wait(B_SF + w, it & 1u);
        if (!ok) break;
        // The value rows of tokens past the session's end hold anything (slots never written, another
        // session's rows): zeroed, since 0 * NaN is NaN.  Values that some row of the unit does not
        // see must not reach it either: if one is not finite it is zeroed too, and the rows that do
        // see it get it back at the end.
        if (!QUANT && tok0 + kTile - 1 > lim_min && (!two || w == 0)) {
          const uint32_t pos = ring + v_position(t, nt, lead);
          ok = wait(B_KVF + pos % kSlots, (pos / kSlots) & 1u);
          if (!ok) break;
          clean_values<D, BF16>(smem + Ly::kKvOff + (pos % kSlots) * Ly::kTileBytes + (row >> 3) * Ly::kGroupBytes +
                                (row & 7) * 128, tok0 + row >= x.S, tok0 + row > lim_min, bad_v);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        fence_after();
        if (busy) {
          float v[2][64];
          tmem_ld64(s_addr, v[0]);
          tmem_ld64(s_addr + 64, v[1]);
          tmem_wait(v[0]);
          tmem_wait(v[1]);
          const bool masked = !__all_sync(full, tok0 + kTile - 1 <= lim);
          const int last = lim - tok0;                        // columns 0 .. last are seen
          float mx[4];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            if (masked) {
#pragma unroll
              for (int k = 0; k < 64; ++k) v[hf][k] = hf * 64 + k <= last ? v[hf][k] : ninf;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = hf ? fmax3(mx[e], v[hf][e], v[hf][e + 4]) : fmaxf(v[hf][e], v[hf][e + 4]);
#pragma unroll
            for (int k = 8; k < 64; k += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = fmax3(mx[e], v[hf][k + e], v[hf][k + e + 4]);
          }
          const float top = fmax3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * c2;
          const bool raise = top > m + kSlack;                // also when m is still -inf
          if (__any_sync(full, raise)) {
            const float mn = raise ? top : m;
            const float al = raise ? ex2(m - mn) : 1.0f;      // 0 from m = -inf
            m = mn;
            l *= al;
            if (i > 0) {                                      // O is at rest: its last product came before this S
#pragma unroll 1
              for (int q = 0; q < D / 16; ++q) {
                float o[16];
                tmem_ld16(o_addr + q * 16, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] *= al;
                tmem_st16(o_addr + q * 16, reinterpret_cast<uint32_t*>(o));
              }
            }
          }
          const float off = m == ninf ? 0.0f : m;
          const float2 c2v = make_float2(c2, c2), offv = make_float2(-off, -off);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
          // p of 32 tokens at a time; a store is waited for after the next 32 are computed, and the
          // second product starts on the first 64
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t u[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float* vp = &v[q >> 1][(q & 1) * 32 + 2 * k];
              const float2 e = fma2(make_float2(vp[0], vp[1]), c2v, offv);
              const float2 p = make_float2(ex2(e.x), ex2(e.y));
              sum[k & 1] = add2(sum[k & 1], p);
              u[k] = pack2<BF16>(p.x, p.y);
            }
            if (q == 2) {
              tmem_wait_st();
              fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(B_PF + 2 * w));
            }
            tmem_st16(s_addr + q * 16, u);
          }
          const float2 s2 = add2(sum[0], sum[1]);
          l += s2.x + s2.y;
          tmem_wait_st();
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if (!busy) mbar_arrive(bar(B_PF + 2 * w));
          mbar_arrive(bar(B_PF + 2 * w + 1));
        }
      }
      if (!ok) break;
      ring += 2 * nt;
      // ---- the unit's results
      const int n_o = nt == 0 ? 0 : (two || nt == 1 ? 1 : 2);   // accumulators this warpgroup reads
      const bool joined = !two && nt > 1;                     // stream 1 hands its half over
      if (joined && w == 1) {
        // its last product is done, so the first warpgroup has read the previous unit's (m, l)
        ok = wait(B_OF + 1, o_uses[1] & 1u);
        if (!ok) break;
        ml[row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_XF));
      }
      const int w0 = two ? w : 0;
      if (two || w == 0) {
        for (int s = 0; ok && s < n_o; ++s) ok = wait(B_OF + w0 + s, o_uses[w0 + s] & 1u);
        if (joined) ok = ok && wait(B_XF, x_uses & 1u);
        if (!ok) break;
        fence_after();
        float al0 = 1.0f, al1 = 0.0f;
        if (joined) {
          const float2 y = ml[row];
          const float M = fmaxf(m, y.x);
          al0 = m == ninf ? 0.0f : ex2(m - M);
          al1 = y.x == ninf ? 0.0f : ex2(y.x - M);
          // a row whose keys gave NaN keeps it: l is NaN then, whatever m says
          l = (l == 0.0f ? 0.0f : l * (m == ninf ? 1.0f : al0)) + (y.y == 0.0f ? 0.0f : y.y * (y.x == ninf ? 1.0f : al1));
          m = M;
        }
        const bool whole = x.t0 == 0 && x.t1 == x.nt;
        const bool fix = *bad_v != 0;
        const bool put = mine && j < x.A;
        const int hq = x.h * a.G + g;
        const int64_t qt = int64_t(x.a0) + j;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int pr = (two ? w * kRows : 0) + row;
        float* part = whole ? nullptr : part_of(a.workspace, n_cta, cta, x.t0 > 0 ? 0 : 1);
        if (busy) {
#pragma unroll 1
          for (int q = 0; q < D / 32; ++q) {
            float o[32];
            if (n_o == 0) {
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = 0.0f;
            } else {
              tmem_ld32(lane_addr + kOCol + w0 * 128 + q * 32, o);
              tmem_wait(o);
              if (joined) {
                float o1[32];
                tmem_ld32(lane_addr + kOCol + 128 + q * 32, o1);
                tmem_wait(o1);
                // a stream that saw nothing of this row left zeros
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = fmaf(o[k], al0, o1[k] * al1);
              }
            }
            if (fix && put) {
              const int first = max(lim_min + 1, x.t0 * kTile), last = min(lim, x.t1 * kTile - 1);
              for (int t = first; t <= last; ++t) {
                const int lb = t / a.BS;
                const int phys = lb < a.MB ? a.block_table[x.r * a.bt_stride_r + lb] : -1;
                if (phys < 0 || phys >= a.NB) continue;
                const int64_t at = a.kv_stride_kv + int64_t(phys) * a.kv_stride_b + int64_t(t - lb * a.BS) * a.kv_stride_s;
                if constexpr (QUANT) {           // 32 values share a scale byte; 255 makes them NaN
                  if (static_cast<const uint8_t*>(a.kv)[at + a.Hkv * D + x.h * (D / 32) + q] == 255)
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __int_as_float(0x7fffffff);
                } else {
                  const uint16_t* vr = static_cast<const uint16_t*>(a.kv) + at + int64_t(x.h) * a.kv_stride_h + q * 32;
#pragma unroll
                  for (int k = 0; k < 32; ++k) {
                    const float f = BF16 ? __uint_as_float(uint32_t(vr[k]) << 16) : __half2float(__ushort_as_half(vr[k]));
                    if (!isfinite(f)) o[k] += f;
                  }
                }
              }
            }
            if (put) {
              if (whole) {
                store_row<D, BF16>(static_cast<uint16_t*>(a.out) + qt * a.out_stride_t + int64_t(hq) * a.out_stride_h + q * 32,
                                   o, inv, vec_out);
              } else {
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                  *reinterpret_cast<float4*>(part + int64_t(pr) * D + q * 32 + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
              }
            }
          }
        }
        if (put) {
          if (whole)
            a.lse[qt * a.lse_stride_t + hq] = l == 0.0f ? ninf : (m == ninf ? l : (m + log2f(l)) * 0.69314718055994531f);
          else
            *reinterpret_cast<float2*>(part + int64_t(2 * kRows) * D + 2 * pr) = make_float2(m, l);
        }
        if (!whole && x.t0 == 0 && row == 0 && w == 0) {
          Desc d = {};
          d.valid = 1;
          d.r = x.r;
          d.h = x.h;
          d.j0 = x.j0;
          d.ntok = x.ntok;
          d.S = x.S;
          d.A = x.A;
          d.a0 = x.a0;
          d.end = x.end;
          d.total = sched.total;
          d.two = two;
          static_cast<Desc*>(a.workspace)[cta] = d;
        }
        fence_before();
        __syncwarp();
        if (lane == 0)
          for (int s = 0; s < n_o; ++s) mbar_arrive(bar(B_OE + w0 + s));
      }
      if (two) {
        ++o_uses[0];
        ++o_uses[1];
      } else {
        if (nt > 0) ++o_uses[0];
        if (nt > 1) ++o_uses[1];
      }
      if (joined) ++x_uses;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_UE + slot));
    }
    fence_before();
  } else if constexpr (QUANT) {
    // ------------------------------------------------------------------ e4m3 -> 16 bits (four warps)
    // A warp takes 32 of a tile's tokens: D / 16 lanes per token read 16 values each (one tile ahead, in
    // registers; the tile three further on is asked of L2), and write them converted into the ring in the
    // layout the TMA would have left.
    constexpr int kLpr = D / 16, kRpi = 32 / kLpr, kLoads = 32 / kRpi;
    const int row0 = (warp - 12) * 32, lr = lane / kLpr, lc = lane % kLpr;
    const uint8_t* rows = static_cast<const uint8_t*>(a.kv);
    struct Item {                                // a K or V tile on its way
      int t, plane, S, h, r, lim_min, t1;
    };
    struct Cursor {                              // the unit being loaded
      int t0, t1, lead, p, S, h, r, lim_min;
    } cu;
    uint32_t n = 0;
    bool ok = true;
    auto wait = [&](int b, uint32_t par) -> bool {
      return __all_sync(full, mbar_wait(bar(b), par, abort_flag, a.status));
    };
    cu.t0 = cu.t1 = cu.p = 0;
    auto next_item = [&](Item& y) -> bool {
      while (cu.p >= 2 * (cu.t1 - cu.t0)) {
        const uint32_t slot = n % kUnitSlots;
        if (!wait(B_UF + slot, (n / kUnitSlots) & 1u)) {
          ok = false;
          return false;
        }
        const volatile Unit& x = sched.units[slot];
        const int r = x.r;
        cu.t0 = x.t0;
        cu.t1 = x.t1;
        cu.lead = x.two ? 1 : 2;
        cu.S = x.S;
        cu.h = x.h;
        cu.r = r;
        cu.lim_min = x.S - x.A + x.j0;
        cu.p = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_UE + slot));
        ++n;
        if (r < 0) return false;
      }
      // ring order: keys 0 .. lead - 1, values t and keys t + lead in turn, the last values
      const int nt = cu.t1 - cu.t0, l0 = min(cu.lead, nt), q = cu.p - l0, both = 2 * (nt - l0);
      if (q < 0) {
        y.t = cu.p;
        y.plane = 0;
      } else if (q < both) {
        y.plane = 1 - (q & 1);
        y.t = (q >> 1) + (y.plane ? 0 : l0);
      } else {
        y.plane = 1;
        y.t = nt - l0 + q - both;
      }
      y.t += cu.t0;
      y.S = cu.S;
      y.h = cu.h;
      y.r = cu.r;
      y.lim_min = cu.lim_min;
      y.t1 = cu.t1;
      ++cu.p;
      return true;
    };
    // slot of this lane's token (row0 + lane) of tile t; -1 past the session's end
    auto row_slot = [&](const Item& y, int t) -> int {
      const int tok = t * kTile + row0 + lane;
      if (tok >= y.S || t >= y.t1) return -1;
      const int lb = tok / a.BS;
      int phys = lb < a.MB ? a.block_table[y.r * a.bt_stride_r + lb] : -1;
      if (phys < 0 || phys >= a.NB) {
        flag(a.status, ACTKV_DEV_BAD_INDEX);
        phys = 0;
      }
      return phys * a.BS + (tok - lb * a.BS);
    };
    auto load = [&](const Item& y, int rs, uint4 (&raw)[kLoads], uint32_t (&sc)[kLoads]) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int s = __shfl_sync(full, rs, i * kRpi + lr);
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        sc[i] = 127u;
        if (s >= 0) {
          const uint8_t* row = rows + y.plane * a.kv_stride_kv + int64_t(s) * a.kv_stride_s;
          raw[i] = __ldg(reinterpret_cast<const uint4*>(row + y.h * D + lc * 16));
          sc[i] = __ldg(row + a.Hkv * D + y.h * (D / 32) + (lc >> 1));
        }
      }
    };
    Item cur, nxt;
    uint4 raw[2][kLoads];
    uint32_t sc[2][kLoads];
    Ring ring;
    bool have = next_item(cur);
    if (have) load(cur, row_slot(cur, cur.t), raw[0], sc[0]);
    bool more = have && next_item(nxt);
    int rs = more ? row_slot(nxt, nxt.t) : -1;
    while (have && ok) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {              // two steps, so that the buffers are registers
        if (!have || !ok) break;
        Item nn = nxt;
        if (more) load(nxt, rs, raw[k ^ 1], sc[k ^ 1]);
        const bool more2 = more && next_item(nn);
        if (!ok) break;
        const int rs2 = more2 ? row_slot(nn, nn.t) : -1;
        const int ahead = row_slot(cur, cur.t + 3);
        ok = wait(B_KVE + ring.slot, ring.par ^ 1u);
        if (!ok) break;
        uint8_t* tile = smem + Ly::kKvOff + ring.slot * Ly::kTileBytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int row = row0 + i * kRpi + lr;
          uint4 o[2];
          uint32_t b = sc[k][i];
          if (cur.plane == 1 && b == 255u && cur.t * kTile + row > cur.lim_min) {
            b = 127u;                            // its values are 0; the rows that see it get NaN at the end
            *bad_v = 1;
          }
          widen16<BF16>(raw[k][i], b, o);
          uint8_t* dst = tile + (row >> 3) * Ly::kGroupBytes + (lc >> 2) * 1024 + (row & 7) * 128;
          // the lanes of a token's two halves write even and odd chunks first: eight banks' worth each time
          const int c0 = (lc & 3) * 2, sw = D == 128 ? lc >> 2 : 0;
          *reinterpret_cast<uint4*>(dst + (((c0 + sw) ^ (row & 7)) << 4)) = sw ? o[1] : o[0];
          *reinterpret_cast<uint4*>(dst + (((c0 + 1 - sw) ^ (row & 7)) << 4)) = sw ? o[0] : o[1];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_KVF + ring.slot));
        ring.next(kSlots);
        if (ahead >= 0)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(rows + cur.plane * a.kv_stride_kv + int64_t(ahead) * a.kv_stride_s +
                                                        cur.h * D));
        cur = nxt;
        nxt = nn;
        rs = rs2;
        have = more;
        more = more2;
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ------------------------------------------------------------------------------------ joining split units
constexpr int kJoinThreads = 256;
constexpr int kJoinSlices = 8;               // CTAs per split unit, rows dealt in turn

// One CTA per (CTA that began a unit and left it, slice of its rows); a warp per row.
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) chunk_combine_kernel(const __grid_constant__ ChunkArgs a, int n_cta) {
  pdl_wait();
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Desc d = static_cast<const Desc*>(a.workspace)[cta];
  if (!d.valid) return;
  const float ninf = -__int_as_float(0x7f800000);
  int last = cta;                            // parts: slot 1 of cta, slot 0 of cta + 1 .. last
  while (last + 1 < n_cta && d.total * (last + 1) / n_cta < d.end) ++last;
  const int tpb = kRows / a.G;
  const int live0 = min(tpb, d.ntok) * a.G, live1 = d.two ? (d.ntok - tpb) * a.G : 0;
  for (int i = blockIdx.y * (kJoinThreads / 32) + warp; i < live0 + live1; i += kJoinSlices * (kJoinThreads / 32)) {
    const int b = i < live0 ? 0 : 1;
    const int row = i - b * live0;
    const int pr = b * kRows + row;
    const int jr = row / a.G, hq = d.h * a.G + row - jr * a.G;
    const int64_t qt = int64_t(d.a0) + d.j0 + b * tpb + jr;
    auto ml_of = [&](int c) {
      return *reinterpret_cast<const float2*>(part_of(a.workspace, n_cta, c, c == cta ? 1 : 0) + int64_t(2 * kRows) * D + 2 * pr);
    };
    float M = ninf;
    for (int c = cta + lane; c <= last; c += 32)
      if (d.total * c / n_cta < d.total * (c + 1) / n_cta) M = fmaxf(M, ml_of(c).x);
    M = warp_max(M);
    float L = 0.0f;
    float o[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] = 0.0f;
    for (int c = cta; c <= last; ++c) {
      if (d.total * c / n_cta >= d.total * (c + 1) / n_cta) continue;      // a CTA without a share
      const float2 y = ml_of(c);
      if (y.y == 0.0f) continue;             // saw none of the row's tokens
      const float al = y.x == ninf ? 1.0f : ex2(y.x - M);
      L += y.y * al;
      const float* p = part_of(a.workspace, n_cta, c, c == cta ? 1 : 0) + int64_t(pr) * D;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) o[k] = fmaf(p[k * 32 + lane], al, o[k]);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t* dst = static_cast<uint16_t*>(a.out) + qt * a.out_stride_t + int64_t(hq) * a.out_stride_h;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) dst[k * 32 + lane] = uint16_t(pack2<BF16>(o[k] * inv, 0.0f));
    if (lane == 0)
      a.lse[qt * a.lse_stride_t + hq] = L == 0.0f ? ninf : (M == ninf ? L : (M + log2f(L)) * 0.69314718055994531f);
  }
}

}  // namespace chunk

// ------------------------------------------------------------------------------------ host side
size_t chunk_workspace_bytes(int n_sm) {
  return align256(size_t(n_sm) * (sizeof(chunk::Desc) + 2 * chunk::kPartFloats * sizeof(float)));
}

bool chunk_umma_supported(const ChunkArgs& a, int dtype, const char** why) {
  auto no = [&](const char* w) {
    *why = w;
    return false;
  };
  if (dtype != ACTKV_BF16 && dtype != ACTKV_F16) return no("needs bf16 or fp16");
  if (a.D != 64 && a.D != 128) return no("needs head_dim 64 or 128");
  if (a.G > chunk::kRows) return no("needs a GQA group of at most 128");
  if (!((a.BS % 8 == 0 && chunk::kTile % a.BS == 0) || a.BS % chunk::kTile == 0))
    return no("needs a block size of 8, 16, 32, 64 or a multiple of 128");
  if (a.kv_stride_b != int64_t(a.BS) * a.kv_stride_s || (!a.quant && a.kv_stride_h != a.D))
    return no("needs heads next to one another and blocks of consecutive slots");
  if ((reinterpret_cast<uintptr_t>(a.kv) | reinterpret_cast<uintptr_t>(a.q)) % 16) return no("q and the cache must be 16-byte aligned");
  const int64_t es = a.quant ? 1 : 2;
  if (a.kv_stride_s * es % 16 || a.kv_stride_kv * es % 16 || a.q_stride_h % 8 || a.q_stride_t % 8 || a.kv_stride_s < 0 ||
      a.kv_stride_kv < 0 || a.q_stride_h < 0 || a.q_stride_t < 0)
    return no("strides of q and the cache must be multiples of 16 bytes");
  if (int64_t(a.NB) * a.BS > 0x7fffffffll) return no("too many slots");
  return true;
}

namespace {

template <int D, bool BF16, bool QUANT>
cudaError_t launch_chunk_t(const CUtensorMap& mkv, const CUtensorMap& mq, const ChunkArgs& a, int grid, cudaStream_t st) {
  auto k = chunk::chunk_umma_kernel<D, BF16, QUANT>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(chunk::Layout<D>::kSmemBytes));
  if (e != cudaSuccess) return e;
  const bool vec_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride_t % 8 == 0 && a.out_stride_h % 8 == 0;
  k<<<grid, chunk::threads(QUANT), chunk::Layout<D>::kSmemBytes, st>>>(mkv, mq, a, vec_out);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, chunk::kJoinSlices);
  cfg.blockDim = dim3(chunk::kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, chunk::chunk_combine_kernel<D, BF16>, a, grid);
}

}  // namespace

cudaError_t launch_chunk_umma(const ChunkArgs& a, int dtype, cudaStream_t st, const char** why) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) {
    *why = "cuTensorMapEncodeTiled unavailable";
    return cudaErrorNotSupported;
  }
  const CUtensorMapDataType dt = dtype == ACTKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  CUtensorMap mkv = {}, mq;
  if (!a.quant) {
    // (64 dims, slot within 8, D-half of a head, group of 8 slots, plane): a box leaves every 8-token
    // group's D-halves next to one another, so the groups of a tile are evenly spaced
    const cuuint32_t halves = cuuint32_t(a.D / 64), rows = cuuint32_t(a.BS < chunk::kTile ? a.BS : chunk::kTile);
    const cuuint64_t row = cuuint64_t(a.kv_stride_s) * 2;
    const cuuint64_t dims[5] = {64, 8, cuuint64_t(a.Hkv) * halves, cuuint64_t(a.NB) * a.BS / 8, 2};
    const cuuint64_t strides[4] = {row, 128, row * 8, cuuint64_t(a.kv_stride_kv) * 2};
    const cuuint32_t box[5] = {64, 8, halves, rows / 8, 1};
    if (enc(&mkv, dt, 5, const_cast<void*>(a.kv), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
      *why = "cuTensorMapEncodeTiled rejected the cache layout";
      return cudaErrorInvalidValue;
    }
  }
  {
    const cuuint64_t dims[3] = {cuuint64_t(a.D), cuuint64_t(a.Hq), cuuint64_t(a.T)};
    const cuuint64_t strides[2] = {cuuint64_t(a.q_stride_h) * 2, cuuint64_t(a.q_stride_t) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(a.G), cuuint32_t(chunk::kRows / a.G)};
    if (enc(&mq, dt, 3, const_cast<void*>(a.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
      *why = "cuTensorMapEncodeTiled rejected the query layout";
      return cudaErrorInvalidValue;
    }
  }
  *why = "chunk attention";
  const int grid = device_sm_count();
  const bool bf = dtype == ACTKV_BF16;
  if (a.quant) {
    if (a.D == 128) return bf ? launch_chunk_t<128, true, true>(mkv, mq, a, grid, st) : launch_chunk_t<128, false, true>(mkv, mq, a, grid, st);
    return bf ? launch_chunk_t<64, true, true>(mkv, mq, a, grid, st) : launch_chunk_t<64, false, true>(mkv, mq, a, grid, st);
  }
  if (a.D == 128) return bf ? launch_chunk_t<128, true, false>(mkv, mq, a, grid, st) : launch_chunk_t<128, false, false>(mkv, mq, a, grid, st);
  return bf ? launch_chunk_t<64, true, false>(mkv, mq, a, grid, st) : launch_chunk_t<64, false, false>(mkv, mq, a, grid, st);
}

}  // namespace actkv
