// Chunk attention over the paged cache on the sm_100a tensor cores (tcgen05 + TMA + TMEM): the newest
// A of a session's S tokens are the queries, query j sees tokens t <= S - A + j, and the call gives
// out = softmax(scale q.k) v and lse = log sum exp(scale q.k) of every (query, head) row.
//
// With c = scale * log2 e and a reference exponent m per row, p_t = 2^(c q.k_t - m), l = sum p_t,
// O = sum p_t v_t, out = O / l, lse = (m + log2 l) ln 2.  m need not be the running maximum, only
// near it: it is raised (and O and l rescaled) when the maximum has grown by more than 2^8, so p
// stays below 2^8 and the rescaling, a pass over O, is rare.  S = Q K^T and O are accumulated in 32
// bits in TMEM, m and l are 32-bit registers; p is rounded to the cache's 16-bit type for the second
// product only (l sums the unrounded values), the same half unit that the output is rounded by (fp16 p, held times
// 2^7: or 2^-32 of the largest, when that is more).  32 bits tell logits apart up to about 2^24.
//
// Work.  A unit is (session, KV head, group of up to 256 query rows): rows are (token, head of the
// GQA group), two tiles of 128.  The units' key tiles of 128 tokens, laid end to end with a fixed
// cost per unit, are cut into one equal share per CTA (one CTA per SM), so ragged batches, one long
// session and many short ones balance alike; a unit that a cut divides leaves 32-bit partial
// results (m, l, O) in the workspace, at most two per CTA, which chunk_combine_kernel joins in a
// fixed order.  Sessions of few query rows are chunk_few.cu's.
//
// Two streams of (S, p, O) run in a CTA, each with its own softmax warpgroup and 256 TMEM columns:
//   two row tiles   both streams take every key tile (one copy of K and V serves 256 rows)
//   one row tile    (few new tokens) stream w takes every second key tile with the same queries,
//                   and the first warpgroup joins the two at the end
// While one stream's softmax runs, the tensor core works on the other's products.
//
// Warp roles: warp 0 walks the schedule, announces units to the others (so that only it spends registers
// on it) and issues the TMA copies (a paged block per lane and tile: one 5-D box of 8-token groups x
// both D-halves, 4 KB for blocks of 16: the copy engine spends ~60 cycles per box whatever its size, and 2 KB
// boxes, one per D-half, gave 7.1 TB/s from L2 against 10.6); warp 1 issues the MMAs (p from TMEM as
// the A operand, V as an MN-major B operand straight from the tile); warps 4-7 and 8-11 are the
// softmax warpgroups (a thread per row, p handed over in halves of 64 tokens).  Over the 8-bit and
// 4-bit caches the TMA brings the tiles as they are, warp 2 their scale bytes, and warps 12-19 widen them into the ring.  Every
// wait is bounded.
//
// What bounds it.  128 x 128 logits take the tensor core 1024 cycles (two products of head size 128) and the
// special-function unit as many (16 exponentials per cycle), so both would have to be full all the time.
// Measured for a 2048-token chunk over 32K tokens (32 heads over 8, 1.07 TFLOP): 1.02 to 1.11 ms by board, 960 to 1040
// TFLOP/s, with the board at its power limit and the SM clock at 1450 to 1600 MHz (cuBLAS at that limit:
// 1385): about 0.6 of the tensor rate at that clock, the rest going into the chain from S through
// softmax (~1900 cycles: 350 to read S, 350 for the maximum, 1100 for the exponentials, which two warps per
// scheduler share) to the products.  The row groups of a head run at the same time at unrelated key tiles, so
// tiles come from DRAM several times over: 1.17 GB for 4 chunks of 512 over 10240, where keys, values and queries are
// 185 MB; at 3.5 TB/s that is no bound by itself, what it takes from the power limit is not known.  Tried on that chunk (head
// size 128, where the tensor core takes as long as the exponentials; not at 64) and not kept: 1 in 2, 4 or 8
// exponentials on the FMA pipe (polynomial of degree 4: 941, 1050, 1097 TFLOP/s against 1098), two threads per row
// (640 threads of 104 registers, spills: 858 against 960), S in halves of 64 tokens with twice the buffers (M128 N64
// products run at 0.6 of their rate from shared memory: 864).  What helped: descriptors in uniform registers (issue by an
// elected lane of a converged warp, 880 to 963), p in halves, packed 32-bit math, and code that fits the
// instruction cache (the 8-bit variant 650 to 480 us for 4 chunks of 512 over 4K to 16K tokens, and to 430 with the
// softmax in a loop over halves of a row and a shorter widening, its cache's hit rate 0.88 to 0.96; 447 and 0.945 since
// it looks for e4m3's NaN; the 4-bit variant, whose tiles are widened by way of 32 bits, 492).
#include <cuda.h>

#include "chunk_common.cuh"

namespace actkv {
namespace chunk {

using namespace umma;

constexpr int kMaxThreads = 640;
constexpr int threads(bool quant) { return quant ? 640 : 384; }
constexpr int kUnitSlots = 4;               // units announced ahead of their results

constexpr uint32_t kSchedBytes = 512;

// BITS: of the cache's values: 16, 8 or 4
template <int D, int BITS>
struct Layout {
  static constexpr bool QUANT = BITS != 16;
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kTileBytes = kTile * D * 2;      // a K, V or Q tile
  static constexpr int kSlots = (BITS == 8 ? 3 : (BITS == 4 ? 4 : 5)) * (128 / D);
  static constexpr uint32_t kGroupBytes = kHalves * 1024;    // 8 tokens of a K / V tile
  static constexpr uint32_t kKvOff = 2 * kTileBytes;
  // the 8- or 4-bit cache's tiles before they are widened, and their scale words per token
  static constexpr int kRaw = QUANT ? (D == 128 ? 3 : 6) : 0;
  static constexpr uint32_t kRawBytes = kTile * D * BITS / 8;
  static constexpr uint32_t kRawOff = kKvOff + kSlots * kTileBytes;
  static constexpr uint32_t kScaleOff = kRawOff + kRaw * kRawBytes;
  static constexpr uint32_t kMlOff = kScaleOff + kRaw * kTile * 4;       // stream 1's (m, l) per row
  static constexpr uint32_t kBarOff = kMlOff + kRows * 8;
  // kv_full[slots] kv_empty[slots] q_full q_empty s_full[2] p_full[2][2] o_full[2] o_empty[2]
  // x_full unit_full[4] unit_empty[4] raw_full[raw] raw_empty[raw] scale_full[raw]
  static constexpr int kNumBars = 2 * kSlots + 13 + 2 * kUnitSlots + 3 * kRaw;
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

struct Sched {               // in shared memory
  Share share;
  uint32_t tmem;
  int abort_flag;
  int bad_v;                 // a value that some row of the unit does not see is not finite
  int gaps;                  // some block was outside the cache: from there on every tile looks for them
  int few_rows;              // sessions of at most so many rows are chunk_few_kernel's in this call
  int64_t scan[kMaxThreads / 32], sums[2];
  Unit units[kUnitSlots];    // from the TMA warp, which alone walks the schedule; r < 0 ends it
};
static_assert(sizeof(Sched) <= kSchedBytes, "the schedule's place in shared memory");

struct Geometry {
  const ChunkArgs* a;
  int tpb;                   // tokens per row tile
  __device__ explicit Geometry(const ChunkArgs& args) : a(&args), tpb(kRows / args.G) {}
  __device__ int groups(int A) const { return (A + 2 * tpb - 1) / (2 * tpb); }
  // key tiles that some query of tokens [j0, j0 + n) sees
  __device__ int tiles(int S, int A, int j_end) const {
    const int last = min(S - A + j_end, table_room(*a)) - 1;
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
  int r, h, j, S, A, a0, few_rows;

  __device__ void load() {
    while (r < a->R) {
      a0 = a->q_off[r];
      A = new_tokens(*a, r);
      S = a->seq_used[r];
      if (A > 0 && A * a->G > few_rows) return;
      ++r;
    }
  }
  __device__ Walker(const ChunkArgs* args, const Sched& s, int cta, int n) : a(args), geo(*args) {
    n = used_ctas(s.share.total, n, 1);
    lo = s.share.total * cta / n;
    hi = cta < n ? s.share.total * (cta + 1) / n : lo;
    r = s.share.r0;
    few_rows = s.few_rows;
    h = j = S = A = a0 = 0;
    at = s.share.pre;
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
__device__ void make_schedule(const ChunkArgs& a, Sched& s, int few_rows, int cta, int n) {
  const Geometry geo(a);
  if (threadIdx.x == 0) s.few_rows = few_rows;
  share_out<kThreads>(a.R, [&](int r) -> int64_t {
    const int A = new_tokens(a, r);
    if (A == 0 || A * a.G <= few_rows) return 0;
    flag_long(a, a.seq_used[r]);
    return a.Hkv * geo.head_weight(a.seq_used[r], A);
  }, s.share, s.scan, cta, n, 1);
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
__device__ __forceinline__ void tmem_fill8(uint32_t taddr, uint32_t x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%1], {%0,%0,%0,%0,%0,%0,%0,%0};" ::"r"(x), "r"(taddr) : "memory");
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

// The waits of this kernel, bounded like mbar_wait's but shorter: the kernel's roles share an instruction
// cache, which the waits' slow paths filled.  false when the wait gave up (about 2^31 cycles; *abort is
// then 1, and the kernel reports it at its end) or another role did.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t abort) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 t0, t1;\n\t.reg .b32 a;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra done;\n\t"
      "mov.u64 t0, %%clock64;\n"
      "again:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n\t"
      "@p bra done;\n\t"
      "ld.volatile.shared.b32 a, [%3];\n\t"
      "setp.ne.b32 q, a, 0;\n\t"
      "@q bra done;\n\t"
      "mov.u64 t1, %%clock64;\n\t"
      "sub.s64 t1, t1, t0;\n\t"
      "setp.lt.s64 q, t1, %5;\n\t"
      "@q bra again;\n\t"
      "st.volatile.shared.b32 [%3], 1;\n"
      "done:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(abort), "r"(kSleepNs), "l"(kTimeoutCycles)
      : "memory");
  return ok != 0;
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

// The K and V tiles of a unit's part in ring order: keys 0 .. lead - 1, then values t and keys t + lead
// in turn, then the last values.
struct UnitItems {
  int t0 = 0, nt = 0, lead = 0, p = 0, S = 0, h = 0, r = 0, hidden = 0;
  __device__ bool done() const { return p >= 2 * nt; }
  __device__ void start(const volatile Unit& x) {
    r = x.r;
    t0 = x.t0;
    nt = r < 0 ? 0 : max(0, x.t1 - x.t0);
    lead = min(x.two ? 1 : 2, nt);
    S = x.S;
    h = x.h;
    hidden = x.S - x.A + x.j0 + 1;           // the first token that some row does not see
    p = 0;
  }
  __device__ void next(int& t, int& plane) {
    const int q = p - lead, both = 2 * (nt - lead);
    plane = q < 0 ? 0 : (q < both ? 1 - (q & 1) : 1);
    t = t0 + (q < 0 ? p : (q < both ? (q >> 1) + (plane ? 0 : lead) : nt - lead + q - both));
    ++p;
  }
};

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

// One token's values of a tile in shared memory: zeroed when the token is past the session's end; when
// `hidden` (some row does not see it), what is not finite is zeroed and *bad_v set.
template <int D, bool BF16>
__device__ __forceinline__ void clean_values(uint8_t* tile, bool past, bool hidden, volatile int* bad_v) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  if (!past && !hidden) return;
#pragma unroll 1
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
template <int D, bool BF16, int BITS>
__global__ void __launch_bounds__(threads(BITS != 16), 1)
    chunk_umma_kernel(const __grid_constant__ CUtensorMap tmap_kv, const __grid_constant__ CUtensorMap tmap_q,
                      const __grid_constant__ ChunkArgs a, bool vec_out) {
  using Ly = Layout<D, BITS>;
  constexpr bool QUANT = BITS != 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Ly::kBarOff);
  Sched& sched = *reinterpret_cast<Sched*>(smem + Ly::kSchedOff);
  volatile int* abort_flag = &sched.abort_flag;
  const uint32_t abort_addr = smem_u32(&sched.abort_flag);
  volatile int* bad_v = &sched.bad_v;
  volatile int* gaps = &sched.gaps;
  // token tok of session r is in a block outside the cache
  auto missing = [&](int r, int tok) {
    const int lb = tok / a.BS;
    return lb >= a.MB || uint32_t(a.block_table[r * a.bt_stride_r + lb]) >= uint32_t(a.NB);
  };
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  constexpr int kSlots = Ly::kSlots;
  constexpr int B_KVF = 0, B_KVE = kSlots, B_QF = 2 * kSlots, B_QE = B_QF + 1, B_SF = B_QE + 1, B_PF = B_SF + 2,
                B_OF = B_PF + 4, B_OE = B_OF + 2, B_XF = B_OE + 2, B_UF = B_XF + 1,
                B_UE = B_UF + kUnitSlots, B_RF = B_UE + kUnitSlots, B_RE = B_RF + Ly::kRaw, B_CF = B_RE + Ly::kRaw;
  const unsigned full = 0xffffffffu;
  const int cta = blockIdx.x, n_cta = gridDim.x;

  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) flag(a.status, ACTKV_DEV_MISALIGNED);
    return;
  }
  const int few_rows = few_rows_now<threads(QUANT)>(a, sched.sums);
  if (few_rows > 0 && sched.sums[0] == sched.sums[1]) {      // every session is of few rows: chunk_few_kernel's
    if (threadIdx.x == 0) wide_parts(a.workspace, n_cta).desc[cta].valid = 0;
    pdl_trigger();
    pdl_wait();
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(bar(B_KVF + i), QUANT ? 8 : 1);
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
      mbar_init(bar(B_UE + i), QUANT ? 18 : 9);   // MMA, softmax, scale and widening warps
    }
    for (int i = 0; i < Ly::kRaw; ++i) {
      mbar_init(bar(B_RF + i), 1);
      mbar_init(bar(B_RE + i), 8);
      mbar_init(bar(B_CF + i), 1);
    }
    sched.share = Share{0, 0, a.R};
    sched.abort_flag = 0;
    sched.bad_v = 0;
    sched.gaps = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    wide_parts(a.workspace, n_cta).desc[cta].valid = 0;
  }
  pdl_trigger();
  __syncthreads();
  make_schedule<threads(QUANT)>(a, sched, few_rows, cta, n_cta);
  if (sched.share.total == 0) {              // nothing to do
    pdl_wait();
    return;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sched.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sched.tmem;
  const int tpb = kRows / a.G;

  // 384 threads of 168 registers: the softmax warps take 208 each, the others keep 88.  With the
  // widening warps 640 threads of 96: 152 and 56, and 56 for those.
  if (warp < 4) {
  if constexpr (QUANT) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (whole warp)
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_kv)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_q)) : "memory");
    }
    const int bs_box = min(a.BS, kTile);         // token rows of a box
    const int bpt = kTile / bs_box;              // boxes per tile (<= 16: one per lane)
    const int mpb = a.BS / bs_box;               // tiles per block, of blocks longer than a tile
    const uint32_t box_bytes = uint32_t(bs_box) * D * BITS / 8;
    // where the copies go: the ring itself, or the tiles to be widened into it
    constexpr int kIn = QUANT ? Ly::kRaw : kSlots, B_FULL = QUANT ? B_RF : B_KVF, B_EMPTY = QUANT ? B_RE : B_KVE;
    Walker wk(&a, sched, cta, n_cta);
    Unit x;
    uint32_t ring = 0, q_uses = 0;
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
      const bool any = wk.next(x);
      ok = __all_sync(full, bar_wait(bar(B_UE + n % kUnitSlots), ((n / kUnitSlots) & 1u) ^ 1u, abort_addr));
      if (!ok) break;
      if (lane == 0) {
        if (!any) x.r = -1;
        sched.units[n % kUnitSlots] = x;
        mbar_arrive(bar(B_UF + n % kUnitSlots));
      }
      if (!any) break;
      if (x.t0 >= x.t1) continue;
      const int lead = x.two ? 1 : 2, nt = x.t1 - x.t0;
      // first token slot (16-bit rows: in units of 8) of lane b's box of key tile t; -2 past the session's end or when
      // the block is outside the cache (its tokens are hidden; the copies' barrier orders `gaps` before the tile)
      auto read_id = [&](int t) -> int {
        if (lane >= bpt || t < x.t0 || t >= x.t1 || t * kTile + lane * bs_box >= x.S) return -2;
        const int lb = mpb == 1 ? t * bpt + lane : t / mpb;
        const int phys = lb < a.MB ? a.block_table[x.r * a.bt_stride_r + lb] : -1;
        if (phys < 0 || phys >= a.NB) {
          flag(a.status, ACTKV_DEV_BAD_INDEX);
          *gaps = 1;
          return -2;
        }
        const int64_t first = int64_t(phys) * a.BS + (mpb == 1 ? 0 : (t - lb * mpb) * kTile);
        return int(first >> (QUANT ? 0 : 3));
      };
      ok = __all_sync(full, bar_wait(bar(B_QE), (q_uses & 1u) ^ 1u, abort_addr));
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
      auto load = [&](int id, int plane) -> bool {
        const int slot = ring % kIn;
        const bool w2 = bar_wait(bar(B_EMPTY + slot), ((ring / kIn) & 1u) ^ 1u, abort_addr);
        if (!__all_sync(full, w2)) return false;
        const int n = __popc(__ballot_sync(full, id >= 0));
        if (lane == 0) mbar_expect_tx(bar(B_FULL + slot), uint32_t(n) * box_bytes);
        __syncwarp();
        if (id >= 0) {
          if constexpr (QUANT)
            tma_load_3d(base + Ly::kRawOff + slot * Ly::kRawBytes + lane * box_bytes, &tmap_kv, bar(B_FULL + slot),
                        x.h * (D * BITS / 8), id, plane);
          else
            tma_load_5d(base + Ly::kKvOff + slot * Ly::kTileBytes + lane * box_bytes, &tmap_kv, bar(B_FULL + slot), 0, 0,
                        x.h * Ly::kHalves, id, plane);
        }
        ++ring;
        return true;
      };
      // keys `lead` tiles ahead of the values; block ids three tiles ahead of the values
      int id0 = -2, id1 = -2, id2 = -2;
#pragma unroll 1
      for (int t = -lead - 3; ok && t < nt; ++t) {
        if (t >= 0) ok = load(id0, 1);
        if (ok && t >= -lead && t + lead < nt) ok = load(lead == 1 ? id1 : id2, 0);
        id0 = id1;
        id1 = id2;
        id2 = read_id(x.t0 + t + 3);
      }
      if (!ok) break;
    }
    if (*abort_flag && lane == 0) {
      for (uint32_t s = 0; s < kIn; ++s) {
        const uint32_t uses = ring / kIn + (s < ring % kIn ? 1u : 0u);
        if (uses) mbar_drain(bar(B_FULL + s), (uses - 1) & 1u);
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
      return __all_sync(full, bar_wait(bar(b), par, abort_addr));
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
      // Either in steps: the second product of step s, then the logits of step s + 2 of the same stream, two row tiles
      // taking every key tile in a step each and one row tile a key tile per step.  Or the same order written out, with
      // streams and tiles known to the compiler, which issues sooner but is longer code.  2048 tokens over 32768: 1120
      // us in steps, 1063 written out; 1088 over 2000 to 10000 623 and 601; head size 64, fp16, 171 and 174; 8-bit
      // rows, whose five roles crowd the instruction cache, only lose by longer code.
      if constexpr (QUANT || D == 64) {
        const int steps = two ? 2 * nt : nt;
        Ring v, k;
#pragma unroll 1
        for (int s = -2; s < steps; ++s) {
          const int w = s & 1;
          const bool opens = !two || w == 0, closes = !two || w == 1, more = s + 2 < steps;
          if (s >= 0) {
            if (opens) {
              v = ring;
              ring.next(kSlots);
              ok = kv_wait(v);
            }
            ok = ok && issue_o(w, v.slot, s < 2);
            if (!ok) break;
            if (closes) commit(B_KVE + v.slot);
          }
          if (more) {
            if (opens) {
              k = ring;
              ring.next(kSlots);
              ok = kv_wait(k);
              if (!ok) break;
            }
            issue_s(w, two ? w : 0, k.slot);
            if (closes) commit(B_KVE + k.slot);
            if (s + 3 == steps) commit(B_QE);
          } else if (s >= 0) {
            finish_o(w);
          }
        }
      } else if (two) {
        ok = kv_wait(ring);
        if (!ok) break;
        issue_s(0, 0, ring.slot);
        issue_s(1, 1, ring.slot);
        commit(B_KVE + ring.slot);
        ring.next(kSlots);
        if (nt == 1) commit(B_QE);
#pragma unroll 1
        for (int i = 0; i < nt; ++i) {
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
#pragma unroll 1
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
  } else if (QUANT && warp == 2) {
    // ------------------------------------------------------------------ scale words of the 8- or 4-bit rows
    // Four tokens per lane, from the cache through registers (one tile ahead) into the tile's words.
    const int bpt = a.BS < kTile ? kTile / a.BS : 1, mpb = a.BS < kTile ? 1 : a.BS / kTile;
    int sub[4], in_block[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sub[i] = mpb == 1 ? (lane + 32 * i) / a.BS : 0;
      in_block[i] = lane + 32 * i - sub[i] * a.BS;
    }
    UnitItems u;
    uint32_t n = 0, w0[4] = {}, w1[4] = {};
    Ring ring;
    bool have = false, more = true;
    auto wait = [&](int b, uint32_t par) -> bool {
      return __all_sync(full, bar_wait(bar(b), par, abort_addr));
    };
    auto put_words = [&]() -> bool {             // the words in hand, when their tile's place is free
      if (!have) return true;
      if (!wait(B_RE + ring.slot, ring.par ^ 1u)) return false;
      uint32_t* dst = reinterpret_cast<uint32_t*>(smem + Ly::kScaleOff) + ring.slot * kTile;
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[lane + 32 * i] = w0[i];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_CF + ring.slot));
      ring.next(Ly::kRaw);
      have = false;
      return true;
    };
    while (have || more) {
      while (more && u.done()) {
        const uint32_t slot = n % kUnitSlots;
        more = wait(B_UF + slot, (n / kUnitSlots) & 1u);
        if (!more) break;
        u.start(sched.units[slot]);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_UE + slot));
        ++n;
        // A unit without tiles: the one after it is announced, kUnitSlots on, only when the unit whose words are
        // in hand is finished, so they go out first.
        more = u.r >= 0 && (!u.done() || put_words());
      }
      if (more) {
        int t, plane;
        u.next(t, plane);
        const int block0 = mpb == 1 ? t * bpt : t / mpb, off = mpb == 1 ? 0 : (t - block0 * mpb) * kTile;
        const int32_t* table = a.block_table + u.r * a.bt_stride_r;
        const uint8_t* p0 = static_cast<const uint8_t*>(a.kv) + plane * a.kv_stride_kv + a.Hkv * (D * BITS / 8) + u.h * (D / 32);
        int phys[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int lb = block0 + sub[i];
          phys[i] = t * kTile + lane + 32 * i < u.S && lb < a.MB ? table[lb] : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t ph = uint32_t(phys[i]) < uint32_t(a.NB) ? phys[i] : 0;   // else hidden, whatever the bytes say
          const uint8_t* p = p0 + uint64_t(ph * uint32_t(a.BS) + uint32_t(in_block[i] + off)) * uint32_t(a.kv_stride_s);
          if constexpr (D == 128) w1[i] = *reinterpret_cast<const uint32_t*>(p);
          else w1[i] = *reinterpret_cast<const uint16_t*>(p) | 0x7f7f0000u;
        }
      }
      if (!put_words()) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) w0[i] = w1[i];
      have = more;
    }
  }
  } else if (warp < 12) {
    if constexpr (QUANT) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
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
      return __all_sync(full, bar_wait(bar(b), par, abort_addr));
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
        // see it get it back at the end.  Tokens of blocks outside the cache were not copied: hidden from all.
        const bool gap = *gaps;
        const bool masked = !__all_sync(full, tok0 + kTile - 1 <= lim && !gap);
        if (!QUANT && (masked || tok0 + kTile - 1 > lim_min) && (!two || w == 0)) {
          const uint32_t pos = ring + v_position(t, nt, lead);
          ok = wait(B_KVF + pos % kSlots, (pos / kSlots) & 1u);
          if (!ok) break;
          clean_values<D, BF16>(smem + Ly::kKvOff + (pos % kSlots) * Ly::kTileBytes + (row >> 3) * Ly::kGroupBytes +
                                (row & 7) * 128, tok0 + row >= x.S || (gap && missing(x.r, tok0 + row)),
                                tok0 + row > lim_min, bad_v);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        fence_after();
        if (busy) {
          // With the widening warps a thread has registers for half a row only: the second half is read for
          // the maximum, and again for p.
          float v[QUANT ? 1 : 2][64];
          const int last = lim - tok0;                        // columns 0 .. last are seen
          float mx[4] = {ninf, ninf, ninf, ninf};
          if (masked) {                                       // hidden columns become -inf where they are
            if (__any_sync(full, gap)) {                      // 8 tokens are in one block
#pragma unroll 1
              for (int q = 0; q < kTile / 8; ++q)
                if (missing(x.r, tok0 + q * 8)) tmem_fill8(s_addr + q * 8, __float_as_uint(ninf));
              tmem_wait_st();
            }
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
              if (__all_sync(full, q * 16 + 15 <= last)) continue;
              float x[16];
              tmem_ld16(s_addr + q * 16, x);
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] = q * 16 + k <= last ? x[k] : ninf;
              tmem_st16(s_addr + q * 16, reinterpret_cast<uint32_t*>(x));
            }
            tmem_wait_st();
          }
          auto half_max = [&](float (&x)[64]) {
#pragma unroll
            for (int k = 0; k < 64; k += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = fmax3(mx[e], x[k + e], x[k + e + 4]);
          };
          if constexpr (QUANT) {
#pragma unroll 1
            for (int h = 1; h >= 0; --h) {
              tmem_ld64(s_addr + h * 64, v[0]);
              tmem_wait(v[0]);
              half_max(v[0]);
            }
          } else {
            tmem_ld64(s_addr, v[0]);
            tmem_ld64(s_addr + 64, v[QUANT ? 0 : 1]);
            tmem_wait(v[0]);
            tmem_wait(v[QUANT ? 0 : 1]);
            half_max(v[0]);
            half_max(v[QUANT ? 0 : 1]);
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
          auto quarter = [&](const float (&x)[64], int at, uint32_t (&u)[16]) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 e = fma2(make_float2(x[at + 2 * k], x[at + 2 * k + 1]), c2v, offv);
              const float2 p = make_float2(ex2(e.x), ex2(e.y));
              sum[k & 1] = add2(sum[k & 1], p);
              u[k] = pack_p<BF16>(p.x, p.y);
            }
          };
          // p of 32 tokens at a time; the second product starts on the first 64
          if constexpr (QUANT) {
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              if (h) {
                tmem_ld64(s_addr + 64, v[0]);
                tmem_wait(v[0]);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PF + 2 * w));
              }
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t u[16];
                quarter(v[0], q * 32, u);
                tmem_st16(s_addr + h * 32 + q * 16, u);
              }
            }
          } else {
            // a store is waited for after the next 32 are computed
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t u[16];
              quarter(v[QUANT ? 0 : q >> 1], (q & 1) * 32, u);
              if (q == 2) {
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PF + 2 * w));
              }
              tmem_st16(s_addr + q * 16, u);
            }
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
        const float inv = over<BF16>(l);
        const int pr = (two ? w * kRows : 0) + row;
        const Parts ps = wide_parts(a.workspace, n_cta);
        const int ps_slot = x.t0 > 0 ? 0 : 1;
        float* part = ps.out(cta, ps_slot);
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
        // values that some row does not see and that are not finite went in as zeros: the rows that do see them
        if (fix && put) {
          uint16_t* dst = static_cast<uint16_t*>(a.out) + qt * a.out_stride_t + int64_t(hq) * a.out_stride_h;
          const int first = max(lim_min + 1, x.t0 * kTile), end = min(lim, x.t1 * kTile - 1);
#pragma unroll 1
          for (int t = first; t <= end; ++t) {
            const int lb = t / a.BS;
            const int phys = lb < a.MB ? a.block_table[x.r * a.bt_stride_r + lb] : -1;
            if (phys < 0 || phys >= a.NB) continue;
            const int64_t at = a.kv_stride_kv + int64_t(phys) * a.kv_stride_b + int64_t(t - lb * a.BS) * a.kv_stride_s;
#pragma unroll 1
            for (int d = 0; d < D; ++d) {
              float f;
              if constexpr (QUANT) {
                if constexpr (BITS == 4) f = value4(static_cast<const uint8_t*>(a.kv) + at, a.Hkv, D, x.h, d);
                else f = quant_value<BF16>(static_cast<const uint8_t*>(a.kv) + at, a.Hkv, D, x.h * D + d);
              } else {
                const uint16_t u = static_cast<const uint16_t*>(a.kv)[at + int64_t(x.h) * a.kv_stride_h + d];
                f = BF16 ? __uint_as_float(uint32_t(u) << 16) : __half2float(__ushort_as_half(u));
              }
              if (isfinite(f)) continue;
              if (whole) {
                const float y = BF16 ? __uint_as_float(uint32_t(dst[d]) << 16) : __half2float(__ushort_as_half(dst[d]));
                dst[d] = uint16_t(pack2<BF16>(y + f, 0.0f));
              } else {
                part[int64_t(pr) * D + d] += f;
              }
            }
          }
        }
        if (put) {
          if (whole)
            a.lse[qt * a.lse_stride_t + hq] = l == 0.0f ? ninf : (m == ninf ? l : (m + log2f(l)) * 0.69314718055994531f);
          else
            *reinterpret_cast<float2*>(ps.ml(cta, ps_slot, D) + 2 * pr) = make_float2(m, l);
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
          d.total = sched.share.total;
          d.heads = 1;
          d.n_used = used_ctas(d.total, n_cta, 1);
          d.two = two;
          ps.desc[cta] = d;
        }
        fence_before();
        __syncwarp();
        if (lane == 0)
          for (int s = 0; s < n_o; ++s) mbar_arrive(bar(B_OE + w0 + s));
      }
      // the accumulators that the unit produced: none where its rows see no token
      if (nt > 0) ++o_uses[0];
      if (nt > (two ? 0 : 1)) ++o_uses[1];
      if (joined) ++x_uses;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_UE + slot));
    }
    fence_before();
  } else if constexpr (QUANT) {
    // ------------------------------------------------------------------ 8 or 4 -> 16 bits (eight warps)
    // A warp takes 16 of a tile's tokens, 16 bytes of one per lane, and leaves them in the ring in the layout the TMA
    // leaves 16-bit rows in.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    constexpr int kLpr = D * BITS / 128, kRpi = 32 / kLpr;   // lanes per token, tokens at a time
    const int row0 = (warp - 12) * 16, lr = lane / kLpr, lc = lane % kLpr;
    // Where a lane's piece comes from and its two 16-byte pieces go within 8 tokens.  The lanes of a token's two
    // halves write even and odd chunks first: eight banks' worth each time.
    const bool sw = D == 128 && lc >= 4;
    constexpr int kPer8 = BITS == 8 ? 8 / kRpi : 1;
    [[maybe_unused]] uint32_t get[kPer8], put0[kPer8], put1[kPer8];
#pragma unroll
    for (int i = 0; i < kPer8; ++i) {
      const int r8 = i * kRpi + lr, c0 = (lc & 3) * 2;
      get[i] = r8 * D + ((lc ^ (D == 128 ? r8 : (r8 >> 1) & 3)) << 4);
      put0[i] = (lc >> 2) * 1024 + r8 * 128 + (((c0 + sw) ^ r8) << 4);
      put1[i] = (lc >> 2) * 1024 + r8 * 128 + (((c0 + 1 - sw) ^ r8) << 4);
    }
    [[maybe_unused]] auto put = [&](uint8_t* p0, uint8_t* p1, const uint32_t (&r)[8]) {
      *reinterpret_cast<uint4*>(p0) = sw ? make_uint4(r[4], r[5], r[6], r[7]) : make_uint4(r[0], r[1], r[2], r[3]);
      *reinterpret_cast<uint4*>(p1) = sw ? make_uint4(r[0], r[1], r[2], r[3]) : make_uint4(r[4], r[5], r[6], r[7]);
    };
    UnitItems u;
    Ring ring, in;
    uint32_t n = 0;
    bool ok = true;
    auto wait = [&](int b, uint32_t par) -> bool {
      return __all_sync(full, bar_wait(bar(b), par, abort_addr));
    };
    while (true) {
      while (ok && u.done()) {
        const uint32_t slot = n % kUnitSlots;
        ok = wait(B_UF + slot, (n / kUnitSlots) & 1u);
        if (!ok) break;
        u.start(sched.units[slot]);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_UE + slot));
        ++n;
        if (u.r < 0) break;
      }
      if (!ok || u.r < 0) break;
      int t, plane;
      u.next(t, plane);
      ok = wait(B_CF + in.slot, in.par) && wait(B_RF + in.slot, in.par) && wait(B_KVE + ring.slot, ring.par ^ 1u);
      if (!ok) break;
      uint32_t sc = reinterpret_cast<const uint32_t*>(smem + Ly::kScaleOff)[in.slot * kTile + row0 + (lane & 15)];
      const int first = t * kTile + row0;                     // the warp's first token
      const bool gap = *gaps, edge = first + 16 > min(u.S, plane ? u.hidden : u.S);
      const bool plain = __all_sync(full, (BITS == 4 ? plain_scales4<BF16>(sc) : plain_scales<BF16>(sc)) && !gap);
      uint32_t gone = 0;                                      // the warp's tokens that are not there: zeros
      if (edge || !plain) {
        const int tok = first + (lane & 15);
        const bool out = tok >= u.S || (gap && missing(u.r, tok));
        gone = __ballot_sync(full, out);
        if (out) sc = 0x7f7f7f7fu;
      }
      const uint8_t* src = smem + Ly::kRawOff + in.slot * Ly::kRawBytes + row0 * (D * BITS / 8);
      uint8_t* dst = smem + Ly::kKvOff + ring.slot * Ly::kTileBytes + (row0 >> 3) * Ly::kGroupBytes;
      if constexpr (BITS == 4) {
        // A lane's 16 bytes are four chunks of 8 dims: of each of four groups (head size 128), of two halves of two (64).
        // Lanes whose tokens share banks take the groups in another order.
        bool found = false;
        const bool swap = (D == 128 ? lr : lr >> 1) & 1;
#pragma unroll 1
        for (int i = 0; i < 16 / kRpi; ++i) {
          const int row = i * kRpi + lr, r8 = row & 7;        // of the warp's 16
          uint4 x = *reinterpret_cast<const uint4*>(src + row * (D / 2) + lc * 16);
          const uint32_t word = __shfl_sync(full, sc, row);
          if (gone >> row & 1u) x = make_uint4(0u, 0u, 0u, 0u);
          const bool hide = plane && first + row >= u.hidden; // some row does not see it: NaN goes in as 0
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t eight;                   // the chunk's values
            int g, chunk;
            if constexpr (D == 128) {
              g = swap ? c ^ 1 : c;
              chunk = (g & 1) * 4 + lc;
              eight = __byte_perm(c < 2 ? x.x : x.y, c < 2 ? x.z : x.w, g & 1 ? 0x7632 : 0x5410);
            } else {
              g = swap ? (c >> 1) ^ 1 : c >> 1;
              chunk = g * 4 + lc * 2 + (c & 1);
              eight = __byte_perm(c & 1 ? x.z : x.x, c & 1 ? x.w : x.y, g & 1 ? 0x7632 : 0x5410);
            }
            const uint32_t b = word >> (8 * g) & 255u;
            uint32_t y[4];
            if (plain) widen4<BF16>(eight, plain_factor4(b), y);
            else widen4_any<BF16>(eight, b, y);
            if (hide) {
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = drop_bad<BF16>(y[k], 0xffffffffu, found);
            }
            *reinterpret_cast<uint4*>(dst + (row >> 3) * Ly::kGroupBytes + (g >> 1) * (D == 128 ? 1024 : 0) + r8 * 128 +
                                      ((chunk ^ r8) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
        if (found) *bad_v = 1;
      } else {
      // Rolled, 8 tokens at a time: the warps of a scheduler are at five places of the kernel, and straight code
      // for all 16 tokens starved it of instructions.
      bool slow = edge || !plain;
      if (!slow) {
        uint32_t seen = 0;
#pragma unroll 1
        for (int g8 = 0; g8 < 2; ++g8) {
#pragma unroll
          for (int i = 0; i < 8 / kRpi; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + g8 * 8 * D + get[i]);
            const uint32_t b = __byte_perm(__shfl_sync(full, sc, g8 * 8 + i * kRpi + lr), 0u, 0x4440 | (lc >> 1));
            uint32_t r[8];
            widen16<BF16>(x, plain_factor<BF16>(b), r, seen);
            put(dst + g8 * Ly::kGroupBytes + put0[i], dst + g8 * Ly::kGroupBytes + put1[i], r);
          }
        }
        slow = __any_sync(full, any_nan_byte(seen));
      }
      if (slow) {
#pragma unroll 1
        for (int i = 0; i < 16 / kRpi; ++i) {
          const int row = i * kRpi + lr, g8 = i * kRpi / 8;     // of the warp's 16
          const bool odd = i * kRpi % 8 != 0;
          uint4 x = *reinterpret_cast<const uint4*>(src + g8 * 8 * D + (odd ? get[8 / kRpi - 1] : get[0]));
          if (gone >> row & 1u) x = make_uint4(0u, 0u, 0u, 0u);
          const uint32_t b = __byte_perm(__shfl_sync(full, sc, row), 0u, 0x4440 | (lc >> 1));
          uint32_t r[8], f[3], seen = 0;
          any_factors<BF16>(b, f);
          widen16<BF16>(x, f[0], r, seen);
          const uint32_t in4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t m = __byte_perm(in4[k >> 1] & 0x7f7f7f7fu, 0u, (k & 1) ? 0x4342 : 0x4140);
            r[k] = put_nan(mul_rest<BF16>(r[k], f[1], f[2]), m);
          }
          if (plane && first + row >= u.hidden) {   // some row does not see it: what is not finite goes in as 0
            bool found = false;
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = drop_bad<BF16>(r[k], 0xffffffffu, found);
            if (found) *bad_v = 1;
          }
          uint8_t* d8 = dst + g8 * Ly::kGroupBytes;
          put(d8 + (odd ? put0[8 / kRpi - 1] : put0[0]), d8 + (odd ? put1[8 / kRpi - 1] : put1[0]), r);
        }
      }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(B_RE + in.slot));
        mbar_arrive(bar(B_KVF + ring.slot));
      }
      ring.next(kSlots);
      in.next(Ly::kRaw);
    }
  }
  __syncthreads();
  pdl_wait();                                // chunk_few_kernel is done too when this one is
  if (threadIdx.x == 0 && *abort_flag) flag(a.status, ACTKV_DEV_TIMEOUT);
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ------------------------------------------------------------------------------------ joining split units
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kJoinSlices = 16;              // CTAs per split unit, rows dealt in turn

// One CTA per (CTA that began a unit and left it, slice of its rows): a warp per row where a row has up to 8
// parts, else its warps take them in turn and the warps' sums are added in order (one token over 2000: 21
// parts, 28.7 -> 22.4 us for the call).  The slices from kJoinSlices on are for the units of
// chunk_few_kernel.  Bound by latency: two dependent reads per eight parts, a row after the other.
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) chunk_combine_kernel(const __grid_constant__ ChunkArgs a, int n_cta,
                                                                     int first_slice) {
  __shared__ float sh_m[kJoinWarps], sh_l[kJoinWarps], sh_o[kJoinWarps][D];
  pdl_wait();
  constexpr int kPer = D / 32;                              // values per lane
  const bool few = first_slice + int(blockIdx.y) >= kJoinSlices;
  const Parts ps = few ? few_parts(a.workspace, n_cta) : wide_parts(a.workspace, n_cta);
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = (first_slice + blockIdx.y) % kJoinSlices;
  const Desc d = ps.desc[cta];
  if (!d.valid) return;
  const float ninf = -__int_as_float(0x7f800000);
  // parts: slot 1 of cta, slot 0 of cta + 1 .. last, the last CTA whose share total * c / n_used starts before end
  const int last = int((d.end * d.n_used - 1) / d.total);
  const int tpb = kRows / a.G;
  const int live0 = (d.two ? tpb : d.ntok) * a.G, live1 = d.two ? (d.ntok - tpb) * a.G : 0, live = live0 + live1;
  // where row i of the unit is: in the parts, and in the results
  auto place = [&](int i, int& pr, int64_t& qt, int& hq) {
    const int hh = i / live, ii = i - hh * live;
    const int b = ii < live0 ? 0 : 1, row = ii - b * live0;
    const int jr = row / a.G;
    pr = few ? i : b * kRows + row;
    hq = (d.h + hh) * a.G + row - jr * a.G;
    qt = int64_t(d.a0) + d.j0 + b * tpb + jr;
  };
  // a warp's sum over the parts c, c + step, ..
  float M, L, o[kPer];
  auto add = [&](float2 y, const float (&x)[kPer]) {
    if (y.y == 0.0f) return;                 // saw none of the row's tokens
    const float Mn = fmaxf(M, y.x), al = M == Mn ? 1.0f : ex2(M - Mn), be = y.x == Mn ? 1.0f : ex2(y.x - Mn);
    M = Mn;
    L = fmaf(L, al, y.y * be);
#pragma unroll
    for (int k = 0; k < kPer; ++k) o[k] = fmaf(o[k], al, x[k] * be);
  };
  auto add_parts = [&](int pr, int c, int step) {
    M = ninf;
    L = 0.0f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) o[k] = 0.0f;
#pragma unroll 4
    for (; c <= last; c += step) {
      const float* p = ps.out(c, c == cta ? 1 : 0);
      const float2 y = *reinterpret_cast<const float2*>(p + int64_t(ps.rows) * D + 2 * pr);
      float x[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) x[k] = p[int64_t(pr) * D + k * 32 + lane];
      add(y, x);
    }
  };
  auto lse_of = [&](float m, float l) { return l == 0.0f ? ninf : (m == ninf ? l : (m + log2f(l)) * 0.69314718055994531f); };
  int pr, hq;
  int64_t qt;
  if (last - cta < kJoinWarps) {              // few parts: a warp per row
    for (int i = slice * kJoinWarps + warp; i < live * d.heads; i += kJoinSlices * kJoinWarps) {
      place(i, pr, qt, hq);
      add_parts(pr, cta, 1);
      uint16_t* dst = static_cast<uint16_t*>(a.out) + qt * a.out_stride_t + int64_t(hq) * a.out_stride_h;
      const float inv = over<BF16>(L);
#pragma unroll
      for (int k = 0; k < kPer; ++k) dst[k * 32 + lane] = uint16_t(pack2<BF16>(o[k] * inv, 0.0f));
      if (lane == 0) a.lse[qt * a.lse_stride_t + hq] = lse_of(M, L);
    }
    return;
  }
  for (int i = slice; i < live * d.heads; i += kJoinSlices) {   // many: the warps share a row's
    place(i, pr, qt, hq);
    // four parts' reads at a time, then their sums (148 parts of one token over 32768, 19 per warp: 36 us part by part)
    add_parts(pr, last + 1, 1);
#pragma unroll 1
    for (int c = cta + warp; c <= last; c += 4 * kJoinWarps) {
      float2 y[4];
      float x[4][kPer];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = make_float2(0.0f, 0.0f);
        if (c + e * kJoinWarps > last) continue;
        const float* p = ps.out(c + e * kJoinWarps, c + e * kJoinWarps == cta ? 1 : 0);
        y[e] = *reinterpret_cast<const float2*>(p + int64_t(ps.rows) * D + 2 * pr);
#pragma unroll
        for (int k = 0; k < kPer; ++k) x[e][k] = p[int64_t(pr) * D + k * 32 + lane];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) add(y[e], x[e]);
    }
    if (lane == 0) {
      sh_m[warp] = M;
      sh_l[warp] = L;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) sh_o[warp][k * 32 + lane] = o[k];
    __syncthreads();
    if (threadIdx.x < D) {
      float m = ninf, l = 0.0f, y = 0.0f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, sh_m[w]);
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        if (sh_l[w] == 0.0f) continue;
        const float al = sh_m[w] == m ? 1.0f : ex2(sh_m[w] - m);
        l = fmaf(sh_l[w], al, l);
        y = fmaf(sh_o[w][threadIdx.x], al, y);
      }
      static_cast<uint16_t*>(a.out)[qt * a.out_stride_t + int64_t(hq) * a.out_stride_h + threadIdx.x] =
          uint16_t(pack2<BF16>(l == 0.0f ? 0.0f : y / (l * kPScale<BF16>), 0.0f));
      if (threadIdx.x == 0) a.lse[qt * a.lse_stride_t + hq] = lse_of(m, l);
    }
    __syncthreads();
  }
}

}  // namespace chunk

// ------------------------------------------------------------------------------------ host side
size_t chunk_workspace_bytes(int n_sm) {
  return align256(chunk::few_offset(n_sm) + chunk::parts_bytes(n_sm, chunk::kFewParts));
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
  if (int64_t(a.NB) * a.BS > 0x7fffffffll || a.kv_stride_s > 0x7fffffffll) return no("too many slots, or too far apart");
  return true;
}

namespace {

template <int D, bool BF16, int BITS>
cudaError_t launch_chunk_t(const CUtensorMap& mkv, const CUtensorMap& mq, const ChunkArgs& a, int grid, cudaStream_t st) {
  auto k = chunk::chunk_umma_kernel<D, BF16, BITS>;
  cudaError_t e = cudaSuccess;
  const bool vec_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride_t % 8 == 0 && a.out_stride_h % 8 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  const bool wide = a.T * int64_t(a.G) > a.few_rows;         // else every session is chunk_few_kernel's
  if (wide) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(chunk::threads(BITS != 16));
    cfg.dynamicSmemBytes = chunk::Layout<D, BITS>::kSmemBytes;
    static SmemLimit limit;
    if ((e = limit.set(reinterpret_cast<const void*>(k), int(cfg.dynamicSmemBytes))) != cudaSuccess) return e;
    cfg.numAttrs = a.few_rows > 0 ? 1 : 0;   // beside chunk_few_kernel's last CTAs
    if ((e = cudaLaunchKernelEx(&cfg, k, mkv, mq, a, vec_out)) != cudaSuccess) return e;
  }
  cfg.gridDim = dim3(grid, ((wide ? 1 : 0) + (a.few_rows > 0 ? 1 : 0)) * chunk::kJoinSlices);
  cfg.blockDim = dim3(chunk::kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, chunk::chunk_combine_kernel<D, BF16>, a, grid, wide ? 0 : chunk::kJoinSlices);
}

template <int BITS>
cudaError_t launch_chunk_bits(const CUtensorMap& mkv, const CUtensorMap& mq, const ChunkArgs& a, int dtype, int grid, cudaStream_t st) {
  const bool bf = dtype == ACTKV_BF16;
  if (a.D == 128) return bf ? launch_chunk_t<128, true, BITS>(mkv, mq, a, grid, st) : launch_chunk_t<128, false, BITS>(mkv, mq, a, grid, st);
  return bf ? launch_chunk_t<64, true, BITS>(mkv, mq, a, grid, st) : launch_chunk_t<64, false, BITS>(mkv, mq, a, grid, st);
}

}  // namespace

cudaError_t launch_chunk_umma(const ChunkArgs& args, int dtype, cudaStream_t st, const char** why) {
  ChunkArgs a = args;
  *why = "chunk attention";
  const int grid = device_sm_count();
  // sessions of few query rows go to a kernel of their own, where a GQA group fits it
  a.few_rows = a.G <= chunk::few_group(a.quant) ? chunk::few_limit(a.quant) : 0;
  if (a.few_rows > 0) {
    const cudaError_t e = a.quant == 4 ? launch_chunk_few4(a, dtype, grid, st) : launch_chunk_few(a, dtype, grid, st);
    if (e != cudaSuccess) return e;
  }
  CUtensorMap mkv, mq;
  if (a.T * int64_t(a.G) > a.few_rows) {     // chunk_umma_kernel is launched
    EncodeTiledFn enc = get_encode_fn();
    if (!enc) {
      *why = "cuTensorMapEncodeTiled unavailable";
      return cudaErrorNotSupported;
    }
    const CUtensorMapDataType dt = dtype == ACTKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint32_t es[5] = {1, 1, 1, 1, 1};
    if (a.quant) {
      // (the heads' values of a row, slot, plane): one head's values of a paged block per box
      const cuuint32_t rows = cuuint32_t(a.BS < chunk::kTile ? a.BS : chunk::kTile);
      const cuuint32_t bytes = cuuint32_t(a.D * a.quant / 8);
      const cuuint64_t dims[3] = {cuuint64_t(a.Hkv) * bytes, cuuint64_t(a.NB) * a.BS, 2};
      const cuuint64_t strides[2] = {cuuint64_t(a.kv_stride_s), cuuint64_t(a.kv_stride_kv)};
      const cuuint32_t box[3] = {bytes, rows, 1};
      if (enc(&mkv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(a.kv), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE,
              a.quant == 4 ? CU_TENSOR_MAP_SWIZZLE_NONE : (a.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B),
              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        *why = "cuTensorMapEncodeTiled rejected the layout of the rows";
        return cudaErrorInvalidValue;
      }
    } else {
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
  }
  *why = "chunk attention";
  if (a.quant == 8) return launch_chunk_bits<8>(mkv, mq, a, dtype, grid, st);
  if (a.quant == 4) return launch_chunk_bits<4>(mkv, mq, a, dtype, grid, st);
  return launch_chunk_bits<16>(mkv, mq, a, dtype, grid, st);
}

}  // namespace actkv
