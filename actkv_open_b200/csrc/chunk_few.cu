// Chunk attention of sessions with few new tokens (a single token, a drafted run: at most 16 query rows,
// token x head of the GQA group, per KV head) over the paged cache: the formulas of chunk_umma.cu.
//
// Such a call reads each key and value once for a handful of products, so memory bounds it: 4 (2 over
// the 8-bit cache) bytes per value pair against 2 * rows operations.  What matters is bytes in flight
// and no hand-overs between them and the sums.  So there are none: a warp copies 16 tokens of keys
// and values (cp.async, a private ring of several steps), reads them as operands of the warp-wide
// m16n8k16 product straight from there, keeps its own running maximum, sum and output in registers,
// and the warps meet once per unit.  The 128-row tensor-core tile of chunk_umma.cu would be at most
// an eighth full here, and over the 8-bit cache would need the widened values in shared memory;
// here they are widened in registers on their way into the product.
//
// Operands.  S = Q K^T: the product sums over dims in any order, as long as both operands agree, so a
// lane's four dims of a k-step are consecutive ones of a 16-byte piece of its token's row.  O = P V:
// columns come in any order, so lane group n takes dims (D / 8) n + j in its j-th product, again
// consecutive bytes of a row; the pairs of tokens that an operand register holds are put together
// by byte permutes.  p goes from the layout of S to that of the second product without a move.
//
// Work is shared out as in chunk_umma.cu: equal shares of key tiles per CTA, a unit being (session, KV head);
// the eight warps of a CTA take every eighth step of 16 tokens of its part.
#include <type_traits>

#include "chunk_common.cuh"

namespace actkv {
namespace chunk {
namespace few {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 16;                   // tokens per step

template <int D, bool QUANT>
struct Ring {
  static constexpr int kEs = QUANT ? 1 : 2;
  static constexpr int kChunks = D * kEs / 16;              // 16-byte pieces of a row
  static constexpr uint32_t kPlane = kStep * D * kEs;       // keys, then values
  static constexpr uint32_t kStage = 2 * kPlane + (QUANT ? 128 : 0);     // and their scale words
  static constexpr int kStages = QUANT ? 6 : (D == 128 ? 3 : 6);
  static constexpr uint32_t kBytes = kWarps * kStages * kStage;
  static constexpr uint32_t kJoinBytes = kWarps * kFewRows * (D + 4) * 4;
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

// Two e4m3 bytes, one atop each half of x (anything below them), times f.
template <bool BF16>
__device__ __forceinline__ uint32_t widen2(uint32_t x, uint32_t f) {
  return mul16x2<BF16>(((x >> (BF16 ? 4 : 1)) & (BF16 ? 0x07f007f0u : 0x3f803f80u)) | (x & 0x80008000u), f);
}
// ... for any scale bytes of the two halves.
template <bool BF16>
__device__ __forceinline__ uint32_t widen2_any(uint32_t x, uint32_t b_lo, uint32_t b_hi) {
  uint32_t l1, l2, h1, h2;
  any_factors<BF16>(b_lo, l1, l2);
  any_factors<BF16>(b_hi, h1, h2);
  uint32_t r = widen2<BF16>(x, __byte_perm(l1, h1, 0x5410));
  if (b_lo == 255u) l2 = BF16 ? 0x3f803f80u : 0x3c003c00u;             // 1: NaN stays
  if (b_hi == 255u) h2 = BF16 ? 0x3f803f80u : 0x3c003c00u;
  r = mul16x2<BF16>(r, __byte_perm(l2, h2, 0x5410));
  if constexpr (!BF16) {                      // past fp16's range: its largest
    asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x7bff7bffu));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0xfbfffbffu));
  }
  return r;
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

struct Sched {
  Share share;
  int64_t scan[kWarps];
  int bad_v;
};
static_assert(sizeof(Sched) <= 512, "the schedule's place in shared memory");

template <int D, bool BF16, bool QUANT>
__global__ void __launch_bounds__(kThreads, 1) chunk_few_kernel(const __grid_constant__ ChunkArgs a) {
  using Rg = Ring<D, QUANT>;
  constexpr int CH = Rg::kChunks, kRowsPerCopy = 32 / CH, kCopies = kStep / kRowsPerCopy;
  constexpr int kKSteps = D / 16, kTiles = D / 8;           // products per S, per O
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
  share_out<kThreads>(a.R, [&](int r) -> int64_t {
    const int A = a.q_off[r + 1] - a.q_off[r];
    return A > 0 && A * a.G <= a.few_rows ? int64_t(a.Hkv) * (kUnitCost + (a.seq_used[r] + kTile - 1) / kTile) : 0;
  }, sched.share, sched.scan, cta, n_cta);
  const int64_t lo = sched.share.total * cta / n_cta, hi = sched.share.total * (cta + 1) / n_cta;
  if (lo >= hi) return;
  int r = sched.share.r0;
  int64_t at = sched.share.pre;              // start of (session r, head h) in the schedule
  int h = 0;
  bool seek = true;
  const float c2 = a.scale * kLog2e;
  const char* kv = static_cast<const char*>(a.kv);
  const int64_t es = QUANT ? 1 : 2, stride_s = a.kv_stride_s * es, stride_b = a.kv_stride_b * es;

  for (; r < a.R && at < hi; ++r, h = 0) {
    const int a0 = a.q_off[r], A = a.q_off[r + 1] - a0, S = a.seq_used[r];
    if (A <= 0 || A * a.G > a.few_rows) continue;
    const int rows = A * a.G;
    const int nt = S > 0 ? (S + kTile - 1) / kTile : 0;
    const int64_t weight = kUnitCost + nt;
    if (seek) {                               // the head that holds lo
      h = int((lo - at) / weight);
      at += h * weight;
      seek = false;
    }
    const int32_t* table = a.block_table + r * a.bt_stride_r;
    for (; h < a.Hkv && at < hi; ++h, at += weight) {
      const int64_t first = at + kUnitCost;
      const int t0 = int(lo > first ? lo - first : 0), t1 = nt == 0 ? 0 : int(min(int64_t(nt), hi - first));
      if (nt == 0 ? at < lo : t0 >= t1) continue;
      const int begin = t0 * kTile, end = min(t1 * kTile, S);
      const int steps = (end - begin + kStep - 1) / kStep;
      const int mine = warp < steps ? (steps - warp + kWarps - 1) / kWarps : 0;    // steps of this warp
      const int lim0 = S - A + r8 / a.G, lim1 = S - A + (r8 + 8) / a.G;           // last tokens the lane's rows see
      const bool wide = rows > 8;
      // ---- queries as the first operand: for each k-step rows r8 and r8 + 8, dims as the keys come
      uint32_t q[kKSteps][4];
      {
        const uint16_t* qp = static_cast<const uint16_t*>(a.q);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = r8 + hf * 8, jq = row / a.G;
          const uint16_t* p = qp + (int64_t(a0) + jq) * a.q_stride_t + int64_t(h * a.G + row - jq * a.G) * a.q_stride_h;
#pragma unroll
          for (int k = 0; k < kKSteps; ++k) {
            // the dims of k-step k: 4 consecutive ones of piece c4 + 4 i
            const int per = QUANT ? 4 : 2;    // k-steps per piece
            const int d = (c4 + 4 * (k / per)) * (per * 4) + (k % per) * 4;
            const uint2 u = row < rows ? *reinterpret_cast<const uint2*>(p + d) : make_uint2(0u, 0u);
            q[k][hf] = u.x;
            q[k][2 + hf] = u.y;
          }
        }
      }
      float o[kTiles][4];
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
      float m0 = ninf, m1 = ninf, l0 = 0.0f, l1 = 0.0f;

      // ---- copies of step i of this warp: lane l < 16 looks up token l's slot a step ahead
      auto look_up = [&](int i) -> int {
        const int tok = begin + (warp + i * kWarps) * kStep + (lane & 15);
        if (i >= mine || tok >= end) return -2;
        const int lb = tok / a.BS;
        return lb < a.MB ? table[lb] : -1;
      };
      int phys = look_up(0);
      auto issue = [&](int i, int slot) {
        const int t = begin + (warp + i * kWarps) * kStep;
        if (i < mine) {
          int ph = phys;
          if (ph != -2 && (ph < 0 || ph >= a.NB)) {
            flag(a.status, ACTKV_DEV_BAD_INDEX);
            ph = 0;
          }
          const int tok = t + (lane & 15);
          const int64_t off = ph < 0 ? -1 : int64_t(ph) * stride_b + int64_t(tok % a.BS) * stride_s;
          const uint32_t dst = ring + slot * Rg::kStage;
          const int64_t head = QUANT ? int64_t(h) * D : int64_t(h) * a.kv_stride_h * 2;
#pragma unroll
          for (int e = 0; e < kCopies; ++e) {
            const int row = e * kRowsPerCopy + lane / CH, c = lane % CH;
            const int64_t from = __shfl_sync(full, off, row);
            const char* p = kv + (from < 0 ? 0 : from + head + c * 16);
            copy16(dst + row * (CH * 16) + key_piece<CH>(row, c) * 16, p, from >= 0);
            copy16(dst + Rg::kPlane + row * (CH * 16) + value_piece<CH>(row, c) * 16,
                   from < 0 ? p : p + a.kv_stride_kv * es, from >= 0);
          }
          if constexpr (QUANT) {              // words: lanes 0-15 the keys', 16-31 the values'
            const int at_word = a.Hkv * D + (D == 128 ? h * 4 : (h * 2) & ~3);
            copy4(dst + 2 * Rg::kPlane + lane * 4, kv + (off < 0 ? 0 : off + at_word + (lane >> 4) * a.kv_stride_kv), off >= 0);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        phys = look_up(i + 1);
      };

      auto step = [&](int i, int slot, auto edge_) {
        constexpr bool EDGE = decltype(edge_)::value;        // hidden tokens, or scale bytes out of the ordinary
        const int t = begin + (warp + i * kWarps) * kStep;
        const uint32_t kb = ring + slot * Rg::kStage, vb = kb + Rg::kPlane, sb = kb + 2 * Rg::kPlane;
        const int sh = QUANT && D == 64 && (h & 1) ? 16 : 0; // the head's bytes within the word
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int row = n * 8 + r8;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
          [[maybe_unused]] const uint32_t word = QUANT ? lds4(sb + row * 4) >> sh : 0u;
#pragma unroll
          for (int p = 0; p < (CH + 3) / 4; ++p) {
            const uint4 u = lds16(kb + row * (CH * 16) + key_piece<CH>(row, c4 + 4 * p) * 16);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            if constexpr (QUANT) {            // 16 dims: four k-steps of one scale group
              const uint32_t b = (word >> ((c4 + 4 * p) / 2 * 8)) & 255u, f = plain_factor<BF16>(b);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t x0 = __byte_perm(w[k], 0u, 0x1404), x1 = __byte_perm(w[k], 0u, 0x3424);
                mma16816<BF16>(s[n], q[p * 4 + k], EDGE ? widen2_any<BF16>(x0, b, b) : widen2<BF16>(x0, f),
                               EDGE ? widen2_any<BF16>(x1, b, b) : widen2<BF16>(x1, f));
              }
            } else {                          // 8 dims: two k-steps
              mma16816<BF16>(s[n], q[p * 2], w[0], w[1]);
              mma16816<BF16>(s[n], q[p * 2 + 1], w[2], w[3]);
            }
          }
        }
        // s[n][0..1]: row r8, tokens t + 8 n + 2 c4, + 1; s[n][2..3]: row r8 + 8
        float top0 = ninf, top1 = ninf;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (EDGE) {
              const int tok = t + 8 * n + 2 * c4 + e;
              s[n][e] = tok <= lim0 && tok < end ? s[n][e] : ninf;
              s[n][2 + e] = tok <= lim1 && tok < end ? s[n][2 + e] : ninf;
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
          const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
          const float e0 = m0 == n0 ? 1.0f : ex2(m0 - n0), e1 = m1 == n1 ? 1.0f : ex2(m1 - n1);
          m0 = n0;
          m1 = n1;
          l0 *= e0;
          l1 *= e1;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            o[j][0] *= e0;
            o[j][1] *= e0;
            o[j][2] *= e1;
            o[j][3] *= e1;
          }
        }
        const float b0 = m0 == ninf ? 0.0f : m0, b1 = m1 == ninf ? 0.0f : m1;
        uint32_t p[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float x = ex2(fmaf(s[n][0], c2, -b0)), y = ex2(fmaf(s[n][1], c2, -b0));
          l0 += x + y;
          p[2 * n] = pack2<BF16>(x, y);
          if (wide) {
            const float z = ex2(fmaf(s[n][2], c2, -b1)), w = ex2(fmaf(s[n][3], c2, -b1));
            l1 += z + w;
            p[2 * n + 1] = pack2<BF16>(z, w);
          }
        }
        // ---- values: tokens 2 c4, 2 c4 + 1 and those + 8, dims kTiles r8 ..
        const int row[4] = {2 * c4, 2 * c4 + 1, 2 * c4 + 8, 2 * c4 + 9};
        uint32_t hide[2] = {0u, 0u};
        if constexpr (EDGE) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
            hide[n] = (t + row[2 * n] > S - A ? 0xffffu : 0u) | (t + row[2 * n + 1] > S - A ? 0xffff0000u : 0u);
        }
        bool found = false;
        if constexpr (QUANT) {
          uint32_t w[4][kTiles / 4], b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t base = vb + row[e] * (CH * 16);
            if constexpr (D == 128) {
              const uint4 u = lds16(base + value_piece<CH>(row[e], r8) * 16);
              w[e][0] = u.x;
              w[e][1] = u.y;
              w[e][kTiles / 4 - 2] = u.z;
              w[e][kTiles / 4 - 1] = u.w;
            } else {
              const uint2 u = lds8(base + value_piece<CH>(row[e], r8 >> 1) * 16 + (r8 & 1) * 8);
              w[e][0] = u.x;
              w[e][1] = u.y;
            }
            b[e] = (lds4(sb + 64 + row[e] * 4) >> (sh + kTiles * r8 / 32 * 8)) & 255u;
            if constexpr (EDGE) {
              if (b[e] == 255u && t + row[e] > S - A) {     // its values are 0; the rows that see it get NaN later
                b[e] = 127u;
                found = true;
              }
            }
          }
          const uint32_t f0 = __byte_perm(plain_factor<BF16>(b[0]), plain_factor<BF16>(b[1]), 0x5410);
          const uint32_t f1 = __byte_perm(plain_factor<BF16>(b[2]), plain_factor<BF16>(b[3]), 0x5410);
#pragma unroll
          for (int k = 0; k < kTiles / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {     // dim 4 k + e: its byte of two tokens atop the halves
              const uint32_t sel = 0x0000u | (e << 4) | ((4 + e) << 12);
              const uint32_t x0 = __byte_perm(w[0][k], w[1][k], sel), x1 = __byte_perm(w[2][k], w[3][k], sel);
              mma16816<BF16>(o[k * 4 + e], p, EDGE ? widen2_any<BF16>(x0, b[0], b[1]) : widen2<BF16>(x0, f0),
                             EDGE ? widen2_any<BF16>(x1, b[2], b[3]) : widen2<BF16>(x1, f1));
            }
        } else {
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
        if (EDGE && found) sched.bad_v = 1;
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
        const int t = begin + (warp + i * kWarps) * kStep;
        bool edge = t + kStep - 1 > S - A || t + kStep > end;
        if constexpr (QUANT) {
          const uint32_t word = lds4(ring + slot * Rg::kStage + 2 * Rg::kPlane + lane * 4);
          edge = edge || !__all_sync(full, plain_scales<BF16>(word));
        }
        if (edge) step(i, slot, std::true_type());
        else step(i, slot, std::false_type());
        __syncwarp();                         // every lane has read the slot that the next copies fill
        slot = slot + 1 == Rg::kStages ? 0 : slot + 1;
        fill = fill + 1 == Rg::kStages ? 0 : fill + 1;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      // ---- the warps meet: (m, l) and O of each through shared memory
      l0 += __shfl_xor_sync(full, l0, 1);
      l0 += __shfl_xor_sync(full, l0, 2);
      l1 += __shfl_xor_sync(full, l1, 1);
      l1 += __shfl_xor_sync(full, l1, 2);
      __syncthreads();                        // the rings are free
      float* jo = reinterpret_cast<float*>(smem) + warp * kFewRows * D;
      float2* jml = reinterpret_cast<float2*>(smem + kWarps * kFewRows * D * 4) + warp * kFewRows;
      if (c4 == 0) {
        jml[r8] = make_float2(m0, l0);
        jml[r8 + 8] = make_float2(m1, l1);
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {      // columns 2 c4, 2 c4 + 1 of product j: dims kTiles n + j
        if (r8 < rows) {
          jo[r8 * D + kTiles * (2 * c4) + j] = o[j][0];
          jo[r8 * D + kTiles * (2 * c4 + 1) + j] = o[j][1];
        }
        if (r8 + 8 < rows) {
          jo[(r8 + 8) * D + kTiles * (2 * c4) + j] = o[j][2];
          jo[(r8 + 8) * D + kTiles * (2 * c4 + 1) + j] = o[j][3];
        }
      }
      __syncthreads();
      const bool whole = t0 == 0 && t1 == nt, fix = sched.bad_v != 0;
      const int ps_slot = t0 > 0 ? 0 : 1;
      const float2* all_ml = reinterpret_cast<const float2*>(smem + kWarps * kFewRows * D * 4);
      for (int x = threadIdx.x; x < rows * D; x += kThreads) {
        const int row = x / D, d = x - row * D;
        float M = ninf;
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, all_ml[w * kFewRows + row].x);
        float L = 0.0f, y = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = all_ml[w * kFewRows + row];
          if (ml.y == 0.0f) continue;         // saw none of the row's tokens
          const float al = ml.x == ninf ? 1.0f : ex2(ml.x - M);
          L = fmaf(ml.y, al, L);
          y = fmaf(reinterpret_cast<const float*>(smem)[(w * kFewRows + row) * D + d], al, y);
        }
        const int jq = row / a.G, hq = h * a.G + row - jq * a.G;
        if (fix) {                            // values that were not finite and that this row does see
          for (int t = max(S - A + 1, begin); t <= min(S - A + jq, end - 1); ++t) {
            const int lb = t / a.BS, ph = lb < a.MB ? table[lb] : -1;
            if (ph < 0 || ph >= a.NB) continue;
            const char* p = kv + a.kv_stride_kv * es + int64_t(ph) * stride_b + int64_t(t - lb * a.BS) * stride_s;
            float f;
            if constexpr (QUANT) {
              f = static_cast<uint8_t>(p[a.Hkv * D + (h * D + d) / 32]) == 255 ? __int_as_float(0x7fffffff) : 0.0f;
            } else {
              const uint16_t u = reinterpret_cast<const uint16_t*>(p)[int64_t(h) * a.kv_stride_h + d];
              f = BF16 ? __uint_as_float(uint32_t(u) << 16) : __half2float(__ushort_as_half(u));
            }
            if (!isfinite(f)) y += f;
          }
        }
        if (whole) {
          const int64_t qt = int64_t(a0) + jq;
          static_cast<uint16_t*>(a.out)[qt * a.out_stride_t + int64_t(hq) * a.out_stride_h + d] =
              uint16_t(pack2<BF16>(L == 0.0f ? 0.0f : y / L, 0.0f));
          if (d == 0)
            a.lse[qt * a.lse_stride_t + hq] = L == 0.0f ? ninf : (M == ninf ? L : (M + log2f(L)) * 0.69314718055994531f);
        } else {
          ps.out(cta, ps_slot)[int64_t(row) * D + d] = y;
          if (d == 0) reinterpret_cast<float2*>(ps.ml(cta, ps_slot, D))[row] = make_float2(M, L);
        }
      }
      if (!whole && t0 == 0 && threadIdx.x == 0) {
        Desc ds = {};
        ds.valid = 1;
        ds.r = r;
        ds.h = h;
        ds.ntok = A;
        ds.S = S;
        ds.A = A;
        ds.a0 = a0;
        ds.end = first + nt;
        ds.total = sched.share.total;
        ps.desc[cta] = ds;
      }
      __syncthreads();                        // the rings are written again
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
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  k<<<grid, chunk::few::kThreads, bytes, st>>>(a);
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
