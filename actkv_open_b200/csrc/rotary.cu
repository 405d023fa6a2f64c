// New tokens on their way into a paged cache: the position rotation of their queries and keys, and keys and
// values written into the cache, as they are (the cache has their type) or quantised into 8- or 4-bit rows
// (quant_row.cuh), every layer in one launch.  Without a rotation it is the writer of the 4-bit rows.
//
// With c, s the cosine and sine of position * frequency i, (x, y) becomes (x c - y s, y c + x s): dims (i, i + rot / 2)
// or (2 i, 2 i + 1) of a head, dims from rot on stay as they are.  Each product and sum is rounded by itself, in
// 32 bits, then the result once to the cache's type: no fused multiply-add, whose one rounding less would depend on
// which of the two products it takes, so that rows quantised here are those of the plain formula bit for bit.
//
// Memory bounds it: every value is read and written once, and the table's row of a token (8 bytes per pair) once per
// warp that works on the token, from L2.  A warp takes a run of one token's passes:
//   where the type stays, a pass is 16 values per lane (two pieces of 8 that turn together: 16-byte accesses; pieces of 4
//     where the rotation ends on no multiple of 16) of as many heads as 32 lanes hold; a lane's dims are the same in every
//     pass, so its sines and cosines stay in registers;
//   into rows, a pass is four heads of a plane, eight lanes each, lane p holding values 4 p .. 4 p + 3 of every group of 32, which
//     is what the 4-bit row keeps together, and a group's maximum is three shuffles (of two groups at once where the
//     values are 16-bit and do not turn).
//
// Measured (32 query over 8 KV heads of 128, bf16): 8 x 1088 tokens, 8 layers, 16-bit cache (1.7 GB) 271 us, 0.97 of the measured copy
// rate; 32 tokens of one layer 3.7 us on the device.  4 x 8704 tokens, where bytes alone would take the time in brackets, us:
//   16-bit cache   all of 128 rotated 142 (131), half 145 (131), pairs 145 (131); 80 wide 110 (82), half of it 132 (82);
//                  96 wide 122 (99); 64 wide 83 (66)
//   4-bit rows, and read back   128 wide 229 (143), pairs 234 (143); 96 wide 215 (107); 64 wide 147 (71); unrotated, without
//                  queries, 128 wide 100 (55)
//   one KV head of 64 with 4 query heads   37 (8.5); into 4-bit rows unrotated, and back, 46 (3.4): a pass is one token's heads, so
//                  most lanes have nothing to do
// Into rows, unrotated: 299 instructions of a warp per 512 values, 63 % of the issue slots and of the logic pipe; the rest waits for
// memory with 40 % of the warps.  Rotated (336 per 512, 124 registers, 22 % of the warps): 45 % of either, no resource near its end.
// Head size 96 rotated spills 72 bytes (its partner from memory), the 16-bit rotation 32.
// Runs of 16 passes instead of 1: the token, its session and its angles are found once (8 x 1088 x 8 layers 998 to 285 us with
// angles in registers).
#include "kernels.cuh"
#include "quant_row.cuh"

namespace actkv {

namespace {

constexpr int kThreads = 128;

// Of a token: its session (R: none's), its position when the table has it, and its place in the cache.
struct Token {
  bool live;                 // a session's, at a position that the table has
  int64_t at;                // offset within a plane of the cache; -1: the block table does not hold it
};

// One token per warp.
__device__ __forceinline__ Token find(const RotateArgs& a, int t, int lane, const float*& angles) {
  Token k{false, -1};
  const int r = session_of(a.tok_off, a.R, t, lane);
  if (r >= a.R) return k;
  if (a.rot) {
    const int p = a.positions[t];
    if (p < 0 || p >= a.P) {
      if (lane == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
      return k;
    }
    angles = a.angles + int64_t(p) * a.angles_stride;
  }
  k.live = true;
  if (a.ok && !a.ok[r]) return k;             // no room: its queries turn, its rows go nowhere
  const int pos = a.seq_used[r] - (a.tok_off[r + 1] - t);
  const int lb = pos / a.BS;
  const int phys = pos >= 0 && lb < a.MB ? a.block_table[r * a.bt_stride_r + lb] : -1;
  if (phys < 0 || phys >= a.NB) {
    if (lane == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
    return k;
  }
  k.at = int64_t(phys) * a.c_b + int64_t(pos - lb * a.BS) * a.c_s;
  return k;
}

// (Scalar operations: packed 32-bit products and sums give other digits, they are fused on the way to machine code.)
__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
  const float u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
  y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
  x = u;
}

// N values as they are in memory.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Piece {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Piece<T, N> load(const T* p, bool vec) {
  Piece<T, N> r;
  if (vec) {
    r = *reinterpret_cast<const Piece<T, N>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = p[i];
  }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const Piece<T, N>& r, bool vec) {
  if (vec) {
    *reinterpret_cast<Piece<T, N>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = r.v[i];
  }
}
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ void narrow2(float2 x, float* p) {
  p[0] = x.x;
  p[1] = x.y;
}
__device__ __forceinline__ void narrow2(float2 x, __half* p) { *reinterpret_cast<__half2*>(p) = __float22half2_rn(x); }
__device__ __forceinline__ void narrow2(float2 x, __nv_bfloat16* p) { *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(x); }

// ------------------------------------------------------------------------------ the type stays
// A lane's 2 N values of a head: pieces at dims d0 and d1 that turn together; i: the pair of the first value, -1: they stay.
struct Item {
  int d0, d1, i;
};
template <int N>
__device__ __forceinline__ Item item_of(const RotateArgs& a, int j) {
  if (2 * N * j >= a.rot) return {2 * N * j, 2 * N * j + N, -1};
  if (a.pairs) return {2 * N * j, 2 * N * j + N, N * j};
  return {N * j, N * j + a.rot / 2, N * j};
}

// Neighbouring pairs of a piece, from pair k of the lane's on.
template <typename T, int N>
__device__ __forceinline__ void turn_pairs(Piece<T, N>& p, const float* c, const float* s) {
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    float u = to_f32(p.v[k]), v = to_f32(p.v[k + 1]);
    turn(u, v, c[k / 2], s[k / 2]);
    p.v[k] = narrow<T>(u);
    p.v[k + 1] = narrow<T>(v);
  }
}

// Passes [first, first + n) of token t: heads in blocks of as many as 32 lanes hold, of q, then k, then v, layer by layer.
template <typename T, int N, bool KV>
__device__ __forceinline__ void same_type(const RotateArgs& a, int t, int first, int n, const Token& tok,
                                          const float* angles, int lane) {
  using P = Piece<T, N>;
  const int per = a.D / (2 * N), block = 32 / per;          // lanes per head, heads per pass
  const int hl = lane / per, j = lane - hl * per;
  const Item it = item_of<N>(a, j);
  float c[N], s[N];
  if (it.i >= 0) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      *reinterpret_cast<float4*>(c + k) = __ldg(reinterpret_cast<const float4*>(angles + it.i + k));
      *reinterpret_cast<float4*>(s + k) = __ldg(reinterpret_cast<const float4*>(angles + a.rot / 2 + it.i + k));
    }
  }
  const int nq = (a.Hq + block - 1) / block, nk = KV ? (a.Hkv + block - 1) / block : 0;
  int l = first / (nq + 2 * nk), hb = first - l * (nq + 2 * nk), w = 0;
  if (KV && hb >= nq) {
    hb -= nq;
    w = 1;
    if (hb >= nk) {
      hb -= nk;
      w = 2;
    }
  }
  constexpr int kAhead = 2;                   // passes in flight
  while (n > 0) {                             // the passes of one array and layer
    const int heads = w == 0 ? a.Hq : a.Hkv, m = min(n, (w == 0 ? nq : nk) - hb), h0 = hb * block + hl;
    const T* src = static_cast<const T*>(a.in[w]) + (int64_t(l) * a.in_l[w] + int64_t(t) * a.in_t[w] + int64_t(h0) * a.in_h[w]);
    const int64_t out_h = w == 0 ? a.out_h : a.c_h;
    T* dst = w == 0 ? static_cast<T*>(a.q_out) + (int64_t(l) * a.out_l + int64_t(t) * a.out_t + int64_t(h0) * out_h)
                    : static_cast<T*>(a.cache) + (int64_t(l) * a.c_l + int64_t(w - 1) * a.c_kv + tok.at + int64_t(h0) * out_h);
    const int64_t src_step = block * a.in_h[w], dst_step = block * out_h;
    const bool turns = w < 2 && it.i >= 0;
    const int live = hl < block && (w == 0 || tok.at >= 0) ? heads - h0 : 0;      // heads from this lane's on
#pragma unroll 1
    for (int i = 0; i < m; i += kAhead, src += kAhead * src_step, dst += kAhead * dst_step) {
      P x[kAhead], y[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e)
        if (i + e < m && (i + e) * block < live) {
          x[e] = load<T, N>(src + e * src_step + it.d0, true);
          y[e] = load<T, N>(src + e * src_step + it.d1, true);
        }
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        if (i + e >= m || (i + e) * block >= live) continue;
        if (turns) {
          if (a.pairs) {
            turn_pairs<T, N>(x[e], c, s);
            turn_pairs<T, N>(y[e], c + N / 2, s + N / 2);
          } else {
#pragma unroll
            for (int k = 0; k < N; k += 2) {
              float2 u = make_float2(to_f32(x[e].v[k]), to_f32(x[e].v[k + 1]));
              float2 v = make_float2(to_f32(y[e].v[k]), to_f32(y[e].v[k + 1]));
              turn(u.x, v.x, c[k], s[k]);
              turn(u.y, v.y, c[k + 1], s[k + 1]);
              narrow2(u, x[e].v + k);
              narrow2(v, y[e].v + k);
            }
          }
        }
        store<T, N>(dst + e * dst_step + it.d0, x[e], true);
        store<T, N>(dst + e * dst_step + it.d1, y[e], true);
      }
    }
    n -= m;
    hb = 0;
    if (!KV || ++w == 3) {
      w = nq > 0 ? 0 : 1;
      ++l;
    }
  }
}

// Any sizes, strides and alignment: a lane takes a pair, or a value that stays.
template <typename T>
__device__ __forceinline__ void any_layout(const RotateArgs& a, int t, int first, int n, const Token& tok,
                                           const float* angles, int lane) {
  const int half = a.rot / 2, per = half + a.D - a.rot;
  const int heads = a.Hq + (a.bits == 0 ? 2 * a.Hkv : 0), units = a.L * heads * per;
  for (int f = first + lane; f < min(first + n, units); f += 32) {
    const int hr = f / per, i = f - hr * per, l = hr / heads, hh = hr - l * heads;
    const int w = hh < a.Hq ? 0 : (hh < a.Hq + a.Hkv ? 1 : 2), h = hh - (w == 0 ? 0 : (w == 1 ? a.Hq : a.Hq + a.Hkv));
    if (w > 0 && tok.at < 0) continue;
    const T* p = static_cast<const T*>(a.in[w]) + (int64_t(l) * a.in_l[w] + int64_t(t) * a.in_t[w] + int64_t(h) * a.in_h[w]);
    T* o = w == 0 ? static_cast<T*>(a.q_out) + (int64_t(l) * a.out_l + int64_t(t) * a.out_t + int64_t(h) * a.out_h)
                  : static_cast<T*>(a.cache) + (int64_t(l) * a.c_l + int64_t(w - 1) * a.c_kv + tok.at + int64_t(h) * a.c_h);
    if (i >= half) {
      o[a.rot + i - half] = p[a.rot + i - half];
      continue;
    }
    const int d0 = a.pairs ? 2 * i : i, d1 = a.pairs ? 2 * i + 1 : i + half;
    T x = p[d0], y = p[d1];
    if (w < 2) {
      float u = to_f32(x), v = to_f32(y);
      turn(u, v, angles[i], angles[half + i]);
      x = narrow<T>(u);
      y = narrow<T>(v);
    }
    o[d0] = x;
    o[d1] = y;
  }
}

// ------------------------------------------------------------------------------ into 8- or 4-bit rows
__device__ __forceinline__ uint32_t max16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The bits of the largest magnitudes of N groups, four values of each per lane, over eight lanes.  Without the sign, floats
// order as their bits do, NaN above all.  Of 16-bit values two groups at a time.
template <typename T, int N>
__device__ __forceinline__ void tops(const Piece<T, 4> (&raw)[N], uint32_t (&top)[N]) {
#pragma unroll
  for (int g = 0; g < N; g += 2) {
    uint32_t m[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint2 w = reinterpret_cast<const uint2&>(raw[g + e < N ? g + e : g]);
      m[e] = max16x2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
    }
    uint32_t both = max16x2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
    for (int o = 1; o < 8; o *= 2) both = max16x2(both, __shfl_xor_sync(0xffffffffu, both, o));
    const uint16_t lo = uint16_t(both), hi = uint16_t(both >> 16);
    top[g] = __float_as_uint(to_f32(reinterpret_cast<const T&>(lo)));
    if (g + 1 < N) top[g + 1 < N ? g + 1 : g] = __float_as_uint(to_f32(reinterpret_cast<const T&>(hi)));
  }
}
template <int N>
__device__ __forceinline__ void tops(const float (&x)[N][4], uint32_t (&top)[N]) {
#pragma unroll
  for (int g = 0; g < N; ++g) {
    top[g] = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) top[g] = max(top[g], __float_as_uint(x[g][k]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 8; o *= 2) top[g] = max(top[g], __shfl_xor_sync(0xffffffffu, top[g], o));
  }
}

template <int BITS>
__device__ __forceinline__ uint32_t byte_of_top(uint32_t top) { return BITS == 4 ? scale_byte4(top) : scale_byte(top); }
template <int BITS, int N>
__device__ __forceinline__ uint32_t bytes_of_tops(const uint32_t (&top)[N]) {
  uint32_t bytes = 0;
#pragma unroll
  for (int g = 0; g < N; ++g) bytes |= byte_of_top<BITS>(top[g]) << (8 * g);
  return bytes;
}
// The scale bytes of N groups, byte g group g's, in all eight lanes (p: which of them).  Of 4 groups a lane goes on with
// half of what it has at each exchange, so that it ends with one group's maximum and makes one byte (8 x 1088 tokens x 8 layers
// into 4 bits and back 189 to 183 us; of 2 groups the choosing costs more than it saves, 12 prompts of head size 64 100 to 103).
template <int BITS, int N>
__device__ __forceinline__ uint32_t scale_bytes(const float (&x)[N][4], int p) {
  if constexpr (N == 4) {
    uint32_t m[N];
#pragma unroll
    for (int g = 0; g < N; ++g) {
      m[g] = __float_as_uint(x[g][0]) & 0x7fffffffu;
#pragma unroll
      for (int k = 1; k < 4; ++k) m[g] = max(m[g], __float_as_uint(x[g][k]) & 0x7fffffffu);
    }
    const bool one = p & 1, two = p & 2;
#pragma unroll
    for (int g = 0; g < 2; ++g) {             // groups 2 g + (p & 1)
      const uint32_t other = __shfl_xor_sync(0xffffffffu, one ? m[2 * g] : m[2 * g + 1], 1);
      m[g] = max(one ? m[2 * g + 1] : m[2 * g], other);
    }
    const uint32_t other = __shfl_xor_sync(0xffffffffu, two ? m[0] : m[1], 2);
    m[0] = max(two ? m[1] : m[0], other);     // group p & 3
    m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 4));
    uint32_t bytes = byte_of_top<BITS>(m[0]) << (8 * (p & 3));
#pragma unroll
    for (int o = 1; o < 4; o *= 2) bytes |= __shfl_xor_sync(0xffffffffu, bytes, o);
    return bytes;
  } else {
    uint32_t top[N];
    tops<N>(x, top);
    return bytes_of_tops<BITS>(top);
  }
}
// ... of 16-bit values as they are in memory
template <int BITS, typename T, int N>
__device__ __forceinline__ uint32_t scale_bytes(const Piece<T, 4> (&raw)[N], int p) {
  static_assert(sizeof(T) == 2);
  if constexpr (N == 4) {
    uint32_t m[2];                            // of two groups, the first in the low half
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      uint32_t w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint2 u = reinterpret_cast<const uint2&>(raw[g + e]);
        w[e] = max16x2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu);
      }
      m[g / 2] = max16x2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[0], w[1], 0x7632));
    }
    const uint32_t other = __shfl_xor_sync(0xffffffffu, p & 1 ? m[0] : m[1], 1);
    uint32_t most = max16x2(p & 1 ? m[1] : m[0], other);    // groups 2 (p & 1) on
    most = max16x2(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = max16x2(most, __shfl_xor_sync(0xffffffffu, most, 4));
    const int high = p >> 1 & 1;              // the lane's of the two
    const uint16_t top = uint16_t(most >> (16 * high));
    uint32_t bytes = byte_of_top<BITS>(__float_as_uint(to_f32(reinterpret_cast<const T&>(top)))) << (8 * (2 * (p & 1) + high));
#pragma unroll
    for (int o = 1; o < 4; o *= 2) bytes |= __shfl_xor_sync(0xffffffffu, bytes, o);
    return bytes;
  } else {
    uint32_t top[N];
    tops<T, N>(raw, top);
    return bytes_of_tops<BITS>(top);
  }
}
// Four values times a power of two.
__device__ __forceinline__ void scale4(float (&x)[4], float f) {
  asm("{\n\t.reg .b64 a, b, s;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\t"
      "mul.rn.f32x2 a, a, s;\n\tmul.rn.f32x2 b, b, s;\n\tmov.b64 {%0, %1}, a;\n\tmov.b64 {%2, %3}, b;\n\t}"
      : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3])
      : "f"(f));
}

// How keys turn on their way into rows: not at all; in halves a whole number of groups apart (1, or 2 of 4), so that the
// values that turn together are in one lane; in neighbouring pairs, which always are; or in any way, the other value of a
// pair fetched from memory.  In a lane, its angles stay in registers.
enum Turns { kStay, kInLane, kPairs, kAny };

// Passes [first, first + n) of token t, plane by plane (k's, then v's, of each layer): four heads each, eight lanes per head.
// G: groups of a head (0: any number, a.D / 32, one at a time).
template <typename T, int BITS, int G, Turns TURNS>
__device__ __forceinline__ void quantise(const RotateArgs& a, int t, int first, int n, const Token& tok,
                                         const float* angles, int lane) {
  const int p = lane & 7, groups = G ? G : a.D / 32, nb = (a.Hkv + 3) / 4;
  [[maybe_unused]] const int half = a.rot / 2;
  constexpr int kAt = G ? G : 1;              // groups at a time
  [[maybe_unused]] float c[kAt][2], s[kAt][2];              // in halves: 4 of group pair i in c[2 i], c[2 i + 1]
  [[maybe_unused]] const int apart = a.rot / 64;            // groups between the halves
  if constexpr (TURNS == kInLane) {
#pragma unroll
    for (int g = 0; g < kAt / 2; ++g)
      if (g < apart)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          c[2 * g + k / 2][k & 1] = __ldg(angles + 32 * g + 4 * p + k);
          s[2 * g + k / 2][k & 1] = __ldg(angles + half + 32 * g + 4 * p + k);
        }
  } else if constexpr (TURNS == kPairs) {
#pragma unroll
    for (int g = 0; g < kAt; ++g)
      if (32 * g + 4 * p < a.rot)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          c[g][k] = __ldg(angles + 16 * g + 2 * p + k);
          s[g][k] = __ldg(angles + half + 16 * g + 2 * p + k);
        }
  }
  // A lane's heads past the last are the last once more, not stored: the shuffles are the whole warp's.
  auto source = [&](int lp, int hb) -> const T* {
    const bool k = (lp & 1) == 0;
    return static_cast<const T*>(k ? a.in[1] : a.in[2]) +
           (int64_t(lp >> 1) * (k ? a.in_l[1] : a.in_l[2]) + int64_t(t) * (k ? a.in_t[1] : a.in_t[2]) +
            int64_t(min(4 * hb + (lane >> 3), a.Hkv - 1)) * (k ? a.in_h[1] : a.in_h[2])) + 4 * p;
  };
  int lp = first / nb, hb = first - lp * nb;  // the pass
  const T* src = source(lp, hb);
  Piece<T, 4> ahead[kAt];                     // the next step's values
#pragma unroll
  for (int g = 0; g < kAt; ++g) ahead[g] = load<T, 4>(src + 32 * g, a.vec_in);
  uint8_t* plane = static_cast<uint8_t*>(a.cache) + (int64_t(lp >> 1) * a.c_l + int64_t(lp & 1) * a.c_kv + tok.at);
#pragma unroll 1
  for (int i = 0, g0 = 0; i < n;) {
    Piece<T, 4> raw[kAt];
#pragma unroll
    for (int g = 0; g < kAt; ++g) raw[g] = ahead[g];
    // the step after this one
    const int this_lp = lp, this_hb = hb, this_g = g0;
    uint8_t* const this_plane = plane;
    [[maybe_unused]] const T* const this_src = src;
    g0 += kAt;
    if (g0 >= groups) {
      g0 = 0;
      ++i;
      if (++hb == nb) {
        hb = 0;
        ++lp;
        plane = static_cast<uint8_t*>(a.cache) + (int64_t(lp >> 1) * a.c_l + int64_t(lp & 1) * a.c_kv + tok.at);
        src = source(min(lp, 2 * a.L - 1), hb);
      } else if (4 * hb + 4 <= a.Hkv) {
        src += 4 * (lp & 1 ? a.in_h[2] : a.in_h[1]);
      } else {
        src = source(lp, hb);
      }
    }
    if (i < n) {
#pragma unroll
      for (int g = 0; g < kAt; ++g) ahead[g] = load<T, 4>(src + 32 * (g0 + g), a.vec_in);
    }
    const bool turns = TURNS != kStay && (this_lp & 1) == 0;
    float x[kAt][4];
#pragma unroll
    for (int g = 0; g < kAt; ++g)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[g][k] = to_f32(raw[g].v[k]);
    if (turns) {
      if constexpr (TURNS == kInLane) {
        auto both = [&](int g, int other, int at) {
#pragma unroll
          for (int k = 0; k < 4; ++k) turn(x[g][k], x[other][k], c[2 * at + k / 2][k & 1], s[2 * at + k / 2][k & 1]);
        };
        if (kAt == 2 || apart == 1) {
          both(0, kAt > 1 ? 1 : 0, 0);
        } else {
          both(0, kAt / 2, 0);
          both(kAt > 2 ? 1 : 0, kAt > 2 ? 3 : 0, kAt > 2 ? 1 : 0);
        }
      } else if constexpr (TURNS == kPairs) {
#pragma unroll
        for (int g = 0; g < kAt; ++g)
          if (32 * g + 4 * p < a.rot) {
            turn(x[g][0], x[g][1], c[g][0], s[g][0]);
            turn(x[g][2], x[g][3], c[g][1], s[g][1]);
          }
      } else {
#pragma unroll
        for (int g = 0; g < kAt; ++g) {
          const int d = 32 * (this_g + g) + 4 * p;
          if (d >= a.rot) continue;
          if (a.pairs) {
            turn(x[g][0], x[g][1], __ldg(angles + d / 2), __ldg(angles + half + d / 2));
            turn(x[g][2], x[g][3], __ldg(angles + d / 2 + 1), __ldg(angles + half + d / 2 + 1));
          } else {
            const bool low = d < half;
            const Piece<T, 4> other = load<T, 4>(this_src + 32 * (this_g + g) + (low ? half : -half), a.vec_in);
            const float* at = angles + (low ? d : d - half);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float u = low ? x[g][k] : to_f32(other.v[k]), v = low ? to_f32(other.v[k]) : x[g][k];
              turn(u, v, __ldg(at + k), __ldg(at + half + k));
              x[g][k] = low ? u : v;
            }
          }
        }
      }
    }
    uint32_t packed[kAt], bytes;
    if constexpr (sizeof(T) == 2) {
      if (turns) bytes = scale_bytes<BITS, kAt>(x, p);       // (the same for the whole warp)
      else bytes = scale_bytes<BITS, T, kAt>(raw, p);
    } else {
      bytes = scale_bytes<BITS, kAt>(x, p);
    }
#pragma unroll
    for (int g = 0; g < kAt; ++g) {
      scale4(x[g], inverse_scale(bytes >> (8 * g) & 255u));  // (anything for 255)
      if constexpr (BITS == 4) packed[g] = f32_e2m1x4(x[g][0], x[g][1], x[g][2], x[g][3]);
      else packed[g] = (f32_e4m3x2(x[g][0], x[g][1]) & 0xffffu) | f32_e4m3x2(x[g][2], x[g][3]) << 16;
    }
    if (__vcmpeq4(bytes, 0xffffffffu)) {      // (of groups that are not there the byte is 0)
#pragma unroll
      for (int g = 0; g < kAt; ++g)
        if ((bytes >> (8 * g) & 255u) == 255u) packed[g] = 0u;
    }
    const int h = 4 * this_hb + (lane >> 3);
    if (h >= a.Hkv) continue;
    uint8_t* vals = this_plane + h * (a.D * BITS / 8);
    uint8_t* scales = this_plane + a.Hkv * (a.D * BITS / 8) + h * groups + this_g;
    if constexpr (BITS == 8) {
#pragma unroll
      for (int g = 0; g < kAt; ++g) {
        uint8_t* dst = vals + 32 * (this_g + g) + 4 * p;
        if (a.vec_out) *reinterpret_cast<uint32_t*>(dst) = packed[g];
        else
          for (int k = 0; k < 4; ++k) dst[k] = uint8_t(packed[g] >> (8 * k));
      }
    } else {
      uint8_t* dst = vals + 2 * groups * p + 2 * this_g;
      if (G == 4 && a.vec_out) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(__byte_perm(packed[0], packed[kAt > 1 ? 1 : 0], 0x5410),
                                                    __byte_perm(packed[kAt > 2 ? 2 : 0], packed[kAt > 3 ? 3 : 0], 0x5410));
      } else if (G == 2 && a.vec_out) {
        *reinterpret_cast<uint32_t*>(dst) = __byte_perm(packed[0], packed[kAt > 1 ? 1 : 0], 0x5410);
      } else {
#pragma unroll
        for (int g = 0; g < kAt; ++g) {
          if (a.vec_out) {
            reinterpret_cast<uint16_t*>(dst)[g] = uint16_t(packed[g]);
          } else {
            dst[2 * g] = uint8_t(packed[g]);
            dst[2 * g + 1] = uint8_t(packed[g] >> 8);
          }
        }
      }
    }
    if (p == 0) {
      if (G == 4 && a.vec_out) *reinterpret_cast<uint32_t*>(scales) = bytes;
      else
#pragma unroll
        for (int g = 0; g < kAt; ++g) scales[g] = uint8_t(bytes >> (8 * g));
    }
  }
}

// ------------------------------------------------------------------------------ the kernel
// A token's work: passes of q (and where the type stays of k and v), then passes of rows to quantise, in runs of `run`
// passes of one kind, a run per warp.
template <typename T, int BITS, int G, Turns TURNS, int PIECE>
__global__ void __launch_bounds__(kThreads, BITS == 0 || TURNS == kStay ? 8 : (G == 4 ? 4 : 5))
    rotate_write_kernel(const __grid_constant__ RotateArgs a, int run, int item_passes, int item_runs, int runs) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int row_passes = BITS == 0 ? 0 : 2 * a.L * ((a.Hkv + 3) / 4);
  for (int64_t w = warp; w < int64_t(a.T) * runs; w += nwarps) {
    const int t = w >> 31 ? int(w / runs) : int(uint32_t(w) / uint32_t(runs)), which = int(w - int64_t(t) * runs);
    const float* angles = nullptr;
    const Token tok = find(a, t, lane, angles);
    if (!tok.live) continue;
    if (TURNS != kStay && which < item_runs) {
      const int first = which * run, n = min(run, item_passes - first);
      if constexpr (PIECE > 0) same_type<T, PIECE, BITS == 0>(a, t, first, n, tok, angles, lane);
      else any_layout<T>(a, t, first * 32, n * 32, tok, angles, lane);
    } else if constexpr (BITS != 0) {
      const int first = (which - item_runs) * run;
      if (tok.at >= 0) quantise<T, BITS, G, TURNS>(a, t, first, min(run, row_passes - first), tok, angles, lane);
    }
  }
}

template <typename T, int BITS, int G, Turns TURNS, int PIECE>
cudaError_t launch(const RotateArgs& a, cudaStream_t st) {
  const int block = PIECE ? 32 / (a.D / (2 * PIECE)) : 1;
  const int64_t items = TURNS == kStay ? 0 : PIECE
      ? int64_t(a.L) * ((a.Hq + block - 1) / block + (BITS == 0 ? 2 * ((a.Hkv + block - 1) / block) : 0))
      : (int64_t(a.L) * (a.Hq + (BITS == 0 ? 2 * a.Hkv : 0)) * (a.rot / 2 + a.D - a.rot) + 31) / 32;
  const int64_t rows = BITS == 0 ? 0 : int64_t(2) * a.L * ((a.Hkv + 3) / 4);
  auto runs = [&](int run) { return (items + run - 1) / run + (rows + run - 1) / run; };
  // long runs find a token once for more work, short ones give a small call more warps
  int run = 16;
  while (run > 1 && a.T * runs(run) < int64_t(device_sm_count()) * 16) run /= 2;
  const int64_t warps = a.T * runs(run), ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (ctas == 0) return cudaSuccess;
  rotate_write_kernel<T, BITS, G, TURNS, PIECE><<<unsigned(ctas < (1 << 20) ? ctas : (1 << 20)), kThreads, 0, st>>>(
      a, run, int(items), int((items + run - 1) / run), int(runs(run)));
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_same(const RotateArgs& a, cudaStream_t st) {
  const bool aligned = a.vec_in && a.vec_out;               // pieces with the rotation's ends on them, and a head in 32 lanes
  if (aligned && a.D % 16 == 0 && a.rot % 16 == 0 && a.D <= 512) return launch<T, 0, 0, kAny, 8>(a, st);
  if (aligned && a.D % 8 == 0 && a.rot % 8 == 0 && a.D <= 256) return launch<T, 0, 0, kAny, 4>(a, st);
  return launch<T, 0, 0, kAny, 0>(a, st);
}

template <typename T, int BITS>
cudaError_t launch_rows(const RotateArgs& all, cudaStream_t st) {
  RotateArgs a = all;
  // The rows' registers leave the queries, which only memory bounds, too few warps: large ones go first, in a launch of their
  // own (4 x 8704 tokens of 32 heads of 128, 143 million values, and back: 276 us in one launch, 229 in two; 8 x 1088 tokens, 36
  // million: 74 and 76; heads of 64, 71 million: 152 and 146; 18 million: 54 and 54).
  constexpr int64_t kApart = 1 << 26;
  if (a.rot > 0 && int64_t(a.T) * a.L * a.Hq * a.D >= kApart) {
    RotateArgs b = a;
    b.Hkv = b.bits = 0;
    b.vec_out = true;                         // (nothing of it goes into the cache)
    const cudaError_t e = launch_same<T>(b, st);
    if (e != cudaSuccess) return e;
    a.Hq = 0;
  }
  if constexpr (BITS == 4)
    if (a.rot == 0) {
      if (a.D == 128) return launch<T, 4, 4, kStay, 8>(a, st);
      if (a.D == 96) return launch<T, 4, 3, kStay, 8>(a, st);
      return a.D == 64 ? launch<T, 4, 2, kStay, 8>(a, st) : launch<T, 4, 0, kStay, 8>(a, st);
    }
  if (!a.vec_in || a.D % 16 || a.rot % 16 || a.D > 512) return launch<T, BITS, 0, kAny, 0>(a, st);
  if (a.D == 128) {
    if (a.pairs) return launch<T, BITS, 4, kPairs, 8>(a, st);
    if (a.rot == 128 || a.rot == 64) return launch<T, BITS, 4, kInLane, 8>(a, st);
  }
  if constexpr (BITS == 4) {
    if (a.D == 64 && a.pairs) return launch<T, 4, 2, kPairs, 8>(a, st);
    if (a.D == 64 && a.rot == 64) return launch<T, 4, 2, kInLane, 8>(a, st);
    if (a.D == 96) return launch<T, 4, 3, kAny, 8>(a, st);
  }
  return launch<T, BITS, 0, kAny, 8>(a, st);
}

template <typename T>
cudaError_t launch_type(const RotateArgs& a, cudaStream_t st) {
  return a.bits == 0 ? launch_same<T>(a, st) : (a.bits == 8 ? launch_rows<T, 8>(a, st) : launch_rows<T, 4>(a, st));
}

}  // namespace

cudaError_t launch_rotate_write(const RotateArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ACTKV_BF16) return launch_type<__nv_bfloat16>(a, st);
  if (dtype == ACTKV_F16) return launch_type<__half>(a, st);
  return launch_type<float>(a, st);
}

}  // namespace actkv
