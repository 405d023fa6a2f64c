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
// warp that works on the token, from L2.  A warp takes a run of one token: where the type stays, items of 16
// values (two pieces of 8 that turn together: 16-byte loads), the same dims for every item of a lane, so that sines
// and cosines stay in registers; for rows, eight lanes per (layer, plane, head), lane p holding values 4 p .. 4 p + 3 of
// every group of 32, which is what the 4-bit row keeps together, and a group's maximum is three shuffles.
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
  if (r >= a.R || (a.ok && !a.ok[r])) return k;
  if (a.rot) {
    const int p = a.positions[t];
    if (p < 0 || p >= a.P) {
      if (lane == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
      return k;
    }
    angles = a.angles + int64_t(p) * a.angles_stride;
  }
  k.live = true;
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

// a / b for a small unsigned a: a shift where b is a power of two.
struct Divisor {
  int b, shift;
  __device__ __forceinline__ explicit Divisor(int n) {
    b = n;
    shift = (n & (n - 1)) == 0 ? __ffs(n) - 1 : -1;
  }
  __device__ __forceinline__ int operator()(int a) const { return shift >= 0 ? a >> shift : a / b; }
};

// Which array, layer and head a row of a token is; heads: q's, then k's, then v's.
struct Row {
  int which, l, h;
};

// ------------------------------------------------------------------------------ the type stays
// An item is 16 values: pieces at dims d0 and d1 that turn together.
struct Item {
  int d0, d1, i;             // i: the pair of the first value, -1: they stay
};
__device__ __forceinline__ Item item_of(const RotateArgs& a, int j) {
  const int turned = a.rot / 16;
  if (j >= turned) return {16 * j, 16 * j + 8, -1};
  if (a.pairs) return {16 * j, 16 * j + 8, 8 * j};
  return {8 * j, 8 * j + a.rot / 2, 8 * j};
}

// Items [first, first + 32 N) of token t.  SAME: the items of a head (`per`) divide 32, so a lane's dims are the
// same in all of its items.
template <typename T, int N, bool SAME>
__device__ __forceinline__ void same_type(const RotateArgs& a, int t, int first, int items, int heads, int per,
                                          const Token& tok, const float* angles, int lane) {
  using P8 = Piece<T, 8>;
  const Divisor by_per(per), by_heads(heads);
  float c[8], s[8];
  auto take = [&](int i) {
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      *reinterpret_cast<float4*>(c + k) = __ldg(reinterpret_cast<const float4*>(angles + i + k));
      *reinterpret_cast<float4*>(s + k) = __ldg(reinterpret_cast<const float4*>(angles + a.rot / 2 + i + k));
    }
  };
  if constexpr (SAME) {
    const int f = first + lane, i = item_of(a, f - by_per(f) * per).i;
    if (i >= 0) take(i);
  }
  P8 x[N], y[N];
  Row row[N];
  Item it[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int f = first + n * 32 + lane;
    row[n].which = -1;
    if (f >= items) continue;
    const int hr = by_per(f);
    it[n] = item_of(a, f - hr * per);
    const int l = by_heads(hr), h = hr - l * heads;
    row[n] = h < a.Hq ? Row{0, l, h} : (h < a.Hq + a.Hkv ? Row{1, l, h - a.Hq} : Row{2, l, h - a.Hq - a.Hkv});
    const int w = row[n].which;
    const T* p = static_cast<const T*>(a.in[w]) + (int64_t(l) * a.in_l[w] + int64_t(t) * a.in_t[w] + int64_t(row[n].h) * a.in_h[w]);
    x[n] = load<T, 8>(p + it[n].d0, true);
    y[n] = load<T, 8>(p + it[n].d1, true);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (row[n].which < 0) continue;
    const int w = row[n].which;
    if (w < 2 && it[n].i >= 0) {
      if constexpr (!SAME) take(it[n].i);
      if (a.pairs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float u = to_f32(x[n].v[2 * i]), v = to_f32(x[n].v[2 * i + 1]), e = to_f32(y[n].v[2 * i]), f = to_f32(y[n].v[2 * i + 1]);
          turn(u, v, c[i], s[i]);
          turn(e, f, c[4 + i], s[4 + i]);
          x[n].v[2 * i] = narrow<T>(u);
          x[n].v[2 * i + 1] = narrow<T>(v);
          y[n].v[2 * i] = narrow<T>(e);
          y[n].v[2 * i + 1] = narrow<T>(f);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float u = to_f32(x[n].v[i]), v = to_f32(y[n].v[i]);
          turn(u, v, c[i], s[i]);
          x[n].v[i] = narrow<T>(u);
          y[n].v[i] = narrow<T>(v);
        }
      }
    }
    T* p;
    if (w == 0) {
      p = static_cast<T*>(a.q_out) + (int64_t(row[n].l) * a.out_l + int64_t(t) * a.out_t + int64_t(row[n].h) * a.out_h);
    } else {
      if (tok.at < 0) continue;
      p = static_cast<T*>(a.cache) + (int64_t(row[n].l) * a.c_l + int64_t(w - 1) * a.c_kv + tok.at + int64_t(row[n].h) * a.c_h);
    }
    store<T, 8>(p + it[n].d0, x[n], true);
    store<T, 8>(p + it[n].d1, y[n], true);
  }
}

// Any sizes, strides and alignment: a lane takes a pair, or a value that stays.
template <typename T>
__device__ __forceinline__ void any_layout(const RotateArgs& a, int t, int first, int n, int units, int heads,
                                           const Token& tok, const float* angles, int lane) {
  const int half = a.rot / 2, per = half + a.D - a.rot;
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
// Rows [first, first + 4 n) of token t's 2 L Hkv (layer, head, plane) rows, eight lanes each.
// G: groups of a head (0: any number, a.D / 32, one at a time).
template <typename T, int BITS, int G>
__device__ __forceinline__ void quantise(const RotateArgs& a, int t, int first, int n, int rows, const Token& tok,
                                         const float* angles, int lane) {
  const int p = lane & 7, groups = G ? G : a.D / 32, half = a.rot / 2;
  const Divisor by_heads(a.Hkv);
  constexpr int kAt = G ? G : 1;              // groups at a time
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int f = first + 4 * i + (lane >> 3);
    const bool on = f < rows;                 // the shuffles below are the whole warp's
    const int lp = on ? by_heads(f) : 0, h = on ? f - lp * a.Hkv : 0, l = lp >> 1, w = 1 + (lp & 1);
    const T* src = static_cast<const T*>(a.in[w]) + (int64_t(l) * a.in_l[w] + int64_t(t) * a.in_t[w] + int64_t(h) * a.in_h[w]) + 4 * p;
    uint8_t* row = static_cast<uint8_t*>(a.cache) + (int64_t(l) * a.c_l + int64_t(w - 1) * a.c_kv + tok.at);
    uint8_t* vals = row + h * (a.D * BITS / 8);
    uint8_t* scales = row + a.Hkv * (a.D * BITS / 8) + h * groups;
    const bool turns = on && w == 1 && a.rot > 0;
#pragma unroll 1
    for (int g0 = 0; g0 < groups; g0 += kAt) {
      Piece<T, 4> raw[kAt], other[kAt];
#pragma unroll
      for (int g = 0; g < kAt; ++g)
        if (on) raw[g] = load<T, 4>(src + 32 * (g0 + g), a.vec_in);
      // the values that turn with them, when those are not in this lane (all of a head's dims in halves: they are)
      const bool inside = G > 1 && a.rot == a.D && a.vec_in;
      if (turns && !a.pairs && !inside) {
#pragma unroll
        for (int g = 0; g < kAt; ++g) {
          const int d = 32 * (g0 + g) + 4 * p;
          if (d < a.rot) other[g] = load<T, 4>(src + 32 * (g0 + g) + (d < half ? half : -half), a.vec_in);
        }
      }
      float x[kAt][4];
#pragma unroll
      for (int g = 0; g < kAt; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k) x[g][k] = on ? to_f32(raw[g].v[k]) : 0.0f;
      if (turns && a.pairs) {
#pragma unroll
        for (int g = 0; g < kAt; ++g) {
          const int d = 32 * (g0 + g) + 4 * p;
          if (d >= a.rot) continue;
          turn(x[g][0], x[g][1], __ldg(angles + d / 2), __ldg(angles + half + d / 2));
          turn(x[g][2], x[g][3], __ldg(angles + d / 2 + 1), __ldg(angles + half + d / 2 + 1));
        }
      } else if (turns && inside) {
#pragma unroll
        for (int g = 0; g < kAt / 2; ++g) {
          const float4 c = __ldg(reinterpret_cast<const float4*>(angles + 32 * g + 4 * p));
          const float4 s = __ldg(reinterpret_cast<const float4*>(angles + half + 32 * g + 4 * p));
          turn(x[g][0], x[g + kAt / 2][0], c.x, s.x);
          turn(x[g][1], x[g + kAt / 2][1], c.y, s.y);
          turn(x[g][2], x[g + kAt / 2][2], c.z, s.z);
          turn(x[g][3], x[g + kAt / 2][3], c.w, s.w);
        }
      } else if (turns) {
#pragma unroll
        for (int g = 0; g < kAt; ++g) {
          const int d = 32 * (g0 + g) + 4 * p;
          if (d >= a.rot) continue;
          const bool low = d < half;
          const float* at = angles + (low ? d : d - half);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float u = low ? x[g][k] : to_f32(other[g].v[k]), v = low ? to_f32(other[g].v[k]) : x[g][k];
            turn(u, v, __ldg(at + k), __ldg(at + half + k));
            x[g][k] = low ? u : v;
          }
        }
      }
      uint32_t packed[kAt], bytes = 0;
#pragma unroll
      for (int g = 0; g < kAt; ++g) {
        // without the sign, floats order as their bits do, NaN above all
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, __float_as_uint(x[g][k]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < 8; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t b = BITS == 4 ? scale_byte4(top) : scale_byte(top);
        const float inv = inverse_scale(b == 255u ? 0u : b);
        uint32_t u;
        if constexpr (BITS == 4)
          u = f32_e2m1x4(x[g][0] * inv, x[g][1] * inv, x[g][2] * inv, x[g][3] * inv);
        else
          u = (f32_e4m3x2(x[g][0] * inv, x[g][1] * inv) & 0xffffu) | f32_e4m3x2(x[g][2] * inv, x[g][3] * inv) << 16;
        packed[g] = b == 255u ? 0u : u;
        bytes |= b << (8 * g);
      }
      if (!on) continue;
      if constexpr (BITS == 8) {
#pragma unroll
        for (int g = 0; g < kAt; ++g) {
          uint8_t* dst = vals + 32 * (g0 + g) + 4 * p;
          if (a.vec_out) *reinterpret_cast<uint32_t*>(dst) = packed[g];
          else
            for (int k = 0; k < 4; ++k) dst[k] = uint8_t(packed[g] >> (8 * k));
        }
      } else {
        uint8_t* dst = vals + 2 * groups * p + 2 * g0;
        if (G == 4 && a.vec_out) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0] | packed[kAt > 1 ? 1 : 0] << 16,
                                                      packed[kAt > 2 ? 2 : 0] | packed[kAt > 3 ? 3 : 0] << 16);
        } else if (G == 2 && a.vec_out) {
          *reinterpret_cast<uint32_t*>(dst) = packed[0] | packed[kAt > 1 ? 1 : 0] << 16;
        } else {
#pragma unroll
          for (int g = 0; g < kAt; ++g) {
            dst[2 * g] = uint8_t(packed[g]);
            dst[2 * g + 1] = uint8_t(packed[g] >> 8);
          }
        }
      }
      if (p == 0) {
        if (G == 4 && a.vec_out) *reinterpret_cast<uint32_t*>(scales) = bytes;
        else
#pragma unroll
          for (int g = 0; g < kAt; ++g) scales[g0 + g] = uint8_t(bytes >> (8 * g));
      }
    }
  }
}

// ------------------------------------------------------------------------------ the kernel
// A token's work in runs of 32 N items (q's, and with BITS 0 also k's and v's), then runs of 4 N rows to
// quantise, a run per warp.
template <typename T, int BITS, int G, int N, bool VEC>
__global__ void __launch_bounds__(kThreads) rotate_write_kernel(const __grid_constant__ RotateArgs a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.Hq + (BITS == 0 ? 2 * a.Hkv : 0);
  const int per = VEC ? a.D / 16 : a.rot / 2 + a.D - a.rot;  // items of a head
  const int items = a.L * heads * per, rows = BITS == 0 ? 0 : 2 * a.L * a.Hkv;
  const int item_runs = (items + 32 * N - 1) / (32 * N), runs = item_runs + (rows + 4 * N - 1) / (4 * N);
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const bool same = VEC && 32 % per == 0;
  for (int64_t w = warp; w < int64_t(a.T) * runs; w += nwarps) {
    const int t = int(w / runs), run = int(w - int64_t(t) * runs);
    const float* angles = nullptr;
    const Token tok = find(a, t, lane, angles);
    if (!tok.live) continue;
    if (run < item_runs) {
      if constexpr (VEC) {
        if (same) same_type<T, N, true>(a, t, run * 32 * N, items, heads, per, tok, angles, lane);
        else same_type<T, N, false>(a, t, run * 32 * N, items, heads, per, tok, angles, lane);
      } else {
        any_layout<T>(a, t, run * 32 * N, 32 * N, items, heads, tok, angles, lane);
      }
    } else if constexpr (BITS != 0) {
      if (tok.at >= 0) quantise<T, BITS, G>(a, t, (run - item_runs) * 4 * N, N, rows, tok, angles, lane);
    }
  }
}

template <typename T, int BITS, int G, int N, bool VEC>
cudaError_t launch(const RotateArgs& a, int64_t warps, cudaStream_t st) {
  const int64_t ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
  rotate_write_kernel<T, BITS, G, N, VEC><<<unsigned(ctas < (1 << 20) ? ctas : (1 << 20)), kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int BITS, int G>
cudaError_t launch_bits(const RotateArgs& a, cudaStream_t st) {
  // whole pieces of 8 values, with the rotation's ends on them, in q (and in the cache where its type stays)
  const bool vec = a.vec_in && (BITS != 0 || a.vec_out) && a.D % 16 == 0 && a.rot % 16 == 0;
  const int heads = a.Hq + (BITS == 0 ? 2 * a.Hkv : 0), per = vec ? a.D / 16 : a.rot / 2 + a.D - a.rot;
  const int64_t items = int64_t(a.L) * heads * per, rows = BITS == 0 ? 0 : int64_t(2) * a.L * a.Hkv;
  auto warps = [&](int n) { return int64_t(a.T) * ((items + 32 * n - 1) / (32 * n) + (rows + 4 * n - 1) / (4 * n)); };
  if (warps(1) == 0) return cudaSuccess;
  // several items per lane hide a call's latency, fewer give a small call more warps
  const bool few = warps(4) < int64_t(device_sm_count()) * 8;
  if (!vec) return few ? launch<T, BITS, G, 1, false>(a, warps(1), st) : launch<T, BITS, G, 4, false>(a, warps(4), st);
  return few ? launch<T, BITS, G, 1, true>(a, warps(1), st) : launch<T, BITS, G, 4, true>(a, warps(4), st);
}

template <typename T>
cudaError_t launch_type(const RotateArgs& a, cudaStream_t st) {
  if (a.bits == 0) return launch_bits<T, 0, 0>(a, st);
  if (a.bits == 8) return a.D == 128 ? launch_bits<T, 8, 4>(a, st) : launch_bits<T, 8, 0>(a, st);
  return a.D == 128 ? launch_bits<T, 4, 4>(a, st) : (a.D == 64 ? launch_bits<T, 4, 2>(a, st) : launch_bits<T, 4, 0>(a, st));
}

}  // namespace

cudaError_t launch_rotate_write(const RotateArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ACTKV_BF16) return launch_type<__nv_bfloat16>(a, st);
  if (dtype == ACTKV_F16) return launch_type<__half>(a, st);
  return launch_type<float>(a, st);
}

}  // namespace actkv
