// Reading rows of the 4-bit paged cache back (the row: quant_row.cuh; rotary.cu writes them).
//
// Bound by memory: per value 17 / 32 bytes of the cache and 2 of 16-bit rows.  Eight lanes per (token, layer,
// plane, head): lane p takes the run of bytes that holds values 4 p .. 4 p + 3 of every group of 32 (one load for
// head sizes 64 and 128) and writes four values per group, 64 bytes of 16-bit values from the eight lanes
// together.  A warp takes kRun passes of four heads of one token, whose session and slot it finds once, plane by plane.
//
// Measured (8 heads of 128, bf16): 8 x 1088 tokens take 21 to 23 us per two layers (90 MB, 4.1 TB/s, 0.63 of the measured copy rate).
// No resource is full: 68 % of the issue slots, 43 % of the logic pipe, 42 % of the warps, which wait most for their reads (the conversions,
// one instruction per two values at half rate, come after).
#include <type_traits>

#include "kernels.cuh"
#include "quant_row.cuh"

namespace actkv {

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 8;

// The slot of packed token t (one per warp), as an offset within a plane; -1 when no session's or (flagged) not held.
__device__ __forceinline__ int64_t slot_of(const QuantMoveArgs& a, int t, int lane) {
  const int r = session_of(a.tok_off, a.R, t, lane);
  if (r >= a.R) return -1;
  const int pos = a.seq_used[r] - (a.tok_off[r + 1] - t);
  const int lb = pos / a.BS;
  const int phys = pos >= 0 && lb < a.MB ? a.block_table[r * a.bt_stride_r + lb] : -1;
  if (phys < 0 || phys >= a.NB) {
    if (lane == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
    return -1;
  }
  return int64_t(phys) * a.rows_stride_b + int64_t(pos - lb * a.BS) * a.rows_stride_s;
}

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};
template <typename T>
__device__ __forceinline__ void store4(T* p, const Four<T>& y, bool vec) {
  if (vec) {
    *reinterpret_cast<Four<T>*>(p) = y;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = y.v[k];
  }
}

// G: groups of a head, 2 to 4 (0: any number, one at a time).  What a lane reads of a row:
template <int G>
struct Raw {
  uint32_t w[(G + 1) / 2], scales;       // (places of groups that there are not: an ordinary scale)
};
template <int G>
__device__ __forceinline__ Raw<G> load_raw(const uint8_t* at, const uint8_t* scale, bool vec) {
  Raw<G> r;
  if (vec && G == 4) {
    const uint2 x = __ldcs(reinterpret_cast<const uint2*>(at));
    r.w[0] = x.x;
    r.w[(G + 1) / 2 - 1] = x.y;
    r.scales = *reinterpret_cast<const uint32_t*>(scale);
  } else if (vec && G == 2) {
    r.w[0] = __ldcs(reinterpret_cast<const uint32_t*>(at));
    r.scales = *reinterpret_cast<const uint16_t*>(scale) | 0x7f7f0000u;
  } else {
    r.scales = G == 4 ? 0u : (G == 3 ? 0x7f000000u : 0x7f7f0000u);
#pragma unroll
    for (int k = 0; k < (G + 1) / 2; ++k) r.w[k] = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t two = vec ? uint32_t(reinterpret_cast<const uint16_t*>(at)[g]) : uint32_t(at[2 * g]) | uint32_t(at[2 * g + 1]) << 8;
      r.w[g / 2] |= two << (16 * (g & 1));
      r.scales |= uint32_t(scale[g]) << (8 * g);
    }
  }
  return r;
}
template <typename T, int G>
__device__ __forceinline__ void write(T* dst, const Raw<G>& r, bool vec) {
  if constexpr (sizeof(T) == 2) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    const bool plain = plain_scales4<BF16>(r.scales);
#pragma unroll
    for (int k = 0; k < (G + 1) / 2; ++k) {
      const uint32_t b0 = r.scales >> (16 * k) & 255u, b1 = r.scales >> (16 * k + 8) & 255u;
      uint32_t y[4];
      if (plain) {
        widen4<BF16>(r.w[k], plain_factor4(b0), plain_factor4(b1), y);
      } else {
        uint32_t z[4];
        widen4_any<BF16>(r.w[k], b0, y);
        widen4_any<BF16>(r.w[k], b1, z);
        y[2] = z[2];
        y[3] = z[3];
      }
      store4<T>(dst + 64 * k, reinterpret_cast<const Four<T>&>(y[0]), vec);
      if (2 * k + 1 < G) store4<T>(dst + 64 * k + 32, reinterpret_cast<const Four<T>&>(y[2]), vec);
    }
  } else {
#pragma unroll
    for (int k = 0; k < (G + 1) / 2; ++k) {
      uint32_t h[4];
      e2m1x8_f16(r.w[k], h[0], h[1], h[2], h[3]);
#pragma unroll
      for (int e = 0; e < 2 && 2 * k + e < G; ++e) {
        const float s = scale_of4(r.scales >> (16 * k + 8 * e) & 255u);
        const float2 lo = f16x2_f32(h[2 * e]), hi = f16x2_f32(h[2 * e + 1]);
        store4<T>(dst + 64 * k + 32 * e, Four<T>{lo.x * s, lo.y * s, hi.x * s, hi.y * s}, vec);
      }
    }
  }
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads) quant4_read_kernel(const __grid_constant__ QuantMoveArgs a, int runs) {
  const int lane = threadIdx.x & 31, p = lane & 7;
  const int groups = G ? G : a.D / 32, nb = (a.Hkv + 3) / 4, passes = a.planes * nb;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  for (int64_t x = warp; x < int64_t(a.T) * runs; x += nwarps) {
    const int t = x >> 31 ? int(x / runs) : int(uint32_t(x) / uint32_t(runs)), first = int(x - int64_t(t) * runs) * kRun;
    const int64_t slot = slot_of(a, t, lane);
    if (slot < 0) continue;
    int n = min(kRun, passes - first), lp = first / nb, hb = first - lp * nb;
    while (n > 0) {                           // the passes of one plane
      const int m = min(n, nb - hb), h = 4 * hb + (lane >> 3), pl = a.both ? lp & 1 : a.only, l = a.both ? lp >> 1 : lp;
      const int64_t step = 4 * a.ext_stride_h[pl];
      T* dst = static_cast<T*>(pl ? a.v : a.k) + (int64_t(l) * a.ext_stride_l[pl] + int64_t(t) * a.ext_stride_t[pl] +
                                                  int64_t(h) * a.ext_stride_h[pl] + 4 * p);
      const uint8_t* row = a.rows + int64_t(l) * a.rows_stride_l + int64_t(pl) * a.rows_stride_kv + slot;
      const uint8_t* at = row + h * (a.D / 2) + 2 * groups * p;
      const uint8_t* scale = row + a.Hkv * (a.D / 2) + h * groups;
      const int live = a.Hkv - h;             // heads from this lane's on
      if constexpr (G > 0) {
        constexpr int kAhead = 4;
#pragma unroll 1
        for (int i = 0; i < m; i += kAhead, dst += kAhead * step, at += kAhead * 4 * (G * 16), scale += kAhead * 4 * G) {
          Raw<G> raw[kAhead];
#pragma unroll
          for (int e = 0; e < kAhead; ++e)
            if (i + e < m && 4 * (i + e) < live) raw[e] = load_raw<G>(at + e * 4 * (G * 16), scale + e * 4 * G, a.vec_rows);
#pragma unroll
          for (int e = 0; e < kAhead; ++e)
            if (i + e < m && 4 * (i + e) < live) write<T, G>(dst + e * step, raw[e], a.vec);
        }
      } else {
        for (int i = 0; i < m && 4 * i < live; ++i, dst += step, at += 2 * a.D, scale += 4 * groups)
          for (int g = 0; g < groups; ++g) {
            const float2 lo = f16x2_f32(e2m1x2_f16(at[2 * g])), hi = f16x2_f32(e2m1x2_f16(at[2 * g + 1]));
            const float s = scale_of4(scale[g]);
            store4<T>(dst + 32 * g, Four<T>{from_f32<T>(lo.x * s), from_f32<T>(lo.y * s), from_f32<T>(hi.x * s), from_f32<T>(hi.y * s)}, a.vec);
          }
      }
      n -= m;
      hb = 0;
      ++lp;
    }
  }
}

template <typename T>
cudaError_t launch(const QuantMoveArgs& a, cudaStream_t st) {
  const int runs = (a.planes * ((a.Hkv + 3) / 4) + kRun - 1) / kRun;
  const int64_t ctas = (int64_t(a.T) * runs + kThreads / 32 - 1) / (kThreads / 32);
  const int grid = int(ctas < (1 << 20) ? ctas : (1 << 20));
  if (grid <= 0) return cudaSuccess;
  if (a.D == 128) quant4_read_kernel<T, 4><<<grid, kThreads, 0, st>>>(a, runs);
  else if (a.D == 96) quant4_read_kernel<T, 3><<<grid, kThreads, 0, st>>>(a, runs);
  else if (a.D == 64) quant4_read_kernel<T, 2><<<grid, kThreads, 0, st>>>(a, runs);
  else quant4_read_kernel<T, 0><<<grid, kThreads, 0, st>>>(a, runs);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quant4_read(const QuantMoveArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ACTKV_BF16) return launch<__nv_bfloat16>(a, st);
  if (dtype == ACTKV_F16) return launch<__half>(a, st);
  return launch<float>(a, st);
}

}  // namespace actkv
