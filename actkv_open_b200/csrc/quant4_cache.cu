// Reading rows of the 4-bit paged cache back (the row: quant_row.cuh; rotary.cu writes them).
//
// Bound by memory: per value 17 / 32 bytes of the cache and 2 of 16-bit rows.  Eight lanes per (token, layer,
// plane, head): lane p takes the run of bytes that holds values 4 p .. 4 p + 3 of every group of 32 (one load for
// head sizes 64 and 128) and writes four values per group, 64 bytes of 16-bit values from the eight lanes
// together.  A warp takes four such rows at a time, kPasses times, of one token, whose session and slot it finds once.
#include <type_traits>

#include "kernels.cuh"
#include "quant_row.cuh"

namespace actkv {

namespace {

constexpr int kThreads = 256;
constexpr int kPasses = 4;

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

// G: groups of a head (0: any number, one at a time).
template <typename T, int G>
__global__ void __launch_bounds__(kThreads) quant4_read_kernel(const __grid_constant__ QuantMoveArgs a) {
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  };
  auto narrow2 = [](float x, float y, T* p) {
    if constexpr (sizeof(T) == 4) {
      p[0] = x;
      p[1] = y;
    } else if constexpr (std::is_same<T, __half>::value) {   // past the range: the largest (NaN stays)
      *reinterpret_cast<__half2*>(p) = __hmin2_nan(__hmax2_nan(__floats2half2_rn(x, y), __float2half2_rn(-65504.0f)),
                                                   __float2half2_rn(65504.0f));
    } else {
      *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
    }
  };
  constexpr int kAt = G ? G : 1;
  const int lane = threadIdx.x & 31, p = lane & 7;
  const int groups = G ? G : a.D / 32, rows = a.planes * a.Hkv;
  const int runs = (rows + 4 * kPasses - 1) / (4 * kPasses);
  const int shift = (a.Hkv & (a.Hkv - 1)) == 0 ? __ffs(a.Hkv) - 1 : -1;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  int last = -1;
  int64_t slot = -1;
  for (int64_t w = warp; w < int64_t(a.T) * runs; w += nwarps) {
    const int t = int(w / runs), run = int(w - int64_t(t) * runs);
    if (t != last) slot = slot_of(a, t, lane);
    last = t;
    if (slot < 0) continue;
    for (int g0 = 0; g0 < groups; g0 += kAt) {
      T* ext[kPasses];
      uint32_t u[kPasses][(kAt + 1) / 2], sc[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int f = (run * kPasses + i) * 4 + (lane >> 3);
        ext[i] = nullptr;
        if (f >= rows) continue;
        const int lp = shift >= 0 ? f >> shift : f / a.Hkv, h = f - lp * a.Hkv;
        const int l = a.both ? lp >> 1 : lp, pl = a.both ? lp & 1 : a.only;
        ext[i] = static_cast<T*>(pl ? a.v : a.k) +
                 (int64_t(l) * a.ext_stride_l[pl] + int64_t(t) * a.ext_stride_t[pl] + int64_t(h) * a.ext_stride_h[pl] + 4 * p + 32 * g0);
        const uint8_t* row = a.rows + int64_t(l) * a.rows_stride_l + int64_t(pl) * a.rows_stride_kv + slot;
        const uint8_t* at = row + h * (a.D / 2) + 2 * groups * p + 2 * g0;
        const uint8_t* scale = row + a.Hkv * (a.D / 2) + h * groups + g0;
        if (G == 4 && a.vec_rows) {
          const uint2 x = __ldcs(reinterpret_cast<const uint2*>(at));
          u[i][0] = x.x;
          u[i][(kAt + 1) / 2 - 1] = x.y;
          sc[i] = *reinterpret_cast<const uint32_t*>(scale);
        } else if (G == 2 && a.vec_rows) {
          u[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(at));
          sc[i] = *reinterpret_cast<const uint16_t*>(scale);
        } else {
          sc[i] = 0;
#pragma unroll
          for (int g = 0; g < kAt; ++g) {
            const uint32_t two = uint32_t(at[2 * g]) | uint32_t(at[2 * g + 1]) << 8;
            u[i][g / 2] = g & 1 ? u[i][g / 2] | two << 16 : two;
            sc[i] |= uint32_t(scale[g]) << (8 * g);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        if (!ext[i]) continue;
#pragma unroll
        for (int g = 0; g < kAt; g += 2) {
          uint32_t h[4];
          if constexpr (G > 0) {
            e2m1x8_f16(u[i][g / 2], h[0], h[1], h[2], h[3]);
          } else {
            h[0] = e2m1x2_f16(u[i][0] & 255u);
            h[1] = e2m1x2_f16(u[i][0] >> 8);
          }
#pragma unroll
          for (int e = 0; e < 2 && g + e < kAt; ++e) {
            const float s = scale_of4(sc[i] >> (8 * (g + e)) & 255u);
            const float2 lo = f16x2_f32(h[2 * e]), hi = f16x2_f32(h[2 * e + 1]);
            Four y;
            narrow2(lo.x * s, lo.y * s, y.v);
            narrow2(hi.x * s, hi.y * s, y.v + 2);
            T* dst = ext[i] + 32 * (g + e);
            if (a.vec) {
              *reinterpret_cast<Four*>(dst) = y;
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) dst[k] = y.v[k];
            }
          }
        }
      }
    }
  }
}

template <typename T>
cudaError_t launch(const QuantMoveArgs& a, cudaStream_t st) {
  const int rows = a.planes * a.Hkv;
  const int64_t warps = int64_t(a.T) * ((rows + 4 * kPasses - 1) / (4 * kPasses));
  const int64_t ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
  const int grid = int(ctas < (1 << 20) ? ctas : (1 << 20));
  if (grid <= 0) return cudaSuccess;
  if (a.D == 128) quant4_read_kernel<T, 4><<<grid, kThreads, 0, st>>>(a);
  else if (a.D == 64) quant4_read_kernel<T, 2><<<grid, kThreads, 0, st>>>(a);
  else quant4_read_kernel<T, 0><<<grid, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quant4_read(const QuantMoveArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ACTKV_BF16) return launch<__nv_bfloat16>(a, st);
  if (dtype == ACTKV_F16) return launch<__half>(a, st);
  return launch<float>(a, st);
}

}  // namespace actkv
