// Writing new K / V rows into the 8-bit paged cache, and reading rows back (the row: quant_row.cuh).
//
// Both are bound by memory: per value 2 bytes of 16-bit rows and 33 / 32 bytes of the cache.  A warp
// takes one token and a run of its flattened (plane, 16 values) items; a lane moves 16 values per
// item (two 16-byte loads, one 16-byte store when writing; the reverse when reading), kItems items
// in flight, so a group of 32 is two neighbouring lanes and its maximum one shuffle.  The token's
// session and slot are found once per warp.
//
// Measured: writing 8 x 1088 tokens of 8 layers (8 heads of 128, bf16; 432 MB) 88 us, 4.9 TB/s, 0.75 of the
// measured copy rate, bound by issue (conversions and a multiplication per value; with a maximum per value instead
// of per pair 92 us); reading 46 K tokens of 4 layers (1.14 GB) 204 to 212 us, 5.4 to 5.6 TB/s, 0.82 to 0.86 of it.
// kItems 2 and 8 were slower (100 and 96 us written, where 4 took 91).
#include "kernels.cuh"
#include "quant_row.cuh"

namespace actkv {

namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;                   // items in flight per lane

// 16 values as they are in memory.
template <typename T>
struct Raw16 {
  uint4 u[sizeof(T)];
};

template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, Raw16<T>& r) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T)); ++i) r.u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T* e = reinterpret_cast<T*>(r.u);
#pragma unroll
    for (int k = 0; k < 16; ++k) e[k] = p[k];
  }
}

__device__ __forceinline__ uint32_t max16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ void store16(T* p, bool vec, const float (&x)[16]) {
  if (vec) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
      uint4 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int k = 0; k < kPer; ++k) e[k] = from_f32<T>(x[i * kPer + k]);
      __stcs(reinterpret_cast<uint4*>(p) + i, u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = from_f32<T>(x[i]);
  }
}

// The cache slot of packed token t (one per warp); -1 (flagged) when the tables do not hold it.
__device__ __forceinline__ int64_t slot_of(const QuantMoveArgs& a, int t, int lane) {
  const int r = session_of(a.tok_off, a.R, t, lane);
  if (r >= a.R || (a.ok && !a.ok[r])) return -1;   // no session's token, or one that was not appended
  const int pos = a.seq_used[r] - (a.tok_off[r + 1] - t);
  const int lb = pos / a.BS;
  const int phys = pos >= 0 && lb < a.MB ? a.block_table[r * a.bt_stride_r + lb] : -1;
  if (phys < 0 || phys >= a.NB) {
    if (lane == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
    return -1;
  }
  return int64_t(phys) * a.rows_stride_b + int64_t(pos - lb * a.BS) * a.rows_stride_s;
}

template <typename T, bool WRITE>
__global__ void __launch_bounds__(kThreads) quant_move_kernel(QuantMoveArgs a) {
  const int lane = threadIdx.x & 31;
  const int per_row = a.Hkv * a.D / 16;                     // items of one plane
  const int shift = (per_row & (per_row - 1)) == 0 ? __ffs(per_row) - 1 : -1;
  const bool packed = a.ext_stride_h[0] == a.D && a.ext_stride_h[1] == a.D;     // heads next to one another
  const int items = a.planes * per_row;                     // items of one token
  const int runs = (items + 32 * kItems - 1) / (32 * kItems);
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  int last = -1;
  int64_t slot = -1;
  for (int64_t w = warp; w < int64_t(a.T) * runs; w += nwarps) {
    const int t = int(w / runs), run = int(w - int64_t(t) * runs);
    if (t != last) slot = slot_of(a, t, lane);
    last = t;
    if (slot < 0) continue;
    T* ext[kItems];
    uint8_t* pay[kItems];
    uint8_t* sc[kItems];
    Raw16<T> in[WRITE ? kItems : 1];
    uint4 raw[kItems];
    uint32_t byte[kItems];
    // whether a lane has item i is the same for both lanes of a pair: per_row is even
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int f = (run * kItems + i) * 32 + lane;
      ext[i] = nullptr;
      if (f >= items) continue;
      const int lp = shift >= 0 ? f >> shift : f / per_row, c = f - lp * per_row;
      const int l = a.both ? lp >> 1 : lp, p = a.both ? lp & 1 : a.only;
      int64_t at = c * 16;
      if (!packed) {
        const int h = c * 16 / a.D;
        at = int64_t(h) * a.ext_stride_h[p] + (c * 16 - h * a.D);
      }
      T* base = static_cast<T*>(p ? a.v : a.k);
      ext[i] = base + (int64_t(l) * a.ext_stride_l[p] + int64_t(t) * a.ext_stride_t[p] + at);
      uint8_t* row = a.rows + int64_t(l) * a.rows_stride_l + int64_t(p) * a.rows_stride_kv + slot;
      pay[i] = row + c * 16;
      sc[i] = row + a.Hkv * a.D + c / 2;
      if constexpr (WRITE) {
        load16(ext[i], a.vec, in[i]);
      } else {
        if (a.vec_rows) {
          raw[i] = __ldcs(reinterpret_cast<const uint4*>(pay[i]));
        } else {
          uint8_t* b = reinterpret_cast<uint8_t*>(&raw[i]);
          for (int k = 0; k < 16; ++k) b[k] = pay[i][k];
        }
        byte[i] = *sc[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if constexpr (WRITE) {
        float x[16];
        uint32_t top = 0;
        const T* e = reinterpret_cast<const T*>(in[i].u);
        // without the sign, floats order as their bits do, NaN above all: 16-bit types in pairs
        if constexpr (sizeof(T) == 2) {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(in[i].u);
#pragma unroll
          for (int k = 0; k < 8; ++k) top = max16x2(top, w[k] & 0x7fff7fffu);
          const uint16_t t16 = uint16_t(max(top & 0xffffu, top >> 16));
          top = __float_as_uint(to_f32(reinterpret_cast<const T&>(t16)));
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          x[k] = to_f32(e[k]);
          if constexpr (sizeof(T) == 4) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
        }
        if (!ext[i]) top = 0;
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));      // the group's other 16 values
        if (!ext[i]) continue;
        const uint32_t b = scale_byte(top);
        const float inv = inverse_scale(b == 255u ? 0u : b);
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t lo = f32_e4m3x2(x[4 * k] * inv, x[4 * k + 1] * inv);
          const uint32_t hi = f32_e4m3x2(x[4 * k + 2] * inv, x[4 * k + 3] * inv);
          u[k] = b == 255u ? 0u : (lo & 0xffffu) | (hi << 16);
        }
        if (a.vec_rows) {
          *reinterpret_cast<uint4*>(pay[i]) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
          for (int k = 0; k < 16; ++k) pay[i][k] = uint8_t(u[k >> 2] >> (8 * (k & 3)));
        }
        if ((lane & 1) == 0) *sc[i] = uint8_t(b);
      } else {
        if (!ext[i]) continue;
        float x[16];
        const float s = scale_of(byte[i]);
        const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2 v = e4m3x2_f32((u[k >> 1] >> (16 * (k & 1))) & 0xffffu);
          x[2 * k] = v.x * s;
          x[2 * k + 1] = v.y * s;
        }
        store16(ext[i], a.vec, x);
      }
    }
  }
}

template <bool WRITE>
cudaError_t launch_move(const QuantMoveArgs& a, int dtype, cudaStream_t st) {
  const int items = a.planes * (a.Hkv * a.D / 16);
  const int64_t warps = int64_t(a.T) * ((items + 32 * kItems - 1) / (32 * kItems));
  const int64_t ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
  const int grid = int(ctas < (1 << 20) ? ctas : (1 << 20));
  if (grid <= 0) return cudaSuccess;
  if (dtype == ACTKV_BF16) quant_move_kernel<__nv_bfloat16, WRITE><<<grid, kThreads, 0, st>>>(a);
  else if (dtype == ACTKV_F16) quant_move_kernel<__half, WRITE><<<grid, kThreads, 0, st>>>(a);
  else quant_move_kernel<float, WRITE><<<grid, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quant_write(const QuantMoveArgs& a, int dtype, cudaStream_t st) { return launch_move<true>(a, dtype, st); }
cudaError_t launch_quant_read(const QuantMoveArgs& a, int dtype, cudaStream_t st) { return launch_move<false>(a, dtype, st); }

}  // namespace actkv
