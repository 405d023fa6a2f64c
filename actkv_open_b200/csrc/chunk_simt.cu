// Attention of each session's newest tokens (a chunk of queries) over its paged cache, with the
// log-sum-exp, on CUDA cores: any dtype, head size (a multiple of 32 up to 256 over the 8-bit
// cache, any up to 256 else), block size, GQA group and stride.  The tensor-core kernel
// (chunk_umma.cu) takes the layouts it can; this one takes the rest (fp32 caches above all).
//
// Query j of a session with S tokens and A new ones sees tokens t <= S - A + j.  With
// x_t = scale * q . k_t:  m = max x, l = sum 2^((x_t - m) log2 e), out = sum p_t v_t / l,
// lse = m + ln l; a query that sees no token gets out 0 and lse -inf.
//
// A CTA takes one (query token, query head): its four warps take every fourth token, a lane the
// dims lane, lane + 32, ..., with a running maximum, sum and output per warp, joined at the end.
// Bound by issue (a warp-wide sum per token), not by memory: 10.3 ms for the 32-session decode batch that
// chunk_few.cu does in 0.38.
#include "kernels.cuh"
#include "quant_row.cuh"

namespace actkv {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxPer = 8;                  // dims per lane: head_dim <= 256

template <typename T, bool QUANT>
__device__ __forceinline__ void load_row(const ChunkArgs& a, const void* base, int64_t off, int h, int lane,
                                         float (&x)[kMaxPer]) {
#pragma unroll
  for (int i = 0; i < kMaxPer; ++i) {
    const int d = lane + 32 * i;
    x[i] = 0.0f;
    if (d >= a.D) continue;
    if constexpr (QUANT) {
      const uint8_t* row = static_cast<const uint8_t*>(base) + off;
      const int e = h * a.D + d;
      x[i] = to_f32(from_f32<T>(e4m3x2_f32(row[e]).x * scale_of(row[a.Hkv * a.D + e / kQuantGroup])));
    } else {
      x[i] = to_f32(static_cast<const T*>(base)[off + int64_t(h) * a.kv_stride_h + d]);
    }
  }
}

template <typename T, bool QUANT>
__global__ void __launch_bounds__(kWarps * 32) chunk_simt_kernel(ChunkArgs a) {
  __shared__ float sh_m[kWarps], sh_l[kWarps], sh_o[kWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = int(blockIdx.x / a.Hq), hq = int(blockIdx.x % a.Hq);
  const int r = session_of(a.q_off, a.R, t, lane);
  if (r >= a.R) return;                      // not a query of any session
  if (a.q_off[r] < 0 || a.q_off[r + 1] > a.T) {             // a session that leaves the call's rows: left alone
    if (threadIdx.x == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
    return;
  }
  const int S = a.seq_used[r];
  const int64_t room = int64_t(a.MB) * a.BS;                // of the table: what is past it is hidden
  const int64_t sees = int64_t(S) - (a.q_off[r + 1] - t) + 1;
  if (S > room && threadIdx.x == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
  const int seen = int(min(max(sees, int64_t(0)), room));   // tokens this query sees
  const int h = hq / a.G;
  float q[kMaxPer], o[kMaxPer];
  const T* qp = static_cast<const T*>(a.q) + int64_t(t) * a.q_stride_t + int64_t(hq) * a.q_stride_h;
#pragma unroll
  for (int i = 0; i < kMaxPer; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < a.D ? to_f32(qp[d]) : 0.0f;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const float c2 = a.scale * kLog2e;
  for (int p = warp; p < seen; p += kWarps) {
    const int lb = p / a.BS;
    const int phys = a.block_table[r * a.bt_stride_r + lb];
    if (phys < 0 || phys >= a.NB) {
      if (lane == 0) flag(a.status, ACTKV_DEV_BAD_INDEX);
      continue;
    }
    const int64_t off = int64_t(phys) * a.kv_stride_b + int64_t(p - lb * a.BS) * a.kv_stride_s;
    float k[kMaxPer], v[kMaxPer];
    load_row<T, QUANT>(a, a.kv, off, h, lane, k);
    load_row<T, QUANT>(a, a.kv, off + a.kv_stride_kv, h, lane, v);
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) x = fmaf(q[i], k[i], x);
    x = warp_sum(x) * c2;
    const float mn = fmaxf(m, x);
    const float base = mn == -INFINITY ? 0.0f : mn;
    const float al = exp2f(m - base), pr = exp2f(x - base);
    l = fmaf(l, al, pr);
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) o[i] = fmaf(o[i], al, pr * v[i]);
    m = mn;
  }
  if (lane == 0) {
    sh_m[warp] = m;
    sh_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kMaxPer; ++i) sh_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sh_m[w]);
  const float base = M == -INFINITY ? 0.0f : M;
  float L = 0.0f, al[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    al[w] = exp2f(sh_m[w] - base);
    L += sh_l[w] * al[w];
  }
  T* op = static_cast<T*>(a.out) + int64_t(t) * a.out_stride_t + int64_t(hq) * a.out_stride_h;
  for (int d = threadIdx.x; d < a.D; d += kWarps * 32) {
    float s = 0.0f;
    for (int w = 0; w < kWarps; ++w) s += sh_o[w][d] * al[w];
    const float y = L == 0.0f ? 0.0f : s / L;
    if constexpr (sizeof(T) == 4) op[d] = y;
    else if constexpr (std::is_same<T, __half>::value) op[d] = __float2half_rn(y);
    else op[d] = __float2bfloat16_rn(y);
  }
  if (threadIdx.x == 0)
    a.lse[int64_t(t) * a.lse_stride_t + hq] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

}  // namespace

cudaError_t launch_chunk_simt(const ChunkArgs& a, int dtype, cudaStream_t st) {
  const int64_t ctas = int64_t(a.T) * a.Hq;
  const dim3 grid = dim3(unsigned(ctas)), block = dim3(kWarps * 32);
  if (a.quant) {
    if (dtype == ACTKV_BF16) chunk_simt_kernel<__nv_bfloat16, true><<<grid, block, 0, st>>>(a);
    else if (dtype == ACTKV_F16) chunk_simt_kernel<__half, true><<<grid, block, 0, st>>>(a);
    else chunk_simt_kernel<float, true><<<grid, block, 0, st>>>(a);
  } else {
    if (dtype == ACTKV_BF16) chunk_simt_kernel<__nv_bfloat16, false><<<grid, block, 0, st>>>(a);
    else if (dtype == ACTKV_F16) chunk_simt_kernel<__half, false><<<grid, block, 0, st>>>(a);
    else chunk_simt_kernel<float, false><<<grid, block, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace actkv
