// extern "C" entry points of chunk attention and of the 8-bit cache (include/actkv_b200.h): host-side
// validation and dispatch.
#include <stdarg.h>
#include <stdio.h>

#include "kernels.cuh"
#include "quant_row.cuh"

namespace actkv {
void set_last_error(const char* msg);
}

using namespace actkv;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

int done(cudaError_t e, const char* where) {
  if (e != cudaSuccess) return fail(ACTKV_ERR_CUDA, "%s: %s", where, cudaGetErrorString(e));
  set_last_error("");
  return ACTKV_OK;
}

bool dtype_ok(int d) { return d == ACTKV_F32 || d == ACTKV_F16 || d == ACTKV_BF16; }

int chunk_attention(ChunkArgs& a, int dtype, int path, size_t workspace_bytes, cudaStream_t st) {
  if (!dtype_ok(dtype)) return fail(ACTKV_ERR_INVALID, "unknown dtype code");
  if (a.Hkv <= 0 || a.Hq <= 0 || a.Hq % a.Hkv != 0) return fail(ACTKV_ERR_INVALID, "n_q_heads %% n_kv_heads != 0");
  if (a.R < 0 || a.T < 0 || a.MB <= 0 || a.NB <= 0 || a.BS <= 0 || a.D <= 0) return fail(ACTKV_ERR_INVALID, "bad sizes");
  if (!(a.scale > 0.0f)) return fail(ACTKV_ERR_INVALID, "scale must be positive");
  if (path != ACTKV_PATH_AUTO && path != ACTKV_PATH_SIMT && path != ACTKV_PATH_TCGEN05)
    return fail(ACTKV_ERR_INVALID, "unknown path %d", path);
  if (a.quant && a.D % kQuantGroup != 0)
    return fail(ACTKV_ERR_INVALID, "the 8-bit cache needs a head_dim that is a multiple of %d", kQuantGroup);
  if (a.quant && a.kv_stride_s < int64_t(a.Hkv) * (a.D + a.D / kQuantGroup))
    return fail(ACTKV_ERR_INVALID, "a row of %lld bytes is shorter than its %lld values and scales",
                (long long)a.kv_stride_s, (long long)a.Hkv * (a.D + a.D / kQuantGroup));
  if (a.R == 0 || a.T == 0) return done(cudaSuccess, "");
  if (!a.q || !a.q_off || !a.kv || !a.block_table || !a.seq_used || !a.out || !a.lse)
    return fail(ACTKV_ERR_INVALID, "q, q_off, the cache, block_table, seq_used, out and lse are required");
  const size_t need = chunk_workspace_bytes(device_sm_count());
  if (!a.workspace || workspace_bytes < need)
    return fail(ACTKV_ERR_WORKSPACE, "workspace of %zu bytes, need %zu", a.workspace ? workspace_bytes : 0, need);
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return fail(ACTKV_ERR_WORKSPACE, "the workspace must be 16-byte aligned");
  a.G = a.Hq / a.Hkv;
  const char* why = "";
  const bool tc = path != ACTKV_PATH_SIMT && chunk_umma_supported(a, dtype, &why);
  if (path == ACTKV_PATH_TCGEN05 && !tc) return fail(ACTKV_ERR_UNSUPPORTED, "chunk attention on tensor cores: %s", why);
  if (tc)
    return done(launch_chunk_umma(a, dtype, st, &why), why);
  if (a.D > 256) return fail(ACTKV_ERR_UNSUPPORTED, "chunk attention: head_dim %d is over 256", a.D);
  if (int64_t(a.T) * a.Hq > 0x7fffffffll) return fail(ACTKV_ERR_UNSUPPORTED, "chunk attention: too many query rows");
  return done(launch_chunk_simt(a, dtype, st), "chunk attention");
}

int check_rows(const QuantMoveArgs& a, int dtype, int L) {
  if (!dtype_ok(dtype)) return fail(ACTKV_ERR_INVALID, "unknown dtype code");
  if (L <= 0 || a.MB <= 0 || a.NB <= 0 || a.BS <= 0 || a.Hkv <= 0 || a.D <= 0 || a.R < 0 || a.T < 0)
    return fail(ACTKV_ERR_INVALID, "bad sizes");
  if (a.D % kQuantGroup != 0)
    return fail(ACTKV_ERR_INVALID, "the 8-bit cache needs a head_dim that is a multiple of %d", kQuantGroup);
  if (a.rows_stride_s < int64_t(a.Hkv) * (a.D + a.D / kQuantGroup))
    return fail(ACTKV_ERR_INVALID, "a row of %lld bytes is shorter than its %lld values and scales",
                (long long)a.rows_stride_s, (long long)a.Hkv * (a.D + a.D / kQuantGroup));
  if (int64_t(2) * L * a.Hkv * a.D / 16 > 0x3fffffffll) return fail(ACTKV_ERR_INVALID, "too many values per token");
  return ACTKV_OK;
}

// 16-byte accesses need aligned bases and strides; the payload starts every row at its base.
void set_vectors(QuantMoveArgs& a, int dtype) {
  const int es = dtype == ACTKV_F32 ? 4 : 2;
  uint64_t ext = 0;
  for (int p = 0; p < 2; ++p) {
    const void* base = p ? a.v : a.k;
    if (base)
      ext |= uint64_t(reinterpret_cast<uintptr_t>(base)) | uint64_t(a.ext_stride_l[p] * es) |
             uint64_t(a.ext_stride_t[p] * es) | uint64_t(a.ext_stride_h[p] * es);
  }
  a.vec = ext % 16 == 0;
  a.vec_rows = (uint64_t(reinterpret_cast<uintptr_t>(a.rows)) | uint64_t(a.rows_stride_l) | uint64_t(a.rows_stride_kv) |
                uint64_t(a.rows_stride_b) | uint64_t(a.rows_stride_s)) % 16 == 0;
}

}  // namespace

extern "C" {

size_t actkv_chunk_workspace_bytes(void) { return chunk_workspace_bytes(device_sm_count()); }

int actkv_chunk_attention(const void* q, int dtype, int64_t q_stride_t, int64_t q_stride_h, const int32_t* q_off, int T,
                          const void* kv, int64_t kv_stride_kv, int64_t kv_stride_b, int64_t kv_stride_s,
                          int64_t kv_stride_h, const int32_t* block_table, int64_t bt_stride_r,
                          const int32_t* seq_used, void* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
                          int64_t lse_stride_t, int R, int MB, int NB, int BS, int Hq, int Hkv, int D, float scale,
                          int path, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  ChunkArgs a{q,   q_stride_t,   q_stride_h,   q_off, kv,           kv_stride_kv, kv_stride_b, kv_stride_s,
              kv_stride_h, block_table, bt_stride_r, seq_used, out, out_stride_t, out_stride_h, lse,
              lse_stride_t, T, R, MB, NB, BS, Hq, Hkv, 0, D, false, scale, workspace, status, 0};
  return chunk_attention(a, dtype, path, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int actkv_chunk_attention_quant(const void* q, int dtype, int64_t q_stride_t, int64_t q_stride_h, const int32_t* q_off,
                                int T, const uint8_t* rows, int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes,
                                int64_t rows_stride_s_bytes, const int32_t* block_table, int64_t bt_stride_r,
                                const int32_t* seq_used, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                float* lse, int64_t lse_stride_t, int R, int MB, int NB, int BS, int Hq, int Hkv,
                                int D, float scale, int path, void* workspace, size_t workspace_bytes,
                                int32_t* status, void* stream) {
  ChunkArgs a{q,   q_stride_t,   q_stride_h,   q_off, rows, rows_stride_kv_bytes, rows_stride_b_bytes, rows_stride_s_bytes,
              0, block_table, bt_stride_r, seq_used, out, out_stride_t, out_stride_h, lse,
              lse_stride_t, T, R, MB, NB, BS, Hq, Hkv, 0, D, true, scale, workspace, status, 0};
  return chunk_attention(a, dtype, path, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int actkv_quantize_write(const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                         int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                         const int32_t* tok_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                         int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                         const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L,
                         int MB, int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  QuantMoveArgs a{const_cast<void*>(k_new), const_cast<void*>(v_new), {k_stride_l, v_stride_l}, {k_stride_t, v_stride_t},
                  {k_stride_h, v_stride_h}, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                  rows_stride_s_bytes, tok_off, block_table, bt_stride_r, seq_used, nullptr, T, R, MB, NB, BS, Hkv, D,
                  2 * L, 1, 0, false, false, status};
  if (int rc = check_rows(a, dtype, L)) return rc;
  if (R == 0 || T == 0) return done(cudaSuccess, "");
  if (!k_new || !v_new || !tok_off || !rows || !block_table || !seq_used)
    return fail(ACTKV_ERR_INVALID, "k_new, v_new, tok_off, rows, block_table and seq_used are required");
  set_vectors(a, dtype);
  return done(launch_quant_write(a, dtype, static_cast<cudaStream_t>(stream)), "quantize_write");
}

int actkv_dequantize_read(void* k_out, void* v_out, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                          int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                          const int32_t* tok_off, int T, const uint8_t* rows, int64_t rows_stride_l_bytes,
                          int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                          const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L,
                          int MB, int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  const bool both = k_out && v_out;
  QuantMoveArgs a{k_out, v_out, {k_stride_l, v_stride_l}, {k_stride_t, v_stride_t}, {k_stride_h, v_stride_h},
                  const_cast<uint8_t*>(rows), rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                  rows_stride_s_bytes, tok_off, block_table, bt_stride_r, seq_used, nullptr, T, R, MB, NB, BS, Hkv, D,
                  both ? 2 * L : L, both ? 1 : 0, k_out ? 0 : 1, false, false, status};
  if (int rc = check_rows(a, dtype, L)) return rc;
  if (R == 0 || T == 0) return done(cudaSuccess, "");
  if ((!k_out && !v_out) || !tok_off || !rows || !block_table || !seq_used)
    return fail(ACTKV_ERR_INVALID, "k_out or v_out, tok_off, rows, block_table and seq_used are required");
  set_vectors(a, dtype);
  return done(launch_quant_read(a, dtype, static_cast<cudaStream_t>(stream)), "dequantize_read");
}

int actkv_quant_append(const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                       int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                       const int32_t* new_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                       int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                       int32_t* block_table, int64_t bt_stride_r, int32_t* seq_used, const int32_t* free_list,
                       int32_t* free_top, int64_t free_capacity, int R, int L, int MB, int NB, int BS, int Hkv, int D,
                       void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  QuantMoveArgs a{const_cast<void*>(k_new), const_cast<void*>(v_new), {k_stride_l, v_stride_l}, {k_stride_t, v_stride_t},
                  {k_stride_h, v_stride_h}, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                  rows_stride_s_bytes, new_off, block_table, bt_stride_r, seq_used, nullptr, T, R, MB, NB, BS, Hkv, D,
                  2 * L, 1, 0, false, false, status};
  if (int rc = check_rows(a, dtype, L)) return rc;
  if (R == 0) return done(cudaSuccess, "");
  if ((T > 0 && (!k_new || !v_new)) || !new_off || !rows || !block_table || !seq_used || !free_list || !free_top)
    return fail(ACTKV_ERR_INVALID, "k_new, v_new, new_off, rows, block_table, seq_used and the free stack are required");
  if (!workspace || workspace_bytes < blocks_workspace_bytes(R))
    return fail(ACTKV_ERR_WORKSPACE, "workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0,
                blocks_workspace_bytes(R));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // tables, lengths and the free stack (no rows), then the rows of the sessions that fit
  cudaError_t e = launch_append(nullptr, L, 0, 0, 0, 0, nullptr, nullptr, 0, 0, new_off, 0, seq_used, block_table,
                                bt_stride_r, MB, BS, free_list, free_top, free_capacity, R, workspace, status, st);
  if (e != cudaSuccess || T == 0) return done(e, "quant_append");
  a.ok = append_ok_flags(workspace, R);
  set_vectors(a, dtype);
  return done(launch_quant_write(a, dtype, st), "quant_append");
}

}  // extern "C"
