// extern "C" entry points of chunk attention, of the 8- and 4-bit caches and of the rotation (include/actkv_b200.h):
// host-side validation and dispatch.
#include <stdarg.h>
#include <stdio.h>

#include <string.h>
#include <type_traits>
#include <utility>

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

int check_row(int bits, int64_t stride_s, int Hkv, int D) {
  if (D % kQuantGroup != 0)
    return fail(ACTKV_ERR_INVALID, "the %d-bit cache needs a head_dim that is a multiple of %d", bits, kQuantGroup);
  if (stride_s < least_row_bytes(bits, Hkv, D))
    return fail(ACTKV_ERR_INVALID, "a row of %lld bytes is shorter than its %lld values and scales",
                (long long)stride_s, (long long)least_row_bytes(bits, Hkv, D));
  return ACTKV_OK;
}

int chunk_attention(ChunkArgs& a, int dtype, int path, size_t workspace_bytes, cudaStream_t st) {
  if (!dtype_ok(dtype)) return fail(ACTKV_ERR_INVALID, "unknown dtype code");
  if (a.Hkv <= 0 || a.Hq <= 0 || a.Hq % a.Hkv != 0) return fail(ACTKV_ERR_INVALID, "n_q_heads %% n_kv_heads != 0");
  if (a.R < 0 || a.T < 0 || a.MB <= 0 || a.NB <= 0 || a.BS <= 0 || a.D <= 0) return fail(ACTKV_ERR_INVALID, "bad sizes");
  if (!(a.scale > 0.0f)) return fail(ACTKV_ERR_INVALID, "scale must be positive");
  if (path != ACTKV_PATH_AUTO && path != ACTKV_PATH_SIMT && path != ACTKV_PATH_TCGEN05)
    return fail(ACTKV_ERR_INVALID, "unknown path %d", path);
  if (a.quant)
    if (int rc = check_row(a.quant, a.kv_stride_s, a.Hkv, a.D)) return rc;
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

int check_rows(const QuantMoveArgs& a, int dtype, int L, int bits) {
  if (!dtype_ok(dtype)) return fail(ACTKV_ERR_INVALID, "unknown dtype code");
  if (L <= 0 || a.MB <= 0 || a.NB <= 0 || a.BS <= 0 || a.Hkv <= 0 || a.D <= 0 || a.R < 0 || a.T < 0)
    return fail(ACTKV_ERR_INVALID, "bad sizes");
  if (int rc = check_row(bits, a.rows_stride_s, a.Hkv, a.D)) return rc;
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

// The rows of k / v into the cache: the 8-bit writer, or the 4-bit one, which is the rotation's without an angle.
cudaError_t write_rows(const QuantMoveArgs& a, int dtype, int L, int bits, cudaStream_t st) {
  if (bits == 8) return launch_quant_write(a, dtype, st);
  const RotateArgs r{{nullptr, a.k, a.v}, {0, a.ext_stride_l[0], a.ext_stride_l[1]}, {0, a.ext_stride_t[0], a.ext_stride_t[1]},
                     {0, a.ext_stride_h[0], a.ext_stride_h[1]}, nullptr, 0, 0, 0, nullptr, nullptr, 0, 0, 0, 0, a.tok_off,
                     a.rows, a.rows_stride_l, a.rows_stride_kv, a.rows_stride_b, a.rows_stride_s, 0, a.block_table,
                     a.bt_stride_r, a.seq_used, a.ok, a.T, a.R, L, a.MB, a.NB, a.BS, 0, a.Hkv, a.D, bits, a.vec,
                     a.vec_rows, a.status};
  return launch_rotate_write(r, dtype, st);
}

int chunk_attention_rows(int bits, const void* q, int dtype, int64_t q_stride_t, int64_t q_stride_h,
                         const int32_t* q_off, int T, const uint8_t* rows, int64_t rows_stride_kv_bytes,
                         int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes, const int32_t* block_table,
                         int64_t bt_stride_r, const int32_t* seq_used, void* out, int64_t out_stride_t,
                         int64_t out_stride_h, float* lse, int64_t lse_stride_t, int R, int MB, int NB, int BS,
                         int Hq, int Hkv, int D, float scale, int path, void* workspace, size_t workspace_bytes,
                         int32_t* status, void* stream) {
  ChunkArgs a{q,   q_stride_t,   q_stride_h,   q_off, rows, rows_stride_kv_bytes, rows_stride_b_bytes, rows_stride_s_bytes,
              0, block_table, bt_stride_r, seq_used, out, out_stride_t, out_stride_h, lse,
              lse_stride_t, T, R, MB, NB, BS, Hq, Hkv, 0, D, bits, scale, workspace, status, 0};
  return chunk_attention(a, dtype, path, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int quantize_write(int bits, const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                   int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                   const int32_t* tok_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                   int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                   const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L, int MB,
                   int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  QuantMoveArgs a{const_cast<void*>(k_new), const_cast<void*>(v_new), {k_stride_l, v_stride_l}, {k_stride_t, v_stride_t},
                  {k_stride_h, v_stride_h}, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                  rows_stride_s_bytes, tok_off, block_table, bt_stride_r, seq_used, nullptr, T, R, MB, NB, BS, Hkv, D,
                  2 * L, 1, 0, false, false, status};
  if (int rc = check_rows(a, dtype, L, bits)) return rc;
  if (R == 0 || T == 0) return done(cudaSuccess, "");
  if (!k_new || !v_new || !tok_off || !rows || !block_table || !seq_used)
    return fail(ACTKV_ERR_INVALID, "k_new, v_new, tok_off, rows, block_table and seq_used are required");
  set_vectors(a, dtype);
  return done(write_rows(a, dtype, L, bits, static_cast<cudaStream_t>(stream)), "quantize_write");
}

int dequantize_read(int bits, void* k_out, void* v_out, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                    int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                    const int32_t* tok_off, int T, const uint8_t* rows, int64_t rows_stride_l_bytes,
                    int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                    const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L, int MB,
                    int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  const bool both = k_out && v_out;
  QuantMoveArgs a{k_out, v_out, {k_stride_l, v_stride_l}, {k_stride_t, v_stride_t}, {k_stride_h, v_stride_h},
                  const_cast<uint8_t*>(rows), rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                  rows_stride_s_bytes, tok_off, block_table, bt_stride_r, seq_used, nullptr, T, R, MB, NB, BS, Hkv, D,
                  both ? 2 * L : L, both ? 1 : 0, k_out ? 0 : 1, false, false, status};
  if (int rc = check_rows(a, dtype, L, bits)) return rc;
  if (R == 0 || T == 0) return done(cudaSuccess, "");
  if ((!k_out && !v_out) || !tok_off || !rows || !block_table || !seq_used)
    return fail(ACTKV_ERR_INVALID, "k_out or v_out, tok_off, rows, block_table and seq_used are required");
  set_vectors(a, dtype);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return done(bits == 4 ? launch_quant4_read(a, dtype, st) : launch_quant_read(a, dtype, st), "dequantize_read");
}

int quant_append(int bits, const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
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
  if (int rc = check_rows(a, dtype, L, bits)) return rc;
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
  return done(write_rows(a, dtype, L, bits, st), "quant_append");
}

int rotate_write(const int32_t* ok, const void* q, int64_t q_stride_l, int64_t q_stride_t, int64_t q_stride_h, void* q_out,
                 int64_t out_stride_l, int64_t out_stride_t, int64_t out_stride_h, const void* k_new,
                 int64_t k_stride_l, int64_t k_stride_t, int64_t k_stride_h, const void* v_new, int64_t v_stride_l,
                 int64_t v_stride_t, int64_t v_stride_h, int dtype, const int32_t* positions, const float* angles,
                 int64_t angles_stride, int P, int rot, int pairs, const int32_t* tok_off, int T, void* cache,
                 int bits, int64_t cache_stride_l, int64_t cache_stride_kv, int64_t cache_stride_b,
                 int64_t cache_stride_s, int64_t cache_stride_h, const int32_t* block_table, int64_t bt_stride_r,
                 const int32_t* seq_used, int R, int L, int MB, int NB, int BS, int Hq, int Hkv, int D,
                 int32_t* status, void* stream) {
  if (!dtype_ok(dtype)) return fail(ACTKV_ERR_INVALID, "unknown dtype code");
  if (bits != 0 && bits != 8 && bits != 4) return fail(ACTKV_ERR_INVALID, "bits %d: 0 (the inputs' type), 8 or 4", bits);
  if (L <= 0 || MB <= 0 || NB <= 0 || BS <= 0 || Hkv <= 0 || D <= 0 || R < 0 || T < 0 || Hq < 0)
    return fail(ACTKV_ERR_INVALID, "bad sizes");
  if (rot <= 0 || rot > D || rot % 2 != 0 || P <= 0)
    return fail(ACTKV_ERR_INVALID, "a rotation of %d of %d dims over %d positions", rot, D, P);
  if (bits && rot % 8 != 0) return fail(ACTKV_ERR_INVALID, "rows in %d bits need a rotated part in multiples of 8", bits);
  if (bits)
    if (int rc = check_row(bits, cache_stride_s, Hkv, D)) return rc;
  if (angles_stride < rot) return fail(ACTKV_ERR_INVALID, "the angles' rows are shorter than the rotated part");
  if (int64_t(L) * (int64_t(Hq) + 2 * int64_t(Hkv)) * D > 0x3fffffffll) return fail(ACTKV_ERR_INVALID, "too many values per token");
  if (R == 0 || T == 0) return done(cudaSuccess, "");
  if (!k_new || !v_new || !positions || !angles || !tok_off || !cache || !block_table || !seq_used || (Hq > 0 && (!q || !q_out)))
    return fail(ACTKV_ERR_INVALID, "k_new, v_new, positions, angles, tok_off, the cache, block_table and seq_used are "
                "required, and with Hq q and q_out");
  RotateArgs a{{q, k_new, v_new}, {q_stride_l, k_stride_l, v_stride_l}, {q_stride_t, k_stride_t, v_stride_t},
               {q_stride_h, k_stride_h, v_stride_h}, q_out, out_stride_l, out_stride_t, out_stride_h, positions, angles,
               angles_stride, P, rot, pairs != 0, tok_off, cache, cache_stride_l, cache_stride_kv, cache_stride_b,
               cache_stride_s, cache_stride_h, block_table, bt_stride_r, seq_used, ok, T, R, L, MB, NB, BS, Hq, Hkv,
               D, bits, false, false, status};
  const uint64_t es = dtype == ACTKV_F32 ? 4 : 2, cs = bits ? 1 : es;
  uint64_t in = uint64_t(reinterpret_cast<uintptr_t>(angles)) | uint64_t(angles_stride) * 4;
  for (int i = q ? 0 : 1; i < 3; ++i)
    in |= uint64_t(reinterpret_cast<uintptr_t>(a.in[i])) | (uint64_t(a.in_l[i]) | uint64_t(a.in_t[i]) | uint64_t(a.in_h[i])) * es;
  if (q)
    in |= uint64_t(reinterpret_cast<uintptr_t>(q_out)) | (uint64_t(out_stride_l) | uint64_t(out_stride_t) | uint64_t(out_stride_h)) * es;
  a.vec_in = in % 16 == 0;
  a.vec_out = (uint64_t(reinterpret_cast<uintptr_t>(cache)) | (uint64_t(cache_stride_l) | uint64_t(cache_stride_kv) |
               uint64_t(cache_stride_b) | uint64_t(cache_stride_s) | uint64_t(cache_stride_h)) * cs) % 16 == 0;
  return done(launch_rotate_write(a, dtype, static_cast<cudaStream_t>(stream)), "rotate_write");
}

// An entry called with its arguments as 64-bit words.
template <typename A>
A from_word(const int64_t& w) {
  if constexpr (std::is_pointer<A>::value) {
    return reinterpret_cast<A>(static_cast<intptr_t>(w));
  } else if constexpr (std::is_same<A, float>::value) {
    float f;
    memcpy(&f, &w, sizeof(f));
    return f;
  } else {
    return static_cast<A>(w);
  }
}
template <typename... A, size_t... I>
int call_words(int (*entry)(A...), const int64_t* w, std::index_sequence<I...>) {
  return entry(from_word<A>(w[I])...);
}
template <typename... A>
int call_words(int (*entry)(A...), const int64_t* w) {
  if (!w) return fail(ACTKV_ERR_INVALID, "the words are required");
  return call_words(entry, w, std::index_sequence_for<A...>());
}

// ... with an argument before them
template <typename... A, size_t... I>
int call_words(int (*entry)(const int32_t*, A...), const int32_t* first, const int64_t* w, std::index_sequence<I...>) {
  return entry(first, from_word<A>(w[I])...);
}
template <typename... A>
int call_rotate(int (*entry)(const int32_t*, A...), const int32_t* fits, const int64_t* w) {
  return call_words(entry, fits, w, std::index_sequence_for<A...>());
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
              lse_stride_t, T, R, MB, NB, BS, Hq, Hkv, 0, D, 0, scale, workspace, status, 0};
  return chunk_attention(a, dtype, path, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int actkv_chunk_attention_quant(const void* q, int dtype, int64_t q_stride_t, int64_t q_stride_h,
                                const int32_t* q_off, int T, const uint8_t* rows, int64_t rows_stride_kv_bytes,
                                int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes, const int32_t* block_table,
                                int64_t bt_stride_r, const int32_t* seq_used, void* out, int64_t out_stride_t,
                                int64_t out_stride_h, float* lse, int64_t lse_stride_t, int R, int MB, int NB,
                                int BS, int Hq, int Hkv, int D, float scale, int path, void* workspace,
                                size_t workspace_bytes, int32_t* status, void* stream) {
  return chunk_attention_rows(8, q, dtype, q_stride_t, q_stride_h, q_off, T, rows, rows_stride_kv_bytes,
                              rows_stride_b_bytes, rows_stride_s_bytes, block_table, bt_stride_r, seq_used, out,
                              out_stride_t, out_stride_h, lse, lse_stride_t, R, MB, NB, BS, Hq, Hkv, D, scale, path,
                              workspace, workspace_bytes, status, stream);
}

int actkv_chunk_attention_quant4(const void* q, int dtype, int64_t q_stride_t, int64_t q_stride_h,
                                 const int32_t* q_off, int T, const uint8_t* rows, int64_t rows_stride_kv_bytes,
                                 int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                                 const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, void* out,
                                 int64_t out_stride_t, int64_t out_stride_h, float* lse, int64_t lse_stride_t, int R,
                                 int MB, int NB, int BS, int Hq, int Hkv, int D, float scale, int path,
                                 void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return chunk_attention_rows(4, q, dtype, q_stride_t, q_stride_h, q_off, T, rows, rows_stride_kv_bytes,
                              rows_stride_b_bytes, rows_stride_s_bytes, block_table, bt_stride_r, seq_used, out,
                              out_stride_t, out_stride_h, lse, lse_stride_t, R, MB, NB, BS, Hq, Hkv, D, scale, path,
                              workspace, workspace_bytes, status, stream);
}

int actkv_quantize_write(const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                         int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                         const int32_t* tok_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                         int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                         const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L,
                         int MB, int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  return quantize_write(8, k_new, v_new, dtype, k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t,
                        v_stride_h, tok_off, T, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                        rows_stride_s_bytes, block_table, bt_stride_r, seq_used, R, L, MB, NB, BS, Hkv, D, status,
                        stream);
}

int actkv_quantize_write4(const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                          int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                          const int32_t* tok_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                          int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                          const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L,
                          int MB, int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  return quantize_write(4, k_new, v_new, dtype, k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t,
                        v_stride_h, tok_off, T, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                        rows_stride_s_bytes, block_table, bt_stride_r, seq_used, R, L, MB, NB, BS, Hkv, D, status,
                        stream);
}

int actkv_dequantize_read(void* k_out, void* v_out, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                          int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                          const int32_t* tok_off, int T, const uint8_t* rows, int64_t rows_stride_l_bytes,
                          int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                          const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L,
                          int MB, int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  return dequantize_read(8, k_out, v_out, dtype, k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t,
                         v_stride_h, tok_off, T, rows, rows_stride_l_bytes, rows_stride_kv_bytes,
                         rows_stride_b_bytes, rows_stride_s_bytes, block_table, bt_stride_r, seq_used, R, L, MB, NB,
                         BS, Hkv, D, status, stream);
}

int actkv_dequantize_read4(void* k_out, void* v_out, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                           int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                           const int32_t* tok_off, int T, const uint8_t* rows, int64_t rows_stride_l_bytes,
                           int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                           const int32_t* block_table, int64_t bt_stride_r, const int32_t* seq_used, int R, int L,
                           int MB, int NB, int BS, int Hkv, int D, int32_t* status, void* stream) {
  return dequantize_read(4, k_out, v_out, dtype, k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t,
                         v_stride_h, tok_off, T, rows, rows_stride_l_bytes, rows_stride_kv_bytes,
                         rows_stride_b_bytes, rows_stride_s_bytes, block_table, bt_stride_r, seq_used, R, L, MB, NB,
                         BS, Hkv, D, status, stream);
}

int actkv_quant_append(const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                       int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                       const int32_t* new_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                       int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                       int32_t* block_table, int64_t bt_stride_r, int32_t* seq_used, const int32_t* free_list,
                       int32_t* free_top, int64_t free_capacity, int R, int L, int MB, int NB, int BS, int Hkv,
                       int D, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return quant_append(8, k_new, v_new, dtype, k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t, v_stride_h,
                      new_off, T, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                      rows_stride_s_bytes, block_table, bt_stride_r, seq_used, free_list, free_top, free_capacity, R,
                      L, MB, NB, BS, Hkv, D, workspace, workspace_bytes, status, stream);
}

int actkv_quant4_append(const void* k_new, const void* v_new, int dtype, int64_t k_stride_l, int64_t k_stride_t,
                        int64_t k_stride_h, int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h,
                        const int32_t* new_off, int T, uint8_t* rows, int64_t rows_stride_l_bytes,
                        int64_t rows_stride_kv_bytes, int64_t rows_stride_b_bytes, int64_t rows_stride_s_bytes,
                        int32_t* block_table, int64_t bt_stride_r, int32_t* seq_used, const int32_t* free_list,
                        int32_t* free_top, int64_t free_capacity, int R, int L, int MB, int NB, int BS, int Hkv,
                        int D, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return quant_append(4, k_new, v_new, dtype, k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t, v_stride_h,
                      new_off, T, rows, rows_stride_l_bytes, rows_stride_kv_bytes, rows_stride_b_bytes,
                      rows_stride_s_bytes, block_table, bt_stride_r, seq_used, free_list, free_top, free_capacity, R,
                      L, MB, NB, BS, Hkv, D, workspace, workspace_bytes, status, stream);
}

int actkv_rotate_write(const void* q, int64_t q_stride_l, int64_t q_stride_t, int64_t q_stride_h, void* q_out,
                       int64_t out_stride_l, int64_t out_stride_t, int64_t out_stride_h, const void* k_new,
                       int64_t k_stride_l, int64_t k_stride_t, int64_t k_stride_h, const void* v_new, int64_t v_stride_l,
                       int64_t v_stride_t, int64_t v_stride_h, int dtype, const int32_t* positions, const float* angles,
                       int64_t angles_stride, int P, int rot, int pairs, const int32_t* tok_off, int T, void* cache,
                       int bits, int64_t cache_stride_l, int64_t cache_stride_kv, int64_t cache_stride_b,
                       int64_t cache_stride_s, int64_t cache_stride_h, const int32_t* block_table, int64_t bt_stride_r,
                       const int32_t* seq_used, int R, int L, int MB, int NB, int BS, int Hq, int Hkv, int D,
                       int32_t* status, void* stream) {
  return rotate_write(nullptr, q, q_stride_l, q_stride_t, q_stride_h, q_out, out_stride_l, out_stride_t,
                      out_stride_h, k_new, k_stride_l, k_stride_t, k_stride_h, v_new, v_stride_l, v_stride_t,
                      v_stride_h, dtype, positions, angles, angles_stride, P, rot, pairs, tok_off, T, cache, bits,
                      cache_stride_l, cache_stride_kv, cache_stride_b, cache_stride_s, cache_stride_h, block_table,
                      bt_stride_r, seq_used, R, L, MB, NB, BS, Hq, Hkv, D, status, stream);
}

int actkv_rotate_write_words(const int64_t* words) { return call_words(actkv_rotate_write, words); }
int actkv_rotate_write_fits(const int32_t* fits, const int64_t* words) {
  if (!words) return fail(ACTKV_ERR_INVALID, "the words are required");
  return call_rotate(rotate_write, fits, words);
}
int actkv_quantize_write_words(int bits, const int64_t* words) {
  return call_words(bits == 4 ? actkv_quantize_write4 : actkv_quantize_write, words);
}
int actkv_dequantize_read_words(int bits, const int64_t* words) {
  return call_words(bits == 4 ? actkv_dequantize_read4 : actkv_dequantize_read, words);
}
int actkv_chunk_attention_quant_words(int bits, const int64_t* words) {
  return call_words(bits == 4 ? actkv_chunk_attention_quant4 : actkv_chunk_attention_quant, words);
}

}  // extern "C"
