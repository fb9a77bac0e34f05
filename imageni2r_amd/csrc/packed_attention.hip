// Attention over packed sequences with a bucketed relative position bias: forward and backward.
#include "packed_rows.h"

bool pa_launch_fwd(int dtype, const PaArgs& a, hipStream_t st);  // packed_fwd.hip
bool pa_is_token(int batch, int nq, int heads, int kv_heads);  // packed_token.hip
long pa_token_ws_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dim);
bool pa_launch_token(int dtype, const PaArgs& a, void* ws, hipStream_t st);
bool pa_launch_dq(int dtype, const PaArgs& a, hipStream_t st);   // packed_dq.hip
bool pa_launch_dkv(int dtype, const PaArgs& a, hipStream_t st);  // packed_dkv.hip

// delta = <dout, out> of each row and head, and the sum of its stats: for dk and dv without dq.  Two threads for each, in the
// dq kernel's order, so that the gradients do not depend on which of them are asked for.
template <typename T>
__global__ __launch_bounds__(256) void pa_delta_kernel(PaArgs a) {
  constexpr int N = 16 / sizeof(T);
  const long item = (long)blockIdx.x * 128 + (threadIdx.x >> 1);
  const long row = item / a.heads, at = item * a.dim;
  float s = 0.0f;
  if (row < a.nq)
    for (int d = (threadIdx.x & 1) * N; d < a.dim; d += 2 * N)
      for (int e = 0; e < N; ++e) s = fmaf((float)((const T*)a.dout)[at + d + e], a.out32_in[at + d + e], s);
  s += __shfl_xor(s, 1, 64);
  const long st = (item % a.heads) * a.nq + row, n = (long)a.heads * a.nq;
  if (row < a.nq && !(threadIdx.x & 1)) a.delta[st] = s, a.delta[st + n] = a.stats[st] + (a.stats[st + n] - Lift<T>::LOG2);
}

// dtable[h][c] = sum of the parts, in a fixed order: each thread a stride of them, then a tree
__global__ __launch_bounds__(256) void pa_dtable_kernel(const float* part, float* dtable, long parts, int heads, int nb) {
  __shared__ float sum[256];
  const int h = blockIdx.x, c = blockIdx.y;
  float s = 0.0f;
  for (long i = threadIdx.x; i < parts; i += 256) s += part[(i * heads + h) * nb + c];
  sum[threadIdx.x] = s;
  for (int n = 128; n > 0; n >>= 1) {
    __syncthreads();
    if (threadIdx.x < n) sum[threadIdx.x] += sum[threadIdx.x + n];
  }
  if (threadIdx.x == 0) dtable[(long)h * nb + c] = sum[0];
}

static long esize(int dtype) { return dtype == 0 ? 4 : 2; }

static int check(const char* what, const i2r_packed_seqs* s, const void* q, const void* k, const void* v, const float* table,
                 int dtype, int nq, int nk, int heads, int kv_heads, int dim, const long (&strides)[6]) {
  I2R_REQUIRE(s && s->cu_q && s->cu_k && s->batch > 0, "%s: no sequences", what);
  I2R_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d is not 0 (fp32), 1 (fp16) or 2 (bf16)", what, dtype);
  I2R_REQUIRE(nq >= 0 && nk >= 0 && nq < 1 << 30 && nk < 1 << 30, "%s: 0 to 2^30 - 1 rows are supported", what);
  I2R_REQUIRE(kv_heads > 0 && heads > 0 && heads < 65536 && heads % kv_heads == 0, "%s: %d heads are no multiple of %d key / value heads",
              what, heads, kv_heads);
  I2R_REQUIRE(((long)std::max(nq, nk) + s->batch + 2) * heads < INT32_MAX / 2, "%s: too many rows times heads", what);
  I2R_REQUIRE(dim >= 8 && dim <= 128 && dim % 8 == 0, "%s: head dim %d is not a multiple of 8 up to 128", what, dim);
  I2R_REQUIRE((q || !nq) && (k || !nk) && (v || !nk), "%s: null tensor", what);
  I2R_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: q, k and v have to be 16-byte aligned", what);
  // Rows of a tile are offset in 32 bits, heads in 64 (a cache that holds head after head: rows * dim apart).
  for (int i = 0; i < 6; ++i)
    I2R_REQUIRE(strides[i] >= 0 && strides[i] < (i % 2 ? 1L << 40 : 1L << 22) && strides[i] * esize(dtype) % 16 == 0,
                "%s: strides have to be whole multiples of 16 bytes, those of tokens below 2^22 elements", what);
  I2R_REQUIRE(!s->pos_q == !s->pos_k, "%s: positions of queries and keys come together", what);
  if (table) {
    I2R_REQUIRE(s->lut && s->num_buckets > 0 && s->num_buckets <= PA_MAX_BUCKETS, "%s: %d buckets: 1 to %d are supported",
                what, s->num_buckets, PA_MAX_BUCKETS);
    I2R_REQUIRE(s->max_distance >= 0 && s->max_distance <= PA_MAX_DISTANCE, "%s: distance %d: 0 to %d are supported", what,
                s->max_distance, PA_MAX_DISTANCE);
  }
  return I2R_OK;
}

extern "C" long i2r_packed_attention_fwd_ws_bytes(int, int batch, int nq, int nk, int heads, int kv_heads, int dim) {
  if (batch <= 0 || nq <= 0 || nk < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0) return 0;
  return pa_is_token(batch, nq, heads, kv_heads) ? pa_token_ws_bytes(batch, nq, nk, heads, kv_heads, dim) : 0;
}

extern "C" int i2r_packed_attention_fwd(const i2r_packed_seqs* seqs, const void* q, const void* k, const void* v,
                                        const float* table, void* out, float* out32, float* stats, void* ws, long ws_bytes,
                                        int dtype, int nq, int nk, int heads, int kv_heads, int dim, long q_row, long q_head,
                                        long k_row, long k_head, long v_row, long v_head, float scale, int zero_outside,
                                        i2r_stream_t stream) {
  if (int rc = check("packed_attention_fwd", seqs, q, k, v, table, dtype, nq, nk, heads, kv_heads, dim,
                     {q_row, q_head, k_row, k_head, v_row, v_head}))
    return rc;
  if (nq == 0) return I2R_OK;
  I2R_REQUIRE(out && (uintptr_t)out % 16 == 0, "packed_attention_fwd: out is null or not 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  PaArgs a = {};
  a.s = *seqs;
  a.q = q, a.k = k, a.v = v, a.table = table, a.out = out, a.out32 = out32, a.stats = stats;
  a.nq = nq, a.nk = nk, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.scale = scale, a.zero_outside = zero_outside;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  const long need = i2r_packed_attention_fwd_ws_bytes(dtype, seqs->batch, nq, nk, heads, kv_heads, dim);
  I2R_REQUIRE(ws_bytes >= need && (ws || !need), "packed_attention_fwd: workspace of %ld bytes, %ld are needed", ws_bytes,
              need);
  I2R_REQUIRE((uintptr_t)ws % 16 == 0, "packed_attention_fwd: the workspace has to be 16-byte aligned");
  if (!(pa_is_token(seqs->batch, nq, heads, kv_heads) ? pa_launch_token(dtype, a, ws, st) : pa_launch_fwd(dtype, a, st)))
    return I2R_ERR_HIP;
  return i2r_check_launch("packed_attention_fwd");
}

static long q_slots(int nq, int batch) { return (nq >> 7) + batch + 2; }

// A key / value head's query heads go to several workgroups, whose sums are joined, where the keys alone are too few: below 256
// blocks of 128 keys, one for each CU, or two of the workgroups of 64 that most widths have.  Split against whole: 8192 tokens,
// 16 heads over 2 (130 blocks), of 128 596 us, 2027; of 64 356, 1111; 6000 tokens, 16 heads of 64 over 4 (188) 252, 418; 2 x
// 1024, over 8 (144) 39.5, 45.7; fp32 of 64, 4096 tokens, over 4 (132) 598, 1571.
static int dkv_parts(int batch, int nk, int heads, int kv_heads) {
  const long busy = ((long)nk / 128 + batch) * kv_heads;
  return busy >= 256 ? 1 : (int)std::min((long)heads / kv_heads, (512 + busy - 1) / busy);
}

extern "C" long i2r_packed_attention_bwd_ws_bytes(int, int batch, int nq, int nk, int heads, int kv_heads, int dim,
                                                  int num_buckets) {
  if (batch <= 0 || nq < 0 || nk < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || num_buckets < 0) return 0;
  const int parts = dkv_parts(batch, nk, heads, kv_heads);
  const long sums = (2 * (long)nq * heads + q_slots(nq, batch) * heads * num_buckets + 3) / 4 * 4;
  return (sums + (parts > 1 ? 2L * parts * nk * kv_heads * dim : 0)) * 4;
}

extern "C" int i2r_packed_attention_bwd(const i2r_packed_seqs* seqs, const void* q, const void* k, const void* v,
                                        const float* table, const float* out32, const float* stats, const void* dout,
                                        void* dq, void* dk, void* dv, float* dtable, void* ws, long ws_bytes, int dtype,
                                        int nq, int nk, int heads, int kv_heads, int dim, long q_row, long q_head, long k_row,
                                        long k_head, long v_row, long v_head, float scale, i2r_stream_t stream) {
  if (int rc = check("packed_attention_bwd", seqs, q, k, v, table, dtype, nq, nk, heads, kv_heads, dim,
                     {q_row, q_head, k_row, k_head, v_row, v_head}))
    return rc;
  I2R_REQUIRE((out32 && stats && dout) || !nq, "packed_attention_bwd: out32, stats and dout are required");
  I2R_REQUIRE(((uintptr_t)out32 | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0,
              "packed_attention_bwd: tensors have to be 16-byte aligned");
  I2R_REQUIRE(!dk == !dv, "packed_attention_bwd: dk and dv come together");
  I2R_REQUIRE((long)heads * dim < 1 << 22, "packed_attention_bwd: more than 2^22 elements a row");
  I2R_REQUIRE(table || !dtable, "packed_attention_bwd: dtable without a table");
  const int nb = dtable ? seqs->num_buckets : 0;
  const long need = i2r_packed_attention_bwd_ws_bytes(dtype, seqs->batch, nq, nk, heads, kv_heads, dim, nb);
  I2R_REQUIRE(ws_bytes >= need && (ws || !need) && (uintptr_t)ws % 16 == 0,
              "packed_attention_bwd: workspace of %ld bytes, %ld are needed, 16-byte aligned", ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  PaArgs a = {};
  a.s = *seqs;
  a.q = q, a.k = k, a.v = v, a.table = table, a.out32_in = out32, a.stats = (float*)stats, a.dout = dout;
  a.dq = dq, a.dk = dk, a.dv = dv, a.delta = (float*)ws, a.part = dtable ? (float*)ws + 2 * (long)nq * heads : nullptr;
  a.nq = nq, a.nk = nk, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.scale = scale;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  a.parts = dkv_parts(seqs->batch, nk, heads, kv_heads);
  a.dkv_part = (float*)ws + (2 * (long)nq * heads + q_slots(nq, seqs->batch) * heads * nb + 3) / 4 * 4;
  const bool need_dq = nq && (dq || dtable), need_dkv = nk && dk;
  if (nq && need_dkv && !need_dq) {
    const dim3 grid(i2r_cdiv((long)nq * heads, 128));
    if (dtype == 0) hipLaunchKernelGGL(pa_delta_kernel<float>, grid, dim3(256), 0, st, a);
    else if (dtype == 1) hipLaunchKernelGGL(pa_delta_kernel<f16_t>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(pa_delta_kernel<bf16_t>, grid, dim3(256), 0, st, a);
  }
  if (need_dq && !pa_launch_dq(dtype, a, st)) return I2R_ERR_HIP;
  if (need_dkv && !pa_launch_dkv(dtype, a, st)) return I2R_ERR_HIP;
  if (dtable)
    hipLaunchKernelGGL(pa_dtable_kernel, dim3(heads, nb), dim3(256), 0, st, a.part, dtable, nq ? q_slots(nq, seqs->batch) : 0,
                       heads, nb);
  return i2r_check_launch("packed_attention_bwd");
}
