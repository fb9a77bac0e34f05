// The relative position bias as a dense (heads, queries, keys) tensor, and its table's gradient.
#include "packed_common.h"

// One thread for each (query, key).
template <typename T>
__global__ __launch_bounds__(256) void relative_bias_fwd_kernel(const float* table, const unsigned char* lut, const int* pos_q,
                                                                const int* pos_k, T* out, int heads, int nq, int nk, int nb,
                                                                int max_distance) {
  const long n = (long)nq * nk;
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long)gridDim.x * 256) {
    const int i = at / nk, j = at % nk;
    const int apart = pa_apart(pos_k ? pos_k[j] : j, pos_q ? pos_q[i] : i + nk - nq);
    const int bucket = lut[pa_entry(apart, max_distance)];
    for (int h = 0; h < heads; ++h) out[h * n + at] = (T)table[(long)h * nb + bucket];
  }
}

// A workgroup sums some rows of one head by bucket, a column of the histogram for each thread; then the parts are summed.
template <typename T>
__global__ __launch_bounds__(256) void relative_bias_bwd_kernel(const T* dout, const unsigned char* lut, const int* pos_q,
                                                                const int* pos_k, float* part, int nq, int nk, int nb,
                                                                int max_distance, int rows) {
  extern __shared__ float hist[];
  const int t = threadIdx.x, h = blockIdx.y;
  for (int c = 0; c < nb; ++c) hist[c * 256 + t] = 0.0f;
  const int i0 = blockIdx.x * rows;
  for (int i = i0; i < min(i0 + rows, nq); ++i) {
    const int pq = pos_q ? pos_q[i] : i + nk - nq;
    const T* row = dout + ((long)h * nq + i) * nk;
    for (int j = t; j < nk; j += 256)
      hist[lut[pa_entry(pa_apart(pos_k ? pos_k[j] : j, pq), max_distance)] * 256 + t] += (float)row[j];
  }
  __syncthreads();
  for (int c = t >> 6; c < nb; c += 4) {
    float s = 0.0f;
    for (int w = 0; w < 4; ++w) s += hist[c * 256 + w * 64 + (t & 63)];
    s = wave_sum(s);
    if ((t & 63) == 0) part[((long)blockIdx.x * gridDim.y + h) * nb + c] = s;
  }
}

__global__ __launch_bounds__(64) void relative_bias_join_kernel(const float* part, float* dtable, int parts, int heads,
                                                                int nb) {
  const int h = blockIdx.x, c = blockIdx.y;
  float s = 0.0f;
  for (int p = threadIdx.x; p < parts; p += 64) s += part[((long)p * heads + h) * nb + c];
  s = wave_sum(s);
  if (threadIdx.x == 0) dtable[(long)h * nb + c] = s;
}

static int check(const char* what, const unsigned char* lut, const int* pos_q, const int* pos_k, int dtype, int heads, int nq,
                 int nk, int nb, int max_distance) {
  I2R_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d is not 0 (fp32), 1 (fp16) or 2 (bf16)", what, dtype);
  I2R_REQUIRE(heads > 0 && heads < 65536 && nq >= 0 && nk >= 0, "%s: bad sizes", what);
  I2R_REQUIRE(lut && nb > 0 && nb <= PA_MAX_BUCKETS, "%s: %d buckets: 1 to %d are supported", what, nb, PA_MAX_BUCKETS);
  I2R_REQUIRE(max_distance >= 0 && max_distance <= PA_MAX_DISTANCE, "%s: distance %d: 0 to %d are supported", what,
              max_distance, PA_MAX_DISTANCE);
  I2R_REQUIRE(!pos_q == !pos_k, "%s: positions of queries and keys come together", what);
  return I2R_OK;
}

extern "C" int i2r_relative_bias_fwd(const float* table, const unsigned char* lut, const int* pos_q, const int* pos_k,
                                     void* out, int dtype, int heads, int nq, int nk, int num_buckets, int max_distance,
                                     i2r_stream_t stream) {
  if (int rc = check("relative_bias_fwd", lut, pos_q, pos_k, dtype, heads, nq, nk, num_buckets, max_distance)) return rc;
  if (nq == 0 || nk == 0) return I2R_OK;
  I2R_REQUIRE(table && out, "relative_bias_fwd: null tensor");
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)std::min(((long)nq * nk + 255) / 256, 1L << 20));
#define RB_FWD(T)                                                                                                       \
  hipLaunchKernelGGL(relative_bias_fwd_kernel<T>, grid, dim3(256), 0, st, table, lut, pos_q, pos_k, (T*)out, heads, nq, nk, \
                     num_buckets, max_distance)
  if (dtype == 0) RB_FWD(float);
  else if (dtype == 1) RB_FWD(f16_t);
  else RB_FWD(bf16_t);
  return i2r_check_launch("relative_bias_fwd");
}

static int bwd_rows(int heads, int nq) { return std::max(1, (int)((long)nq * heads / 2048)); }

extern "C" long i2r_relative_bias_bwd_ws_bytes(int heads, int nq, int, int num_buckets) {
  if (heads <= 0 || nq <= 0 || num_buckets <= 0) return 0;
  return (long)i2r_cdiv(nq, bwd_rows(heads, nq)) * heads * num_buckets * 4;
}

extern "C" int i2r_relative_bias_bwd(const void* dout, const unsigned char* lut, const int* pos_q, const int* pos_k,
                                     float* dtable, void* ws, long ws_bytes, int dtype, int heads, int nq, int nk,
                                     int num_buckets, int max_distance, i2r_stream_t stream) {
  if (int rc = check("relative_bias_bwd", lut, pos_q, pos_k, dtype, heads, nq, nk, num_buckets, max_distance)) return rc;
  I2R_REQUIRE(dtable && (dout || !nq || !nk), "relative_bias_bwd: null tensor");
  I2R_REQUIRE(ws_bytes >= i2r_relative_bias_bwd_ws_bytes(heads, nq, nk, num_buckets) && (ws || !nq),
              "relative_bias_bwd: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  const int rows = bwd_rows(heads, nq), parts = nk ? i2r_cdiv(nq, rows) : 0, lds = num_buckets * 256 * 4;
  float* part = (float*)ws;
#define RB_BWD(T)                                                                                                  \
  hipLaunchKernelGGL(relative_bias_bwd_kernel<T>, dim3(parts, heads), dim3(256), lds, st, (const T*)dout, lut, pos_q, \
                     pos_k, part, nq, nk, num_buckets, max_distance, rows)
  if (parts > 0) {
    if (dtype == 0) RB_BWD(float);
    else if (dtype == 1) RB_BWD(f16_t);
    else RB_BWD(bf16_t);
  }
  hipLaunchKernelGGL(relative_bias_join_kernel, dim3(heads, num_buckets), dim3(64), 0, st, part, dtable, parts, heads,
                     num_buckets);
  return i2r_check_launch("relative_bias_bwd");
}
