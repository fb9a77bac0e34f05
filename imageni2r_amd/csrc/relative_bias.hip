// The relative position bias as a dense (heads, queries, keys) tensor, and its table's gradient.
//
// Bound by writing, or reading, the dense tensor once.  A thread takes 8 neighbouring keys of a query: their bucket numbers
// are looked up once for all heads (forward) and are mostly one and the same, so that the gradient's 8 terms are added in
// registers and seldom reach the histogram.  Measured, 16 x 2048 x 2048 in bf16: forward 29 us (4.6 TB/s), gradient 41 + 4 us
// (3.0 TB/s; torch's sum of a large tensor reads 4.0).
#include "packed_common.h"

struct BiasArgs {
  const float* table;
  const unsigned char* lut;
  const int *pos_q, *pos_k;
  int heads, nq, nk, nb, far;
  int groups, lanes;  // groups of 8 keys of a query; threads of a workgroup that stand side by side on one query
};

#define GROUP 8
constexpr int DEEP = 4;    // queries whose terms a thread of the gradient has on their way at a time
constexpr int HEADS = 32;  // of a workgroup in the forward: what its table in LDS holds
constexpr int AHEAD = 8;   // places of the LDS bucket list on both sides beyond max_distance

// The bucket numbers by distance in LDS; 8 more places on both sides, so that 8 neighbouring keys' are neighbours there.
__device__ __forceinline__ void load_lut(unsigned char* lut, const BiasArgs& a) {
  for (int n = threadIdx.x; n <= 2 * (a.far + AHEAD); n += blockDim.x)
    lut[n] = (unsigned char)min((int)a.lut[min(max(n - AHEAD, 0), 2 * a.far)], a.nb - 1);
}

__device__ __forceinline__ void buckets_of(const BiasArgs& a, const unsigned char* lut, int i, int j, int (&b)[GROUP]) {
  if (a.pos_k) {
    const int pos_q = a.pos_q[i];
#pragma unroll
    for (int e = 0; e < GROUP; ++e) b[e] = lut[AHEAD + pa_entry(pa_apart(a.pos_k[min(j + e, a.nk - 1)], pos_q), a.far)];
  } else {
    const unsigned char* at = lut + min(max(j - (i + a.nk - a.nq), -a.far - GROUP), a.far) + a.far + AHEAD;
#pragma unroll
    for (int e = 0; e < GROUP; ++e) b[e] = at[e];
  }
}

// VEC: all rows begin on 16 bytes
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void relative_bias_fwd_kernel(BiasArgs a, T* out, int rows) {
  __shared__ float table[HEADS * PA_MAX_BUCKETS];
  __shared__ unsigned char lut[2 * (PA_MAX_DISTANCE + AHEAD) + 1];
  const int h0 = blockIdx.z * HEADS, heads = min(a.heads - h0, HEADS);
  for (int n = threadIdx.x; n < heads * a.nb; n += 256) table[n] = a.table[(long)h0 * a.nb + n];
  load_lut(lut, a);
  __syncthreads();
  const int lane = threadIdx.x % a.lanes, side = 256 / a.lanes, j = (blockIdx.y * a.lanes + lane) * GROUP;
  if (j >= a.nk) return;
  const int i1 = min((int)(blockIdx.x + 1) * rows, a.nq);
  for (int i = blockIdx.x * rows + threadIdx.x / a.lanes; i < i1; i += side) {
    int b[GROUP];
    buckets_of(a, lut, i, j, b);
    int one = true;
#pragma unroll
    for (int e = 1; e < GROUP; ++e) one &= (int)(b[e] == b[0]);
    const bool same = __all(one);
    for (int h = 0; h < heads; ++h) {
      float x[GROUP];
      x[0] = table[h * a.nb + b[0]];
#pragma unroll
      for (int e = 1; e < GROUP; ++e) x[e] = same ? x[0] : table[h * a.nb + b[e]];
      T* to = out + ((long)(h0 + h) * a.nq + i) * a.nk + j;
      if (VEC) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int c = 0; c < GROUP / N; ++c) {
          if (j + c * N >= a.nk) break;
          vec y;
#pragma unroll
          for (int e = 0; e < N; ++e) y[e] = (T)x[c * N + e];
          *(vec*)(to + c * N) = y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < GROUP; ++e)
          if (j + e < a.nk) to[e] = (T)x[e];
      }
    }
  }
}

// A workgroup sums some rows of one head by bucket, a column of the histogram for each thread (a read, an addition and a
// write: no other thread touches it), then over the threads.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void relative_bias_bwd_kernel(BiasArgs a, const T* dout, float* part, int rows) {
  extern __shared__ float hist[];
  __shared__ unsigned char lut[2 * (PA_MAX_DISTANCE + AHEAD) + 1];
  const int t = threadIdx.x, h = blockIdx.y;
  float* mine = hist + t;
  for (int c = 0; c < a.nb; ++c) mine[c * 256] = 0.0f;
  load_lut(lut, a);
  __syncthreads();
  const int lane = t % a.lanes, side = 256 / a.lanes, i1 = min((int)(blockIdx.x + 1) * rows, a.nq);
  const int low = lut[0], high = lut[2 * (a.far + AHEAD)];
  int now = 0;        // the bucket that is being added up in a register, and its sum
  float sum = 0.0f;
  for (int g = lane; g < a.groups; g += a.lanes) {
    const int j = g * GROUP;
    for (int i0 = blockIdx.x * rows + t / a.lanes; i0 < i1; i0 += DEEP * side) {
      // (unconverted until all are on their way)
      T raw[DEEP][GROUP];
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const T* from = dout + ((long)h * a.nq + min(i0 + u * side, i1 - 1)) * a.nk + j;
        if (VEC) {  // (of a last group of fp32 half may be there)
          typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
          constexpr int N = 16 / sizeof(T);
#pragma unroll
          for (int c = 0; c < GROUP / N; ++c) *(vec*)(raw[u] + c * N) = *(const vec*)(from + (j + c * N < a.nk ? c * N : 0));
        } else {
#pragma unroll
          for (int e = 0; e < GROUP; ++e) raw[u][e] = from[min(e, a.nk - 1 - j)];
        }
      }
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const int i = i0 + u * side;
        if (i >= i1) break;
        float x[GROUP];
#pragma unroll
        for (int e = 0; e < GROUP; ++e) x[e] = j + e < a.nk ? (float)raw[u][e] : 0.0f;
        int b[GROUP], one = true;
        const int apart = j - (i + a.nk - a.nq);
        if (!a.pos_k && __all((int)(apart >= a.far) | (int)(apart + GROUP - 1 <= -a.far))) {
          b[0] = apart > 0 ? high : low;  // all of the wave's beyond max_distance: nothing to look up
        } else {
          buckets_of(a, lut, i, j, b);
#pragma unroll
          for (int e = 1; e < GROUP; ++e) one &= (int)(b[e] == b[0]) | (int)(j + e >= a.nk);
        }
        if (one) {
          const float s = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
          if (b[0] != now) {
            mine[now * 256] += sum;
            now = b[0], sum = s;
          } else {
            sum += s;
          }
        } else {
#pragma unroll
          for (int e = 0; e < GROUP; ++e)
            if (j + e < a.nk) mine[b[e] * 256] += x[e];
        }
      }
    }
  }
  mine[now * 256] += sum;
  __syncthreads();
  // some threads for each bucket, each a stride of its 256 sums (from another place for each bucket: other banks)
  int each = 1;
  while (2 * each * a.nb <= 256) each *= 2;
  const int c = t / each, first = t % each;
  float s = 0.0f;
  if (c < a.nb)
    for (int k = 0; k < 256; k += each) s += hist[c * 256 + ((k + first + c * each) & 255)];
  for (int o = each / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (c < a.nb && first == 0) part[((long)blockIdx.x * a.heads + h) * a.nb + c] = s;
}

// (with one part, or none, the workgroups' sums are the gradient)
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
  I2R_REQUIRE(heads > 0 && heads < 65536 && nq >= 0 && nk >= 0 && nq < 1 << 30 && nk < 1 << 30, "%s: bad sizes", what);
  I2R_REQUIRE(lut && nb > 0 && nb <= PA_MAX_BUCKETS, "%s: %d buckets: 1 to %d are supported", what, nb, PA_MAX_BUCKETS);
  I2R_REQUIRE(max_distance >= 0 && max_distance <= PA_MAX_DISTANCE, "%s: distance %d: 0 to %d are supported", what,
              max_distance, PA_MAX_DISTANCE);
  I2R_REQUIRE(!pos_q == !pos_k, "%s: positions of queries and keys come together", what);
  return I2R_OK;
}

static BiasArgs bias_args(const float* table, const unsigned char* lut, const int* pos_q, const int* pos_k, int heads, int nq,
                          int nk, int nb, int far) {
  BiasArgs a = {table, lut, pos_q, pos_k, heads, nq, nk, nb, far, i2r_cdiv(nk, GROUP), 1};
  while (a.lanes < 256 && a.lanes < a.groups) a.lanes *= 2;
  return a;
}

extern "C" int i2r_relative_bias_fwd(const float* table, const unsigned char* lut, const int* pos_q, const int* pos_k,
                                     void* out, int dtype, int heads, int nq, int nk, int num_buckets, int max_distance,
                                     i2r_stream_t stream) {
  if (int rc = check("relative_bias_fwd", lut, pos_q, pos_k, dtype, heads, nq, nk, num_buckets, max_distance)) return rc;
  if (nq == 0 || nk == 0) return I2R_OK;
  I2R_REQUIRE(table && out, "relative_bias_fwd: null tensor");
  hipStream_t st = (hipStream_t)stream;
  const BiasArgs a = bias_args(table, lut, pos_q, pos_k, heads, nq, nk, num_buckets, max_distance);
  const int side = 256 / a.lanes, columns = i2r_cdiv(a.groups, a.lanes), chunks = i2r_cdiv(heads, HEADS);
  I2R_REQUIRE(columns < 65536, "relative_bias_fwd: %d keys are too many", nk);
  // about 2048 workgroups (8 for each CU), each with a few queries a thread
  const int rows = std::max(1, (int)((long)nq * columns * chunks / ((long)side * 2048))) * side;
  const dim3 grid(i2r_cdiv(nq, rows), columns, chunks);
  const bool vec = (long)nk * (dtype == 0 ? 4 : 2) % 16 == 0 && (uintptr_t)out % 16 == 0;
#define RB_FWD(T)                                                                                              \
  if (vec) hipLaunchKernelGGL((relative_bias_fwd_kernel<T, true>), grid, dim3(256), 0, st, a, (T*)out, rows);  \
  else hipLaunchKernelGGL((relative_bias_fwd_kernel<T, false>), grid, dim3(256), 0, st, a, (T*)out, rows);
  if (dtype == 0) { RB_FWD(float) }
  else if (dtype == 1) { RB_FWD(f16_t) }
  else { RB_FWD(bf16_t) }
  return i2r_check_launch("relative_bias_fwd");
}

// queries of a workgroup: 32 K terms and more, so that the histogram is worth its clearing, and about 1024 workgroups: four on
// a CU, all at once
static int bwd_rows(int heads, int nq, int nk) {
  const long row = std::max(nk, 1), most = std::max(1L, 32768 / row), few = (long)nq * heads / 1024;
  return (int)std::min((long)std::max(nq, 1), std::max(most, few));
}

extern "C" long i2r_relative_bias_bwd_ws_bytes(int heads, int nq, int nk, int num_buckets) {
  if (heads <= 0 || nq <= 0 || nk <= 0 || num_buckets <= 0) return 0;
  const int parts = i2r_cdiv(nq, bwd_rows(heads, nq, nk));
  return parts > 1 ? (long)parts * heads * num_buckets * 4 : 0;
}

extern "C" int i2r_relative_bias_bwd(const void* dout, const unsigned char* lut, const int* pos_q, const int* pos_k,
                                     float* dtable, void* ws, long ws_bytes, int dtype, int heads, int nq, int nk,
                                     int num_buckets, int max_distance, i2r_stream_t stream) {
  if (int rc = check("relative_bias_bwd", lut, pos_q, pos_k, dtype, heads, nq, nk, num_buckets, max_distance)) return rc;
  I2R_REQUIRE(dtable && (dout || !nq || !nk), "relative_bias_bwd: null tensor");
  const long need = i2r_relative_bias_bwd_ws_bytes(heads, nq, nk, num_buckets);
  I2R_REQUIRE(ws_bytes >= need && (ws || !need), "relative_bias_bwd: workspace of %ld bytes, %ld are needed", ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  const BiasArgs a = bias_args(nullptr, lut, pos_q, pos_k, heads, nq, nk, num_buckets, max_distance);
  const int rows = bwd_rows(heads, nq, nk), parts = nq && nk ? i2r_cdiv(nq, rows) : 0, lds = num_buckets * 256 * 4;
  const bool vec = (long)nk * (dtype == 0 ? 4 : 2) % 16 == 0 && (uintptr_t)dout % 16 == 0;
  float* part = parts > 1 ? (float*)ws : dtable;
  const dim3 grid(parts, heads);
#define RB_BWD(T)                                                                                                          \
  {                                                                                                                        \
    static bool done[2][64];                                                                                               \
    const void* kern = vec ? (const void*)relative_bias_bwd_kernel<T, true> : (const void*)relative_bias_bwd_kernel<T, false>; \
    if (!i2r_lds_attr(kern, PA_MAX_BUCKETS * 256 * 4, done[vec])) return I2R_ERR_HIP;                                      \
    if (vec) hipLaunchKernelGGL((relative_bias_bwd_kernel<T, true>), grid, dim3(256), lds, st, a, (const T*)dout, part, rows); \
    else hipLaunchKernelGGL((relative_bias_bwd_kernel<T, false>), grid, dim3(256), lds, st, a, (const T*)dout, part, rows); \
  }
  if (parts > 0) {
    if (dtype == 0) RB_BWD(float)
    else if (dtype == 1) RB_BWD(f16_t)
    else RB_BWD(bf16_t)
  }
  if (parts != 1)
    hipLaunchKernelGGL(relative_bias_join_kernel, dim3(heads, num_buckets), dim3(64), 0, st, part, dtable, parts, heads,
                       num_buckets);
  return i2r_check_launch("relative_bias_bwd");
}
