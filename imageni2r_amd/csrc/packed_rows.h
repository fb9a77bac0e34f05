// Packed sequences on the device: where a row belongs, and the operators of one row, one wave each.
//
// The row functions are the definition written out: a lane is a key (or a query, for dk / dv), a hidden pair is skipped
// and never multiplied by zero, every sum is fp32.
#pragma once
#include "packed_common.h"

struct PaArgs {
  i2r_packed_seqs s;
  const void *q, *k, *v, *dout;
  const float *table, *out32_in;
  void *out, *dq, *dk, *dv;
  float *out32, *stats, *delta, *part, *dkv_part;
  int nq, nk, heads, kv_heads, dim, zero_outside, parts;
  long q_row, q_head, k_row, k_head, v_row, v_head;
  float scale;
};

__device__ __forceinline__ int pa_clamp(int x, int n) { return min(max(x, 0), n); }

// Rows lie in batch + 2 spans: those before the first sequence, the sequences, those behind the last.  Span i starts at
// row S_i and takes the tiles from S_i / size + i on: one more than it can need, so that the tile a workgroup works on
// follows from the starts alone -- no count of tiles, no list of them, nothing from the host.
// -> the span of tile `slot` (wave-uniform; every lane of the wave calls), its first row in `start`.
__device__ __forceinline__ int pa_span(const int* cu, int batch, int n, int shift, long slot, int& start) {
  const int lane = threadIdx.x & 63;
  int count = 1;  // span 0 starts at row 0
  for (int i0 = 0; i0 <= batch; i0 += 64) {
    int i = i0 + lane;
    bool before = false;
    if (i <= batch) before = (long)(pa_clamp(cu[i], n) >> shift) + i + 1 <= slot;
    count += __popcll(__ballot(before));
  }
  start = count == 1 ? 0 : pa_clamp(cu[count - 2], n);
  return count - 1;
}

// the sequence that a row (of some sequence) belongs to: the last that starts at or before it (every lane of the wave calls)
__device__ __forceinline__ int pa_seq_of(const int* cu, int batch, int n, int row) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int i0 = 0; i0 < batch; i0 += 64) count += __popcll(__ballot(i0 + lane < batch && pa_clamp(cu[i0 + lane], n) <= row));
  return max(count - 1, 0);
}

struct PaSeq {
  int q0, lq, k0, lk;  // first row and length among the queries, and among the keys
};

__device__ __forceinline__ PaSeq pa_seq(const i2r_packed_seqs& s, int nq, int nk, int b) {
  PaSeq r;
  r.q0 = pa_clamp(s.cu_q[b], nq);
  r.lq = max(pa_clamp(s.cu_q[b + 1], nq) - r.q0, 0);
  r.k0 = pa_clamp(s.cu_k[b], nk);
  r.lk = max(pa_clamp(s.cu_k[b + 1], nk) - r.k0, 0);
  if (s.len_k) r.lk = min(max(s.len_k[b], 0), r.lk);
  return r;
}

__device__ __forceinline__ int pa_pos_q(const i2r_packed_seqs& s, const PaSeq& w, int i) {
  return s.pos_q ? s.pos_q[w.q0 + i] : i + w.lk - w.lq;
}
__device__ __forceinline__ int pa_pos_k(const i2r_packed_seqs& s, const PaSeq& w, int j) {
  return s.pos_k ? s.pos_k[w.k0 + j] : j;
}

template <typename T>
__device__ __forceinline__ float pa_dot(const T* a, const T* b, int dim) {
  float acc = 0.0f;
  for (int d = 0; d < dim; d += 8) {
    float x[8], y[8];
    load8(a + d, x);
    load8(b + d, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = fmaf(x[i], y[i], acc);
  }
  return acc;
}

// Score of (query i, key j) in log2 units; `bucket` is set when there is a bias.
template <typename T>
__device__ __forceinline__ float pa_score(const PaArgs& a, const PaSeq& w, int h, const T* qi, const T* kj, int pos_q, int j,
                                          int& bucket) {
  float b = 0.0f;
  bucket = 0;
  if (a.table) {
    bucket = min((int)a.s.lut[pa_entry(pa_apart(pa_pos_k(a.s, w, j), pos_q), a.s.max_distance)], a.s.num_buckets - 1);
    b = pa_log2_units(a.table[(long)h * a.s.num_buckets + bucket]);
    if (b == -INFINITY) return b;  // hidden, whatever the key holds
  }
  return fmaf(pa_dot(qi, kj, a.dim), a.scale * PA_LOG2E, b);
}

// out, out32 and stats of query i, head h.
template <typename T>
__device__ __forceinline__ void pa_row_fwd(const PaArgs& a, const PaSeq& w, int i, int h) {
  const int lane = threadIdx.x & 63, g = h / (a.heads / a.kv_heads);
  const long row = w.q0 + i;
  const T* qi = (const T*)a.q + row * a.q_row + h * a.q_head;
  const int seen = a.s.causal ? min(i + w.lk - w.lq + 1, w.lk) : w.lk;
  const int pos_q = a.table ? pa_pos_q(a.s, w, i) : 0;
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  bool any = false;
  for (int j0 = 0; j0 < seen; j0 += 64) {
    const int j = j0 + lane;
    int bucket;
    float x = -INFINITY;
    if (j < seen)
      x = pa_score(a, w, h, qi, (const T*)a.k + (long)(w.k0 + j) * a.k_row + g * a.k_head, pos_q, j, bucket);
    unsigned long long open = __ballot(!(x == -INFINITY));
    if (!open) continue;
    any = true;
    const float mn = fmaxf(m, wave_max(x)), fall = m == -INFINITY ? 0.0f : exp2f(m - mn);
    const float p = x == -INFINITY ? 0.0f : exp2f(x - mn);
    l = l * fall + wave_sum(p);
    o0 *= fall;
    o1 *= fall;
    m = mn;
    for (; open; open &= open - 1) {
      const int t = __ffsll(open) - 1;
      const float pt = __shfl(p, t, 64);
      const T* vj = (const T*)a.v + (long)(w.k0 + j0 + t) * a.v_row + g * a.v_head;
      if (lane < a.dim) o0 = fmaf(pt, (float)vj[lane], o0);
      if (lane + 64 < a.dim) o1 = fmaf(pt, (float)vj[lane + 64], o1);
    }
  }
  const float r = any ? 1.0f / l : 0.0f;
  const long at = (row * a.heads + h) * a.dim;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int d = lane + 64 * c;
    const float o = (c ? o1 : o0) * r;
    if (d >= a.dim) continue;
    ((T*)a.out)[at + d] = (T)o;
    if (a.out32) a.out32[at + d] = o;
  }
  if (a.stats && lane == 0) {  // p = exp2(score - stats[0] - stats[1]); a row without keys: 0
    a.stats[(long)h * a.nq + row] = any ? m : 0.0f;
    a.stats[(long)(a.heads + h) * a.nq + row] = any ? log2f(l) : INFINITY;
  }
}

// p and ds of one pair
template <typename T>
__device__ __forceinline__ void pa_pair(const PaArgs& a, float x, long row, int h, const T* doi, const T* vj, float& p,
                                        float& ds) {
  const long at = (long)h * a.nq + row;
  p = exp2f((x - a.stats[at]) - a.stats[at + (long)a.heads * a.nq]);
  ds = p * (pa_dot(doi, vj, a.dim) - a.delta[at]);
}

// dq of query i, head h; with `hist` (a lane's column of it, 64 apart) its ds by bucket too, each lane's keys to its own column.
template <typename T>
__device__ __forceinline__ void pa_row_dq(const PaArgs& a, const PaSeq& w, int i, int h, float* hist = nullptr) {
  const int lane = threadIdx.x & 63, g = h / (a.heads / a.kv_heads);
  const long row = w.q0 + i, at = (row * a.heads + h) * a.dim;
  const T* qi = (const T*)a.q + row * a.q_row + h * a.q_head;
  const T* doi = (const T*)a.dout + at;
  const int seen = a.s.causal ? min(i + w.lk - w.lq + 1, w.lk) : w.lk;
  const int pos_q = a.table ? pa_pos_q(a.s, w, i) : 0;
  float d0 = 0.0f, d1 = 0.0f;
  for (int j0 = 0; j0 < seen; j0 += 64) {
    const int j = j0 + lane;
    int bucket = 0;
    float x = -INFINITY, p = 0.0f, ds = 0.0f;
    if (j < seen) {
      x = pa_score(a, w, h, qi, (const T*)a.k + (long)(w.k0 + j) * a.k_row + g * a.k_head, pos_q, j, bucket);
      if (!(x == -INFINITY)) {
        pa_pair(a, x, row, h, doi, (const T*)a.v + (long)(w.k0 + j) * a.v_row + g * a.v_head, p, ds);
        if (hist) hist[bucket * 64] += ds / Lift<T>::DOWN;
      }
    }
    for (unsigned long long open = __ballot(!(x == -INFINITY)); open; open &= open - 1) {
      const int t = __ffsll(open) - 1;
      const float dt = __shfl(ds, t, 64);
      const T* kj = (const T*)a.k + (long)(w.k0 + j0 + t) * a.k_row + g * a.k_head;
      if (lane < a.dim) d0 = fmaf(dt, (float)kj[lane], d0);
      if (lane + 64 < a.dim) d1 = fmaf(dt, (float)kj[lane + 64], d1);
    }
  }
  if (a.dq) {
    if (lane < a.dim) ((T*)a.dq)[at + lane] = (T)(d0 * a.scale);
    if (lane + 64 < a.dim) ((T*)a.dq)[at + lane + 64] = (T)(d1 * a.scale);
  }
}

// dk and dv of key j (which has to be one of the sequence's keys), key / value head g.
template <typename T>
__device__ __forceinline__ void pa_row_dkv(const PaArgs& a, const PaSeq& w, int j, int g) {
  const int lane = threadIdx.x & 63, group = a.heads / a.kv_heads;
  const T* kj = (const T*)a.k + (long)(w.k0 + j) * a.k_row + g * a.k_head;
  const T* vj = (const T*)a.v + (long)(w.k0 + j) * a.v_row + g * a.v_head;
  const int first = a.s.causal ? max(j - (w.lk - w.lq), 0) : 0;
  float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
  for (int h = g * group; h < (g + 1) * group; ++h)
    for (int i0 = first; i0 < w.lq; i0 += 64) {
      const int i = i0 + lane;
      float x = -INFINITY, p = 0.0f, ds = 0.0f;
      if (i < w.lq) {
        int bucket;
        const long row = w.q0 + i;
        x = pa_score(a, w, h, (const T*)a.q + row * a.q_row + h * a.q_head, kj, a.table ? pa_pos_q(a.s, w, i) : 0, j,
                     bucket);
        if (!(x == -INFINITY)) pa_pair(a, x, row, h, (const T*)a.dout + (row * a.heads + h) * a.dim, vj, p, ds);
      }
      for (unsigned long long open = __ballot(!(x == -INFINITY)); open; open &= open - 1) {
        const int t = __ffsll(open) - 1;
        const long row = w.q0 + i0 + t;
        const float pt = __shfl(p, t, 64), dt = __shfl(ds, t, 64);
        const T* qi = (const T*)a.q + row * a.q_row + h * a.q_head;
        const T* doi = (const T*)a.dout + (row * a.heads + h) * a.dim;
        if (lane < a.dim) v0 = fmaf(pt, (float)doi[lane], v0), k0 = fmaf(dt, (float)qi[lane], k0);
        if (lane + 64 < a.dim) v1 = fmaf(pt, (float)doi[lane + 64], v1), k1 = fmaf(dt, (float)qi[lane + 64], k1);
      }
    }
  const long at = ((long)(w.k0 + j) * a.kv_heads + g) * a.dim;
  if (lane < a.dim) ((T*)a.dk)[at + lane] = (T)(k0 * a.scale), ((T*)a.dv)[at + lane] = (T)v0;
  if (lane + 64 < a.dim) ((T*)a.dk)[at + lane + 64] = (T)(k1 * a.scale), ((T*)a.dv)[at + lane + 64] = (T)v1;
}
