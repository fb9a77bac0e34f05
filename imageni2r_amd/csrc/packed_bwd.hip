// Backward of packed-sequence attention on the matrix cores.
//
// Two kernels, both recomputing the scores: dq (a query a column, keys pass by) and dk / dv (a key a column, the queries of
// all heads of its group pass by).  Seven products where five would do with dq added up atomically -- but no float is ever
// added in an order that could change, and nothing but the outputs is written.
#include "packed_tiles.h"

// Adds four keys' ds to the lane's column of the histogram, those of one bucket first: neighbours mostly share one, and a
// read, an addition and a write cost the LDS less than ds_add_f32 (192 cycles an instruction of 64 lanes, measured,
// against 7 for the integer one).  No other lane touches the column, so nothing has to be atomic.
__device__ __forceinline__ void add_four(float* mine, const Entry* e, const float* x) {
  const int b0 = e[0].bucket, b1 = e[1].bucket, b2 = e[2].bucket, b3 = e[3].bucket;
  const int same1 = b1 == b0, same2 = b2 == b0, same3 = b3 == b0;
  const int last1 = (b1 == b3) & ~same1, last2 = (b2 == b3) & ~same2;
  const float s0 = ((x[0] + (same1 ? x[1] : 0.0f)) + (same2 ? x[2] : 0.0f)) + (same3 ? x[3] : 0.0f);
  const float s3 = (x[3] + (last1 ? x[1] : 0.0f)) + (last2 ? x[2] : 0.0f);
  const float h0 = mine[b0 * 64], h3 = mine[b3 * 64];
  mine[b0 * 64] = h0 + s0;
  if (!same3) mine[b3 * 64] = h3 + s3;
  const int alone1 = !(same1 | last1), alone2 = !(same2 | last2);
  if (__any(alone1 | alone2)) {
    if (alone1) mine[b1 * 64] += x[1];
    if (alone2) mine[b2 * 64] += x[2];
  }
}

template <typename T, int DP>
struct DqShape {
  static constexpr int WAVES = 4, ROWS = 32 * WAVES, KEYS = sizeof(T) == 4 ? 32 : 64;
  typedef Tile<T, DP, KEYS> Tl;
  static constexpr int BUFFER = 2 * Tl::BYTES + 256;  // k, v, positions
  static constexpr int PER_SIMD = sizeof(T) == 4 && DP == 128 ? 1 : 2, UNROLL = DP == 128 ? 1 : 2;
  static constexpr bool APART = DP == 128;  // the products' operands would not fit the registers all at once
  static int lds(bool bias, int max_distance, int buckets) {
    return 2 * BUFFER + (bias ? table_places(max_distance) * 8 + buckets * 64 * 4 * WAVES : 0);
  }
};

// dq of 32 queries a wave, delta = <dout, out> and the two stats' sum on the way for the other kernel, and ds summed by bucket: each lane its own column of a histogram
// in LDS, so that no two lanes add to one word.
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256, (DqShape<T, DP>::PER_SIMD)) void pa_dq_kernel(PaArgs a, long slots) {
  typedef DqShape<T, DP> S;
  typedef typename S::Tl Tl;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31,
            half = lane >> 5;
  long slot;
  int h, start;
  if (!tile_of(slots, a.heads, slot, h)) return;
  slot = slots - 1 - slot;
  const bool sums = BIAS && a.part;
  const int nb = a.s.num_buckets;
  const int span = pa_span(a.s.cu_q, a.s.batch, a.nq, 7, slot, start);
  const long row0 = start + ((slot - (start >> 7) - span) << 7);
  PaSeq w = {};
  if (span > 0 && span <= a.s.batch) w = pa_seq(a.s, a.nq, a.nk, span - 1);
  if (row0 >= w.q0 + w.lq) {
    if (span == 0 || span > a.s.batch) {  // rows of no sequence
      const int end = (int)min(row0 + S::ROWS, (long)(span == 0 ? pa_clamp(a.s.cu_q[0], a.nq) : a.nq));
      if (a.dq)
        for (long i = (row0 * a.dim) + threadIdx.x; i < (long)end * a.dim; i += 256)
          ((T*)a.dq)[(i / a.dim * a.heads + h) * a.dim + i % a.dim] = (T)0.0f;
    }
    if (sums && threadIdx.x < nb) a.part[(slot * a.heads + h) * nb + threadIdx.x] = 0.0f;
    return;
  }
  const int g = h / (a.heads / a.kv_heads);
  const int i0 = (int)(row0 - w.q0), iw = i0 + wave * 32, i = iw + col;
  const bool valid = i < w.lq;
  const int ahead = w.lk - w.lq;
  int keys = w.lk;
  if (a.s.causal) keys = min(keys, min(i0 + S::ROWS, w.lq) + ahead);

  Loader<T, DP, S::KEYS, S::WAVES> lk, lv;
  lk.init((const T*)a.k + (long)w.k0 * a.k_row + g * a.k_head, a.k_row, a.dim);
  lv.init((const T*)a.v + (long)w.k0 * a.v_row + g * a.v_head, a.v_row, a.dim);
  const int far = a.s.max_distance;
  Entry* by_distance = (Entry*)(lds + 2 * S::BUFFER);
  float* hist = (float*)(by_distance + table_places(far)) + wave * nb * 64;
  auto load = [&](int n) {
    char* b = lds + (n & 1) * S::BUFFER;
    lk.load(b, n * S::KEYS, keys);
    lv.load(b + Tl::BYTES, n * S::KEYS, keys);
    if (BIAS && a.s.pos_k) load_words(b + 2 * Tl::BYTES, a.s.pos_k + w.k0, n * S::KEYS, keys);
  };
  const int tiles = keys > 0 ? (keys + S::KEYS - 1) / S::KEYS : 0;
  if (tiles > 0) load(0);

  const long to = ((long)(w.q0 + i) * a.heads + h) * a.dim;
  frag_t<T> q[Tl::STEPS], dout[Tl::STEPS];
  load_rows<T>(q, (const T*)a.q + (long)(w.q0 + i) * a.q_row + h * a.q_head, valid, a.dim, half);
  load_rows<T>(dout, (const T*)a.dout + to, valid, a.dim, half);
  float delta = 0.0f;
  if (valid)
#pragma unroll
    for (int s = 0; s < Tl::STEPS; ++s) {
      constexpr int N = 16 / sizeof(T);
      const int d = (2 * s + half) * N;
      if (d < a.dim)
#pragma unroll
        for (int e = 0; e < N; ++e) delta = fmaf((float)dout[s][e], a.out32_in[to + d + e], delta);
    }
  delta += other_half(delta);
  const long st = (long)h * a.nq + w.q0 + i;
  const float m = valid ? a.stats[st] : 0.0f, ll = (valid ? a.stats[st + (long)a.heads * a.nq] : INFINITY) - Lift<T>::LOG2;
  const float ref = m + ll;
  if (valid && half == 0) a.delta[st] = delta, a.delta[st + (long)a.heads * a.nq] = ref;
  const float sc = a.scale * PA_LOG2E;
  const int pos_q = BIAS && valid ? pa_pos_q(a.s, w, i) : 0;
  if (BIAS) load_table(by_distance, a.s, a.table, h);
  if (BIAS)
    for (int c = 0; c < nb; ++c) hist[c * 64 + lane] = 0.0f;

  f32x16 dq[Tl::BLOCKS];
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b) dq[b] = (f32x16)0.0f;

  typename Tl::Lane at(lane);
  auto tile = [&](auto masked, auto mode, const char* kt, int j0) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(masked)::value;
    constexpr int MODE = decltype(mode)::value;
    const char* vt = kt + Tl::BYTES;
    at.fresh();
    const int last = a.s.causal ? min(keys, i + ahead + 1) : keys;
#pragma unroll S::UNROLL
    for (int kb = 0; kb < S::KEYS / 32; ++kb) {
      f32x16 x = (f32x16)0.0f, dp = (f32x16)0.0f;
#pragma unroll
      for (int s = 0; s < Tl::STEPS; ++s) mma_step(x, Tl::frag(kt, kb * 32, s, at), q[s]);
      if (S::APART) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < Tl::STEPS; ++s) mma_step(dp, Tl::frag(vt, kb * 32, s, at), dout[s]);
      if (S::APART) __builtin_amdgcn_sched_barrier(0);
      Entry e[MODE == NONE ? 1 : 16];
      float sum = 0.0f;
      if constexpr (MODE == NONE) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float ds = __builtin_amdgcn_exp2f(fmaf(x[r], sc, -ref)) * (dp[r] - delta);
          x[r] = MASK && !(j0 + kb * 32 + acc_row(r, half) < last) ? 0.0f : ds;
        }
      } else {
        e[0] = by_distance[j0 < iw + ahead ? 0 : 2 * (far + PAD)];
        const Entry* near = by_distance + (min(max(j0 + 4 * half - pos_q, -far - 60), far) + far + PAD);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = kb * 32 + acc_row(r, half);
          if (MODE == ONE) e[r] = e[0];
          if (MODE == NEAR) e[r] = near[kb * 32 + acc_row(r, 0)];
          if (MODE == GIVEN) e[r] = by_distance[PAD + pa_entry(pa_apart(((const int*)(vt + Tl::BYTES))[row], pos_q), far)];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          // hidden by its place or by its bucket: whatever the key and its value hold
          const float b = MASK && !(j0 + kb * 32 + acc_row(r, half) < last) ? -INFINITY : e[r].bias;
          const float p = __builtin_amdgcn_exp2f((fmaf(x[r], sc, b) - m) - ll);
          x[r] = b == -INFINITY ? 0.0f : p * (dp[r] - delta);
          sum += x[r];
        }
      }
      if (S::APART) __builtin_amdgcn_sched_barrier(0);
      Probs<T> ds;  // rounded to the type for the product: half a step each, as much as rounding dq once more
      ds.set(x);
#pragma unroll
      for (int b = 0; b < Tl::BLOCKS; ++b) Tl::mma_t(kt, kb * 32, b, at, ds, dq[b]);
      // (behind the products, which run meanwhile)
      if constexpr (MODE == ONE) {
        hist[e[0].bucket * 64 + lane] += sum;
      } else if constexpr (MODE != NONE) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float four[4] = {x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]};
          add_four(hist + lane, e + 4 * t, four);
        }
      }
    }
  };
  auto step = [&](int n) {
    tiles_ready();
    if (n + 1 < tiles) load(n + 1);
  };
  // (counts of tiles; the wave's queries iw .. iw + 31 lie at the keys' places + ahead)
  Passage way = {};
  const int whole = keys / S::KEYS;  // tiles with no row behind the last key
  const int end = iw >= w.lq ? 0 : a.s.causal ? min(tiles, floor_div(iw + 31 + ahead, S::KEYS) + 1) : tiles;
  way.near0 = way.near1 = way.far1 = max(end, 0);
  if constexpr (!BIAS) {
    way.far0 = max(0, min(end, a.s.causal ? min(whole, floor_div(iw + ahead + 1, S::KEYS)) : whole));
    walk(way, tiles, step, [&](int n) { tile(False(), Mode<NONE>(), lds + (n & 1) * S::BUFFER, n * S::KEYS); },
         [&](int n) { tile(True(), Mode<NONE>(), lds + (n & 1) * S::BUFFER, n * S::KEYS); });
  } else if (a.s.pos_q) {
    walk(way, tiles, step, [](int) {},
         [&](int n) { tile(True(), Mode<GIVEN>(), lds + (n & 1) * S::BUFFER, n * S::KEYS); });
  } else {
    way.far0 = max(0, min(min(end, whole), floor_div(iw + ahead - far + 1, S::KEYS)));
    if (!a.s.causal) {
      way.near0 = max(way.far0, min(end, -floor_div(-(far + iw + 31 + ahead), S::KEYS)));
      way.far1 = max(way.near0, min(end, whole));
    }
    walk(way, tiles, step, [&](int n) { tile(False(), Mode<ONE>(), lds + (n & 1) * S::BUFFER, n * S::KEYS); },
         [&](int n) { tile(True(), Mode<NEAR>(), lds + (n & 1) * S::BUFFER, n * S::KEYS); });
  }

  float finite = 0.0f;
  if (a.dq)
#pragma unroll
    for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int d = b * 32 + 8 * t + 4 * half;
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = dq[b][4 * t + e] * (a.scale * Lift<T>::DOWN);
          finite = fmaf(z, 0.0f, finite);
          y[e] = (T)z;
        }
        if (valid && d < a.dim) *(t4*)((T*)a.dq + to + d) = y;
      }
  if (sums) {
    __syncthreads();
    const float* all = (const float*)(by_distance + table_places(far));
    for (int c = wave; c < nb; c += S::WAVES) {
      float s = 0.0f;
      for (int v = 0; v < S::WAVES; ++v) s += all[(v * nb + c) * 64 + lane];
      s = wave_sum(s);
      if (lane == 0) a.part[(slot * a.heads + h) * nb + c] = s * Lift<T>::DOWN;
    }
  }
  // a hidden pair's 0 times NaN, or a lifted ds beyond fp16: pair by pair
  const unsigned long long again = __ballot(valid && !(finite == 0.0f));
  for (unsigned rows = (unsigned)again | (unsigned)(again >> 32); rows; rows &= rows - 1)
    pa_row_dq<T>(a, w, iw + __ffs(rows) - 1, h);
}

// The lane's column of a sum, times `factor`, to its row; -> whether any of it is not finite.
template <typename T, int BLOCKS>
__device__ __forceinline__ bool store_sum(const f32x16 (&sum)[BLOCKS], T* to, bool there, bool valid, float factor, int dim,
                                          int half) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  float finite = 0.0f;
  factor *= Lift<T>::DOWN;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int d = b * 32 + 8 * t + 4 * half;
      t4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = sum[b][4 * t + e] * factor;
        finite = fmaf(f, 0.0f, finite);
        y[e] = valid ? (T)f : (T)0.0f;
      }
      if (there && d < dim) *(t4*)(to + d) = y;
    }
  return !(finite == 0.0f);
}
template <typename T, int BLOCKS>
__device__ __forceinline__ void store_part(const f32x16 (&sum)[BLOCKS], float* to, bool there, bool valid, float factor,
                                           int dim, int half) {
  factor *= Lift<T>::DOWN;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int d = b * 32 + 8 * t + 4 * half;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = valid ? sum[b][4 * t + e] * factor : 0.0f;
      if (there && d < dim) *(f32x4*)(to + d) = y;
    }
}

// dk and dv of a (key, key / value head) from the parts of its group's heads, a wave each.
template <typename T>
__global__ __launch_bounds__(256) void pa_dkv_join_kernel(PaArgs a) {
  const int lane = threadIdx.x & 63;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6), all = (long)a.nk * a.kv_heads;
  if (item >= all) return;
  float finite = 0.0f;
  for (int d = lane; d < a.dim; d += 64) {
    float k = 0.0f, v = 0.0f;
    for (int p = 0; p < a.parts; ++p) {
      k += a.dkv_part[(2 * p * all + item) * a.dim + d];
      v += a.dkv_part[((2 * p + 1) * all + item) * a.dim + d];
    }
    finite = fmaf(k, 0.0f, fmaf(v, 0.0f, finite));
    ((T*)a.dk)[item * a.dim + d] = (T)k;
    ((T*)a.dv)[item * a.dim + d] = (T)v;
  }
  if (!__any(!(finite == 0.0f))) return;
  const int row = (int)(item / a.kv_heads);
  const PaSeq w = pa_seq(a.s, a.nq, a.nk, pa_seq_of(a.s.cu_k, a.s.batch, a.nk, row));
  if (row >= w.k0 && row < w.k0 + w.lk) pa_row_dkv<T>(a, w, row - w.k0, (int)(item % a.kv_heads));
}

// RG groups of waves share the keys: each takes its 32 rows of a tile of queries, and their sums are added at the end.  (Four
// waves with keys of their own are half as many workgroups, each twice as long: 286 us against 222 for eight documents of up
// to 2048 tokens, 16 heads of 64 over 4.)
template <typename T, int DP>
struct DkvShape {
  static constexpr int RG = 2;
  static constexpr int WAVES = 4, COLS = 32 * WAVES / RG, ROWS = sizeof(T) == 4 ? 32 * RG : 64, SPAN = ROWS / RG;
  typedef Tile<T, DP, ROWS> Tl;
  static constexpr int BUFFER = 2 * Tl::BYTES + 4 * 256;  // q, dout, delta, stats, positions
  static constexpr int PER_SIMD = DP == 128 ? 1 : 2, UNROLL = DP == 128 || sizeof(T) == 4 ? 1 : 2;
  static constexpr bool APART = DP * sizeof(T) >= 256;
  static constexpr int JOIN = 2 * COLS * (DP + 4) * 4;  // dk and dv of one group, where the tiles were
  static int lds(bool bias, int max_distance) {
    const int n = 2 * BUFFER + (bias ? table_places(max_distance) * 4 : 0);
    return n > JOIN ? n : JOIN;
  }
};

template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256, (DkvShape<T, DP>::PER_SIMD)) void pa_dkv_kernel(PaArgs a, long slots) {
  typedef DkvShape<T, DP> S;
  typedef typename S::Tl Tl;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31,
            half = lane >> 5;
  const int group = a.heads / a.kv_heads;
  long slot;
  int g, start;
  if (!tile_of(slots, a.kv_heads * a.parts, slot, g)) return;
  const int part = g % a.parts;  // of the group's heads
  g /= a.parts;
  constexpr int SHIFT = 6;
  const int span = pa_span(a.s.cu_k, a.s.batch, a.nk, SHIFT, slot, start);
  const long row0 = start + ((slot - (start >> SHIFT) - span) << SHIFT);
  const int end = span > a.s.batch ? a.nk : pa_clamp(a.s.cu_k[span], a.nk);  // of the span's rows, keys or not
  if (row0 >= end) return;
  PaSeq w = {};
  if (span > 0 && span <= a.s.batch) w = pa_seq(a.s, a.nq, a.nk, span - 1);
  const int kg = wave % 2, rg = wave / 2;  // the wave's keys and rows
  const int jg = (int)(row0 - start), jw = jg + kg * 32, j = jw + col;  // first key of workgroup, wave; lane's own
  const bool valid = j < w.lk;
  const int ahead = w.lk - w.lq;
  const int see = a.s.causal ? ahead : 1 << 30;  // key j is seen by queries i with j <= i + see
  const int first = a.s.causal ? max(jg - ahead, 0) : 0;  // first query that sees one of the workgroup's keys
  const int tiles = jg < w.lk && first < w.lq ? (w.lq - first + S::ROWS - 1) / S::ROWS : 0;
  const int far = a.s.max_distance;
  float* by_distance = (float*)(lds + 2 * S::BUFFER);

  frag_t<T> k[Tl::STEPS], v[Tl::STEPS];
  load_rows<T>(k, (const T*)a.k + (long)(w.k0 + j) * a.k_row + g * a.k_head, valid, a.dim, half);
  load_rows<T>(v, (const T*)a.v + (long)(w.k0 + j) * a.v_row + g * a.v_head, valid, a.dim, half);
  const float sc = a.scale * PA_LOG2E;
  const int pos_k = BIAS && valid ? pa_pos_k(a.s, w, j) : 0;

  f32x16 dk[Tl::BLOCKS], dv[Tl::BLOCKS];
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b) dk[b] = dv[b] = (f32x16)0.0f;

  // (counts of tiles, from query `first` on; the wave's keys jw .. jw + 31 lie at the queries' places + ahead)
  Passage way = {};
  const int first_w = first + rg * S::SPAN, mine = jw < w.lk ? tiles : 0;
  const int whole = floor_div(w.lq - first_w - S::SPAN, S::ROWS) + 1;
  const int at0 = first_w + ahead - jw;  // where the wave's first query lies, seen from its first key
  way.begin = a.s.causal ? max(0, min(mine, -floor_div(at0 + S::SPAN - 1, S::ROWS))) : 0;
  way.near0 = way.near1 = mine;
  way.far0 = way.begin;
  if (!BIAS) {  // hidden in part by the mask; not at all; by the last query's end
    way.near0 = a.s.causal ? max(way.begin, min(mine, -floor_div(at0 - 31, S::ROWS))) : way.begin;
    way.far1 = max(way.near0, min(mine, whole));
  } else if (a.s.pos_q) {
    way.far1 = mine;
  } else {
    if (!a.s.causal) way.far0 = max(way.begin, min(min(mine, whole), floor_div(-at0 - far - S::SPAN + 1, S::ROWS) + 1));
    way.near0 = max(way.far0, min(mine, -floor_div(at0 - 31 - far, S::ROWS)));
    way.far1 = max(way.near0, min(mine, whole));
  }

  const int h0 = g * group + group * part / a.parts, h1 = g * group + group * (part + 1) / a.parts;
  for (int h = h0; h < h1 && tiles > 0; ++h) {
    Loader<T, DP, S::ROWS, S::WAVES> lq, ld;
    lq.init((const T*)a.q + (long)w.q0 * a.q_row + h * a.q_head, a.q_row, a.dim);
    ld.init((const T*)a.dout + ((long)w.q0 * a.heads + h) * a.dim, (long)a.heads * a.dim, a.dim);
    const float* stats = a.stats + (long)h * a.nq + w.q0;
    const float* delta = a.delta + (long)h * a.nq + w.q0;
    auto load = [&](int n) {
      char* b = lds + (n & 1) * S::BUFFER;
      const int r = first + n * S::ROWS;
      lq.load(b, r, w.lq);
      ld.load(b + Tl::BYTES, r, w.lq);
      char* e = b + 2 * Tl::BYTES;
      load_words(e, delta, r, w.lq);
      load_words(e + 256, BIAS ? stats : delta + (long)a.heads * a.nq, r, w.lq);
      if (BIAS) load_words(e + 512, stats + (long)a.heads * a.nq, r, w.lq);
      if (BIAS && a.s.pos_q) load_words(e + 768, a.s.pos_q + w.q0, r, w.lq);
    };
    __syncthreads();  // the last head's tiles and table are read
    load(0);
    if (BIAS) load_table(by_distance, a.s, a.table, h);
    typename Tl::Lane at(lane);
    auto tile = [&](auto masked, auto mode, const char* qt, int i0) __attribute__((always_inline)) {
      constexpr bool MASK = decltype(masked)::value;
      constexpr int MODE = decltype(mode)::value;
      const char* dt = qt + Tl::BYTES;
      at.fresh();
      const float* rows = (const float*)(dt + Tl::BYTES);  // delta; ref, or m and ll; positions
      const float one = MODE == ONE ? by_distance[jw < i0 + rg * S::SPAN + ahead ? 0 : 2 * (far + PAD)] : 0.0f;
      const float* near = by_distance + (min(max(pos_k - ahead - i0 - 4 * half, -far), far + 60) + far + PAD);
#pragma unroll S::UNROLL
      for (int qn = 0; qn < S::SPAN / 32; ++qn) {
        const int qb = rg * (S::SPAN / 32) + qn;
        f32x16 x = (f32x16)0.0f, dp = (f32x16)0.0f;
#pragma unroll
        for (int s = 0; s < Tl::STEPS; ++s) mma_step(x, Tl::frag(qt, qb * 32, s, at), k[s]);
        if (S::APART) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < Tl::STEPS; ++s) mma_step(dp, Tl::frag(dt, qb * 32, s, at), v[s]);
        if (S::APART) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int row0 = qb * 32 + 8 * t + 4 * half;
          const f32x4 delta = *(const f32x4*)(rows + row0), ref = *(const f32x4*)(rows + 64 + row0);
          f32x4 ll;
          i32x4 pos;
          if (MODE != NONE) ll = *(const f32x4*)(rows + 128 + row0);
          if (MODE == GIVEN) pos = *(const i32x4*)(rows + 192 + row0);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = i0 + row0 + e, r = 4 * t + e;
            // A hidden pair's score is -inf: p and ds come out 0, or NaN where what is hidden is not finite -- then the
            // key's row is done again.
            float y = x[r];
            if constexpr (MODE == NONE) {
              y = fmaf(y, sc, -ref[e]);
            } else {
              float b = one;
              if (MODE == NEAR) b = near[-(qb * 32 + acc_row(r, 0))];
              if (MODE == GIVEN) b = by_distance[PAD + pa_entry(pa_apart(pos_k, pos[e]), far)];
              y = (fmaf(y, sc, b) - ref[e]) - (ll[e] - Lift<T>::LOG2);
            }
            if (MASK) y = (int)(i < w.lq) & (int)(j <= i + see) ? y : -INFINITY;
            const float p = __builtin_amdgcn_exp2f(y);
            x[r] = p;
            dp[r] = p * (dp[r] - delta[e]);
          }
        }
        Probs<T> pp, ds;  // rounded to the type: half a step each
        pp.set(x);
        ds.set(dp);
#pragma unroll
        for (int b = 0; b < Tl::BLOCKS; ++b) {
          Tl::mma_t(dt, qb * 32, b, at, pp, dv[b]);
          Tl::mma_t(qt, qb * 32, b, at, ds, dk[b]);
        }
      }
    };
    auto step = [&](int n) {
      tiles_ready();
      if (n + 1 < tiles) load(n + 1);
    };
    walk(way, tiles, step,
         [&](int n) {
           tile(False(), Mode<BIAS ? ONE : NONE>(), lds + (n & 1) * S::BUFFER, first + n * S::ROWS);
         },
         [&](int n) {
           const char* qt = lds + (n & 1) * S::BUFFER;
           if constexpr (!BIAS) tile(True(), Mode<NONE>(), qt, first + n * S::ROWS);
           else if (a.s.pos_q) tile(True(), Mode<GIVEN>(), qt, first + n * S::ROWS);
           else tile(True(), Mode<NEAR>(), qt, first + n * S::ROWS);
         });
  }

  float* sums = (float*)lds + kg * 2 * 32 * (DP + 4) + col * (DP + 4) + 4 * half;
  __syncthreads();
  if (rg == 1) {
#pragma unroll
    for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 y = {dk[b][4 * t], dk[b][4 * t + 1], dk[b][4 * t + 2], dk[b][4 * t + 3]};
        const f32x4 z = {dv[b][4 * t], dv[b][4 * t + 1], dv[b][4 * t + 2], dv[b][4 * t + 3]};
        *(f32x4*)(sums + b * 32 + 8 * t) = y;
        *(f32x4*)(sums + 32 * (DP + 4) + b * 32 + 8 * t) = z;
      }
  }
  __syncthreads();
  if (rg == 1) return;
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 y = *(const f32x4*)(sums + b * 32 + 8 * t), z = *(const f32x4*)(sums + 32 * (DP + 4) + b * 32 + 8 * t);
#pragma unroll
      for (int e = 0; e < 4; ++e) dk[b][4 * t + e] += y[e], dv[b][4 * t + e] += z[e];
    }
  const bool there = row0 + kg * 32 + col < end;  // keys' gradients, and zeros behind a sequence's keys
  const long to = ((row0 + kg * 32 + col) * a.kv_heads + g) * a.dim;
  if (a.parts > 1) {
    const long all = (long)a.nk * a.kv_heads * a.dim;
    store_part<T>(dk, a.dkv_part + 2 * part * all + to, there, valid, a.scale, a.dim, half);
    store_part<T>(dv, a.dkv_part + (2 * part + 1) * all + to, there, valid, 1.0f, a.dim, half);
    return;
  }
  const bool bad_k = store_sum<T>(dk, (T*)a.dk + to, there, valid, a.scale, a.dim, half);
  const bool bad_v = store_sum<T>(dv, (T*)a.dv + to, there, valid, 1.0f, a.dim, half);
  const unsigned long long again = __ballot(valid && (bad_k | bad_v));
  for (unsigned rows = (unsigned)again | (unsigned)(again >> 32); rows; rows &= rows - 1)
    pa_row_dkv<T>(a, w, jw + __ffs(rows) - 1, g);
}

// The same for a head dim of 128, where both gradients' sums and both operands do not leave a SIMD's registers room for a
// second wave: two waves share the keys, one with k and dv's sums, one with v and dk's.  The first makes the probabilities
// while the second multiplies dout and v, and hands them over through LDS in fp32.
template <typename T, int DP>
struct PairShape {
  static constexpr int WAVES = 8, COLS = 128, ROWS = sizeof(T) == 4 ? 32 : 64;
  typedef Tile<T, DP, ROWS> Tl;
  static constexpr int BUFFER = 2 * Tl::BYTES + 4 * 256, PROBS = 4 * ROWS * 32 * 4;
  static int lds(bool bias, int max_distance) { return 2 * BUFFER + PROBS + 64 + (bias ? table_places(max_distance) * 4 : 0); }
};

template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(512, 2) void pa_dkv_pair_kernel(PaArgs a, long slots) {
  typedef PairShape<T, DP> S;
  typedef typename S::Tl Tl;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31,
            half = lane >> 5;
  const int kg = wave & 3;
  const bool second = wave >> 2;  // v and dk; the other: k and dv
  const int group = a.heads / a.kv_heads;
  long slot;
  int g, start;
  if (!tile_of(slots, a.kv_heads * a.parts, slot, g)) return;
  const int part = g % a.parts;  // of the group's heads
  g /= a.parts;
  const int span = pa_span(a.s.cu_k, a.s.batch, a.nk, 7, slot, start);
  const long row0 = start + ((slot - (start >> 7) - span) << 7);
  const int end = span > a.s.batch ? a.nk : pa_clamp(a.s.cu_k[span], a.nk);  // of the span's rows, keys or not
  if (row0 >= end) return;
  PaSeq w = {};
  if (span > 0 && span <= a.s.batch) w = pa_seq(a.s, a.nq, a.nk, span - 1);
  const int jg = (int)(row0 - start), jw = jg + kg * 32, j = jw + col;  // first key of workgroup, wave; lane's own
  const bool valid = j < w.lk;
  const int ahead = w.lk - w.lq;
  const int see = a.s.causal ? ahead : 1 << 30;           // key j is seen by queries i with j <= i + see
  const int first = a.s.causal ? max(jg - ahead, 0) : 0;  // first query that sees one of the workgroup's keys
  const int tiles = jg < w.lk && first < w.lq ? (w.lq - first + S::ROWS - 1) / S::ROWS : 0;
  const int far = a.s.max_distance;
  float* by_distance = (float*)(lds + 2 * S::BUFFER + S::PROBS + 64);
  char* probs = lds + 2 * S::BUFFER + kg * (S::PROBS / 4) + lane * 16;

  frag_t<T> kv[Tl::STEPS];
  if (second) load_rows<T>(kv, (const T*)a.v + (long)(w.k0 + j) * a.v_row + g * a.v_head, valid, a.dim, half);
  else load_rows<T>(kv, (const T*)a.k + (long)(w.k0 + j) * a.k_row + g * a.k_head, valid, a.dim, half);
  const float sc = a.scale * PA_LOG2E;
  const int pos_k = BIAS && valid ? pa_pos_k(a.s, w, j) : 0;
  f32x16 sum[Tl::BLOCKS];  // of dv, of dk
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b) sum[b] = (f32x16)0.0f;

  Passage way = {};
  const int mine = jw < w.lk ? tiles : 0;
  const int whole = floor_div(w.lq - first - S::ROWS, S::ROWS) + 1;
  const int at0 = first + ahead - jw;  // where the first query lies, seen from the wave's first key
  way.begin = a.s.causal ? max(0, min(mine, -floor_div(at0 + S::ROWS - 1, S::ROWS))) : 0;
  way.near0 = way.near1 = mine;
  way.far0 = way.begin;
  if (!BIAS) {
    way.near0 = a.s.causal ? max(way.begin, min(mine, -floor_div(at0 - 31, S::ROWS))) : way.begin;
    way.far1 = max(way.near0, min(mine, whole));
  } else if (a.s.pos_q) {
    way.far1 = mine;
  } else {
    if (!a.s.causal) way.far0 = max(way.begin, min(min(mine, whole), floor_div(-at0 - far - S::ROWS + 1, S::ROWS) + 1));
    way.near0 = max(way.far0, min(mine, -floor_div(at0 - 31 - far, S::ROWS)));
    way.far1 = max(way.near0, min(mine, whole));
  }

  typename Tl::Lane at(lane);
  const int h0 = g * group + group * part / a.parts, h1 = g * group + group * (part + 1) / a.parts;
  for (int h = h0; h < h1 && tiles > 0; ++h) {
    Loader<T, DP, S::ROWS, S::WAVES> lq, ld;
    lq.init((const T*)a.q + (long)w.q0 * a.q_row + h * a.q_head, a.q_row, a.dim);
    ld.init((const T*)a.dout + ((long)w.q0 * a.heads + h) * a.dim, (long)a.heads * a.dim, a.dim);
    const float* stats = a.stats + (long)h * a.nq + w.q0;
    const float* delta = a.delta + (long)h * a.nq + w.q0;
    auto load = [&](int n) {
      char* b = lds + (n & 1) * S::BUFFER;
      const int r = first + n * S::ROWS;
      lq.load(b, r, w.lq);
      ld.load(b + Tl::BYTES, r, w.lq);
      char* e = b + 2 * Tl::BYTES;
      load_words(e, delta, r, w.lq);
      load_words(e + 256, BIAS ? stats : delta + (long)a.heads * a.nq, r, w.lq);
      if (BIAS) load_words(e + 512, stats + (long)a.heads * a.nq, r, w.lq);
      if (BIAS && a.s.pos_q) load_words(e + 768, a.s.pos_q + w.q0, r, w.lq);
    };
    __syncthreads();  // the last head's tiles and table are read
    load(0);
    if (BIAS) load_table(by_distance, a.s, a.table, h);
    auto handed_over = [&] {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    auto tile = [&](auto masked, auto mode, const char* qt, int i0) __attribute__((always_inline)) {
      constexpr bool MASK = decltype(masked)::value;
      constexpr int MODE = decltype(mode)::value, PARTS = S::ROWS / 32;
      const char* dt = qt + Tl::BYTES;
      const float* rows = (const float*)(dt + Tl::BYTES);  // delta; ref, or m and ll; positions
      at.fresh();
      f32x16 x[PARTS];
      const char* left = second ? dt : qt;
#pragma unroll
      for (int qb = 0; qb < PARTS; ++qb) {
        x[qb] = (f32x16)0.0f;
#pragma unroll
        for (int s = 0; s < Tl::STEPS; ++s) mma_step(x[qb], Tl::frag(left, qb * 32, s, at), kv[s]);
      }
      if (!second) {
        const float one = MODE == ONE ? by_distance[jw < i0 + ahead ? 0 : 2 * (far + PAD)] : 0.0f;
        const float* near = by_distance + (min(max(pos_k - ahead - i0 - 4 * half, -far), far + 60) + far + PAD);
#pragma unroll
        for (int qb = 0; qb < PARTS; ++qb)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int r0 = qb * 32 + 8 * t + 4 * half;
            const f32x4 ref = *(const f32x4*)(rows + 64 + r0);
            f32x4 ll, p;
            i32x4 pos;
            if (MODE != NONE) ll = *(const f32x4*)(rows + 128 + r0);
            if (MODE == GIVEN) pos = *(const i32x4*)(rows + 192 + r0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = i0 + r0 + e;
              float y = x[qb][4 * t + e];
              if constexpr (MODE == NONE) {
                y = fmaf(y, sc, -ref[e]);
              } else {
                float b = one;
                if (MODE == NEAR) b = near[-(qb * 32 + 8 * t + e)];
                if (MODE == GIVEN) b = by_distance[PAD + pa_entry(pa_apart(pos_k, pos[e]), far)];
                y = (fmaf(y, sc, b) - ref[e]) - (ll[e] - Lift<T>::LOG2);
              }
              if (MASK) y = (int)(i < w.lq) & (int)(j <= i + see) ? y : -INFINITY;
              p[e] = x[qb][4 * t + e] = __builtin_amdgcn_exp2f(y);
            }
            *(f32x4*)(probs + (qb * 4 + t) * 1024) = p;
          }
      }
      handed_over();
#pragma unroll
      for (int qb = 0; qb < PARTS; ++qb) {
        if (second)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const f32x4 p = *(const f32x4*)(probs + (qb * 4 + t) * 1024);
            const f32x4 delta = *(const f32x4*)(rows + qb * 32 + 8 * t + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[qb][4 * t + e] = p[e] * (x[qb][4 * t + e] - delta[e]);
          }
        Probs<T> r;  // p, ds rounded to the type: half a step each
        r.set(x[qb]);
#pragma unroll
        for (int b = 0; b < Tl::BLOCKS; ++b) Tl::mma_t(second ? qt : dt, qb * 32, b, at, r, sum[b]);
      }
    };
    auto step = [&](int n) {
      tiles_ready();
      if (n + 1 < tiles) load(n + 1);
    };
    walk(way, tiles, step,
         [&](int n) {
           tile(False(), Mode<BIAS ? ONE : NONE>(), lds + (n & 1) * S::BUFFER, first + n * S::ROWS);
         },
         [&](int n) {
           const char* qt = lds + (n & 1) * S::BUFFER;
           if constexpr (!BIAS) tile(True(), Mode<NONE>(), qt, first + n * S::ROWS);
           else if (a.s.pos_q) tile(True(), Mode<GIVEN>(), qt, first + n * S::ROWS);
           else tile(True(), Mode<NEAR>(), qt, first + n * S::ROWS);
         },
         handed_over);
  }

  const bool there = row0 + kg * 32 + col < end;  // keys' gradients, and zeros behind a sequence's keys
  const long to = ((row0 + kg * 32 + col) * a.kv_heads + g) * a.dim;
  if (a.parts > 1) {
    store_part<T>(sum, a.dkv_part + (2 * part + !second) * ((long)a.nk * a.kv_heads * a.dim) + to, there, valid,
                  second ? a.scale : 1.0f, a.dim, half);
    return;
  }
  const bool bad = store_sum<T>(sum, (T*)(second ? a.dk : a.dv) + to, there, valid, second ? a.scale : 1.0f, a.dim, half);
  // rows to do again are done by the first of the two waves, once both have stored theirs
  const unsigned long long again = __ballot(valid && bad);
  unsigned rows = (unsigned)again | (unsigned)(again >> 32);
  unsigned* marks = (unsigned*)(lds + 2 * S::BUFFER + S::PROBS);
  if (lane == 0) marks[wave] = rows;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (second) return;
  for (rows |= marks[wave + 4]; rows; rows &= rows - 1) pa_row_dkv<T>(a, w, jw + __ffs(rows) - 1, g);
}

#define PA_LAUNCH(KERNEL, SLOTS, HEADS, LDS, MOST)                                                         \
  {                                                                                                        \
    static bool done[64];                                                                                  \
    if (!i2r_lds_attr((const void*)KERNEL, MOST, done)) return false;                                      \
    hipLaunchKernelGGL(KERNEL, dim3(tile_grid(SLOTS, HEADS)), dim3(256), LDS, st, a, SLOTS);               \
  }

template <typename T, int DP>
static bool launch_dkv(const PaArgs& a, hipStream_t st) {
  typedef DkvShape<T, DP> S;
  const long slots = a.nk / S::COLS + a.s.batch + 2;
  if (a.table)
    PA_LAUNCH((pa_dkv_kernel<T, DP, true>), slots, a.kv_heads * a.parts, S::lds(true, a.s.max_distance), S::lds(true, PA_MAX_DISTANCE))
  else PA_LAUNCH((pa_dkv_kernel<T, DP, false>), slots, a.kv_heads * a.parts, S::lds(false, 0), S::lds(false, 0))
  return true;
}

template <typename T, int DP>
static bool launch_pair(const PaArgs& a, hipStream_t st) {
  typedef PairShape<T, DP> S;
  const long slots = a.nk / S::COLS + a.s.batch + 2;
  static bool done[2][64];
#define PA_PAIR(B)                                                                                                   \
  {                                                                                                                  \
    if (!i2r_lds_attr((const void*)pa_dkv_pair_kernel<T, DP, B>, S::lds(B, PA_MAX_DISTANCE), done[B])) return false;  \
    hipLaunchKernelGGL((pa_dkv_pair_kernel<T, DP, B>), dim3(tile_grid(slots, a.kv_heads * a.parts)), dim3(512),       \
                       S::lds(B, a.s.max_distance), st, a, slots);                                                    \
  }
  if (a.table) PA_PAIR(true) else PA_PAIR(false)
  return true;
}

template <typename T, int DP>
static bool launch_bwd(const PaArgs& a, hipStream_t st, bool dq, bool dkv) {
  const int far = a.s.max_distance;
  const long slots_q = (a.nq >> 7) + a.s.batch + 2;
  if (dq) {
    typedef DqShape<T, DP> S;
    if (a.table) PA_LAUNCH((pa_dq_kernel<T, DP, true>), slots_q, a.heads, S::lds(true, far, a.s.num_buckets),
                           S::lds(true, PA_MAX_DISTANCE, PA_MAX_BUCKETS))
    else PA_LAUNCH((pa_dq_kernel<T, DP, false>), slots_q, a.heads, S::lds(false, 0, 0), S::lds(false, 0, 0))
  }
  if (dkv) {
    bool ok;
    // 128 wide: one wave a SIMD against the pair's two; four documents of 2048 tokens, 32 heads: bf16 1126 us against 938, but
    // fp32, whose products take 8 times as long and hide everything else, 1403 against 1487 (1024 tokens)
    if constexpr (DP == 128 && sizeof(T) == 2) ok = launch_pair<T, DP>(a, st);
    else ok = launch_dkv<T, DP>(a, st);
    if (!ok) return false;
    if (a.parts > 1)
      hipLaunchKernelGGL(pa_dkv_join_kernel<T>, dim3(i2r_cdiv((long)a.nk * a.kv_heads, 4)), dim3(256), 0, st, a);
  }
  return true;
}

bool pa_launch_bwd(int dtype, const PaArgs& a, hipStream_t st, bool dq, bool dkv) {
#define PA_BY_DIM(T)                                            \
  return a.dim <= 32   ? launch_bwd<T, 32>(a, st, dq, dkv)      \
         : a.dim <= 64 ? launch_bwd<T, 64>(a, st, dq, dkv)      \
                       : launch_bwd<T, 128>(a, st, dq, dkv);
  if (dtype == 0) PA_BY_DIM(float)
  if (dtype == 1) PA_BY_DIM(f16_t)
  PA_BY_DIM(bf16_t)
}
