// Backward of packed-sequence attention on the matrix cores: dk and dv (packed_dq.hip has the other half).
//
// A key is a column, the queries of its group's heads pass by in tiles: both gradients of a key stay in one wave's
// accumulators until the end, shared heads are summed there, and no addition is atomic.
//
// Bound by neither kind of instruction alone (counters): 128 wide, two documents of 4096 tokens, 32 heads over 8, the matrix
// pipes are busy 29 % of the time, the vector pipes 20 %, and waves wait for half of theirs: for each other (two barriers a
// tile) and at the end, for the longest workgroups; 64 wide with a bias, eight documents of up to 2048, 16 % and 28 %, with one
// wave a SIMD on average, where two fit; fp32, 8 wide, 42 % and 25 %.  Measured (kernel traces, causal, bf16): eight documents of
// 2048 tokens, 32 heads of 128 over 8 795 us (691 TFLOP/s), 32 heads of 64 410 us (670); two documents of 4096 tokens, 32
// heads of 128 over 8, with a bias 678 us (810); 8192 tokens, 16 heads of 128 over 2, split over the group's heads, 621 us and
// 15 us of joining (865).
#include "packed_tiles.h"

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
template <typename T, int W>
struct DkvShape {
  static constexpr int RG = 2;
  static constexpr int DP = Tile<T, W, 32>::DP;
  static constexpr int WAVES = 4, COLS = 32 * WAVES / RG, ROWS = sizeof(T) == 4 ? 32 * RG : 64, SPAN = ROWS / RG;
  typedef Tile<T, W, ROWS> Tl;
  static constexpr int BUFFER = 2 * Tl::BYTES + 4 * 256;  // q, dout, delta, stats, positions
  static constexpr int UNROLL = DP == 128 || sizeof(T) == 4 ? 1 : 2;
  static constexpr bool APART = DP * sizeof(T) >= 256;
  // The two that miss a third wave a SIMD (168 registers) by two are held to it.  In turn with dq, two waves against three: 64
  // wide in bf16, eight documents of 2048 tokens, 32 heads 424 -> 359 us (a kernel trace has 410 for the latter), 16 over 4
  // 77 -> 67, 12 heads of 1024 both ways 79 -> 66; fp32, 32 wide with a bias, 32 x 384 121 -> 97.  It loses where the
  // grid is two rounds of two workgroups a CU, of three a whole round and a third of one: 4096 tokens, 16 heads of 64 over 4
  // (1024 workgroups), 108 -> 117.  (Where two a CU hold all there is it gains nothing: fp32 of 32 with a bias, 4 x 1024,
  // 154 -> 157.)
  static constexpr int per_simd(bool bias) {
    return DP == 128 ? 1 : (sizeof(T) == 2 ? W == 64 && !bias : W == 32 && bias) ? 3 : 2;
  }
  static constexpr int JOIN = 2 * COLS * (DP + 4) * 4;  // dk and dv of one group, where the tiles were
  static int lds(bool bias, int max_distance) {
    const int n = 2 * BUFFER + (bias ? table_places(max_distance) * 4 : 0);
    return n > JOIN ? n : JOIN;
  }
};

template <typename T, int W, bool BIAS>
__global__ __launch_bounds__(256, (DkvShape<T, W>::per_simd(BIAS))) void pa_dkv_kernel(PaArgs a, long slots) {
  typedef DkvShape<T, W> S;
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
    Loader<T, W, S::ROWS, S::WAVES> lq, ld;
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

  float* sums = (float*)lds + kg * 2 * 32 * (S::DP + 4) + col * (S::DP + 4) + 4 * half;
  __syncthreads();
  if (rg == 1) {
#pragma unroll
    for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 y = {dk[b][4 * t], dk[b][4 * t + 1], dk[b][4 * t + 2], dk[b][4 * t + 3]};
        const f32x4 z = {dv[b][4 * t], dv[b][4 * t + 1], dv[b][4 * t + 2], dv[b][4 * t + 3]};
        *(f32x4*)(sums + b * 32 + 8 * t) = y;
        *(f32x4*)(sums + 32 * (S::DP + 4) + b * 32 + 8 * t) = z;
      }
  }
  __syncthreads();
  if (rg == 1) return;
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 y = *(const f32x4*)(sums + b * 32 + 8 * t), z = *(const f32x4*)(sums + 32 * (S::DP + 4) + b * 32 + 8 * t);
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
template <typename T, int W>
struct PairShape {
  static constexpr int DP = Tile<T, W, 32>::DP;
  static constexpr int WAVES = 8, COLS = 128, ROWS = sizeof(T) == 4 ? 32 : 64;
  typedef Tile<T, W, ROWS> Tl;
  static constexpr int BUFFER = 2 * Tl::BYTES + 4 * 256, PROBS = 4 * ROWS * 32 * 4;
  static int lds(bool bias, int max_distance) { return 2 * BUFFER + PROBS + 64 + (bias ? table_places(max_distance) * 4 : 0); }
};

template <typename T, int W, bool BIAS>
__global__ __launch_bounds__(512, 2) void pa_dkv_pair_kernel(PaArgs a, long slots) {
  typedef PairShape<T, W> S;
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
    Loader<T, W, S::ROWS, S::WAVES> lq, ld;
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
      for (int qb = 0; qb < PARTS; ++qb) x[qb] = (f32x16)0.0f;
#pragma unroll
      for (int s = 0; s < Tl::STEPS; ++s)
#pragma unroll
        for (int qb = 0; qb < PARTS; ++qb) mma_step(x[qb], Tl::frag(left, qb * 32, s, at), kv[s]);
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

template <typename T, int W>
static bool launch_dkv(const PaArgs& a, hipStream_t st) {
  typedef DkvShape<T, W> S;
  const long slots = a.nk / S::COLS + a.s.batch + 2;
  // Two workgroups a CU where that holds them all, by as much LDS as lets no third in: it would stand on some CUs while others
  // have one.  4 x 1024 tokens, 16 heads over 8, both ways, with against without: fp32 of 32 with a bias 157 us, 218; bf16 of
  // 64 50, 55.
  const int least = a.nk / S::COLS * (long)a.kv_heads * a.parts <= 512 ? 56 << 10 : 0;
  if (a.table)
    PA_LAUNCH((pa_dkv_kernel<T, W, true>), slots, a.kv_heads * a.parts, std::max(least, S::lds(true, a.s.max_distance)),
              std::max(56 << 10, S::lds(true, PA_MAX_DISTANCE)))
  else
    PA_LAUNCH((pa_dkv_kernel<T, W, false>), slots, a.kv_heads * a.parts, std::max(least, S::lds(false, 0)),
              std::max(56 << 10, S::lds(false, 0)))
  return true;
}

template <typename T, int W>
static bool launch_pair(const PaArgs& a, hipStream_t st) {
  typedef PairShape<T, W> S;
  const long slots = a.nk / S::COLS + a.s.batch + 2;
  static bool done[2][64];
#define PA_PAIR(B)                                                                                                   \
  {                                                                                                                  \
    if (!i2r_lds_attr((const void*)pa_dkv_pair_kernel<T, W, B>, S::lds(B, PA_MAX_DISTANCE), done[B])) return false;  \
    hipLaunchKernelGGL((pa_dkv_pair_kernel<T, W, B>), dim3(tile_grid(slots, a.kv_heads * a.parts)), dim3(512),       \
                       S::lds(B, a.s.max_distance), st, a, slots);                                                    \
  }
  if (a.table) PA_PAIR(true) else PA_PAIR(false)
  return true;
}

template <typename T, int W>
static bool launch_both(const PaArgs& a, hipStream_t st) {
  bool ok;
  // 128 wide: one wave a SIMD against the pair's two; eight documents of 2048 tokens, 32 heads: bf16 1126 us against 938, but
  // fp32, whose products take 8 times as long and hide everything else, 1403 against 1487 (1024 tokens)
  if constexpr (W > 64 && sizeof(T) == 2) ok = launch_pair<T, W>(a, st);
  else ok = launch_dkv<T, W>(a, st);
  if (ok && a.parts > 1)
    hipLaunchKernelGGL(pa_dkv_join_kernel<T>, dim3(i2r_cdiv((long)a.nk * a.kv_heads, 4)), dim3(256), 0, st, a);
  return ok;
}

bool pa_launch_dkv(int dtype, const PaArgs& a, hipStream_t st) {
#define PA_CALL(T, W) launch_both<T, W>(a, st)
  if (dtype == 0) PA_BY_WIDTH(float, PA_CALL);
  if (dtype == 1) PA_BY_WIDTH(f16_t, PA_CALL);
  PA_BY_WIDTH(bf16_t, PA_CALL);
}
