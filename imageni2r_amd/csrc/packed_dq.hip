// Backward of packed-sequence attention on the matrix cores: dq and the table's gradient.
//
// The backward is two kernels, both recomputing the scores: dq (a query a column, keys pass by) and dk / dv (a key a
// column, the queries of all heads of its group pass by).  Seven products where five would do with dq added up atomically -- but no float is ever
// added in an order that could change, and nothing but the outputs is written.
//
// Bound by matrix and vector instructions, and by what keeps two waves a SIMD from filling each other's gaps (counters: 128
// wide, two documents of 4096 tokens, matrix pipes busy 37 % of the time, vector pipes 30 %; 64 wide with a bias, eight of up to
// 2048, 15 % and 39 %; fp32, 8 wide, bias by times, 25 % and 29 %); with a bias at 128 the histogram leaves room for one
// workgroup a CU.  Measured (events, causal, bf16): eight documents of 2048 tokens, 32 heads of 128 over 8 493 us (837
// TFLOP/s), 32 heads of 64 266 us (776); two documents of 4096, 32 heads of 128 over 8, with a bias and the table's gradient
// 733 us (562).
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

template <typename T, int W>
struct DqShape {
  static constexpr int DP = Tile<T, W, 32>::DP;
  static constexpr int WAVES = 4, ROWS = 32 * WAVES, KEYS = sizeof(T) == 4 ? 32 : 64;
  typedef Tile<T, W, KEYS> Tl;
  static constexpr int BUFFER = 2 * Tl::BYTES + 256;  // k, v, positions
  static constexpr int PER_SIMD = sizeof(T) == 4 && DP == 128 ? 1 : 2, UNROLL = DP == 128 ? 1 : 2;
  static constexpr bool APART = DP == 128;  // the products' operands would not fit the registers all at once
  static int lds(bool bias, int max_distance, int buckets) {
    return 2 * BUFFER + (bias ? table_places(max_distance) * 8 + buckets * 64 * 4 * WAVES : 0);
  }
};

// dq of 32 queries a wave, delta = <dout, out> and the two stats' sum on the way for the other kernel, and ds summed by
// bucket: each lane its own column of a histogram in LDS, so that no two lanes add to one word.
template <typename T, int W, bool BIAS>
__global__ __launch_bounds__(256, (DqShape<T, W>::PER_SIMD)) void pa_dq_kernel(PaArgs a, long slots) {
  typedef DqShape<T, W> S;
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

  Loader<T, W, S::KEYS, S::WAVES> lk, lv;
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
  // A hidden pair's 0 times NaN, or a lifted ds beyond fp16: those queries are done again, pair by pair.  What no query of the
  // tile sees reaches the histogram too, where its score is -inf or the column holds no query (and a made-up place, 0): if a
  // bucket's sum comes out not finite, the columns that are to blame are emptied, and their queries' ds added pair by pair.
  // (A test of each pair's score instead would be two instructions more in the loop over the keys.)
  const unsigned long long again = __ballot(valid && !(finite == 0.0f));
  unsigned rows = (unsigned)again | (unsigned)(again >> 32), by_bucket = 0;
  int own = lane;
  asm volatile("" : "+v"(own));  // (keeps the columns' places below out of the registers above: 64 wide they would be 169)
#pragma unroll 1
  for (bool first = true;; first = false) {
    bool done = true;
    if (sums) {
      __syncthreads();
      const float* all = (const float*)(by_distance + table_places(far));
      float off = 0.0f;
      for (int c = wave; c < nb; c += S::WAVES) {
        float s = 0.0f;
        for (int v = 0; v < S::WAVES; ++v) s += all[(v * nb + c) * 64 + own];
        s = wave_sum(s);
        off = fmaf(s, 0.0f, off);
        if (own == 0) a.part[(slot * a.heads + h) * nb + c] = s * Lift<T>::DOWN;
      }
      if (first) {
        int* marks = (int*)lds;  // (the tiles are read)
        if (own == 0) marks[wave] = off == 0.0f;
        __syncthreads();
        for (int v = 0; v < S::WAVES; ++v) done &= marks[v] != 0;
        if (!done) {
          off = 0.0f;
          for (int c = 0; c < nb; ++c) off = fmaf(hist[c * 64 + own], 0.0f, off);
          const unsigned long long bad = __ballot(!(off == 0.0f)), live = __ballot(valid);
          by_bucket = (unsigned)bad | (unsigned)(bad >> 32);
          if (by_bucket >> (own & 31) & 1)
            for (int c = 0; c < nb; ++c) hist[c * 64 + own] = 0.0f;
          by_bucket &= (unsigned)live;
        }
      }
    }
    for (rows |= by_bucket; rows; rows &= rows - 1) {
      const int c = __ffs(rows) - 1;
      pa_row_dq<T>(a, w, iw + c, h, by_bucket >> c & 1 ? hist + own : nullptr);
    }
    by_bucket = 0;
    if (done) break;
  }
}

#define PA_LAUNCH(KERNEL, SLOTS, HEADS, LDS, MOST)                                                         \
  {                                                                                                        \
    static bool done[64];                                                                                  \
    if (!i2r_lds_attr((const void*)KERNEL, MOST, done)) return false;                                      \
    hipLaunchKernelGGL(KERNEL, dim3(tile_grid(SLOTS, HEADS)), dim3(256), LDS, st, a, SLOTS);               \
  }

template <typename T, int W>
static bool launch_dq(const PaArgs& a, hipStream_t st) {
  typedef DqShape<T, W> S;
  const long slots = (a.nq >> 7) + a.s.batch + 2;
  if (a.table) PA_LAUNCH((pa_dq_kernel<T, W, true>), slots, a.heads, S::lds(true, a.s.max_distance, a.s.num_buckets),
                         S::lds(true, PA_MAX_DISTANCE, PA_MAX_BUCKETS))
  else PA_LAUNCH((pa_dq_kernel<T, W, false>), slots, a.heads, S::lds(false, 0, 0), S::lds(false, 0, 0))
  return true;
}

bool pa_launch_dq(int dtype, const PaArgs& a, hipStream_t st) {
#define PA_CALL(T, W) launch_dq<T, W>(a, st)
  if (dtype == 0) PA_BY_WIDTH(float, PA_CALL);
  if (dtype == 1) PA_BY_WIDTH(f16_t, PA_CALL);
  PA_BY_WIDTH(bf16_t, PA_CALL);
}
