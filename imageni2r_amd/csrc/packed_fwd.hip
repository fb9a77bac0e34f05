// Forward of packed-sequence attention on the matrix cores.
#include "packed_tiles.h"

// One workgroup: 4 waves x 32 queries of one sequence and head; keys come in tiles of KEYS, the next tile loading while
// this one is worked on (two LDS buffers, one barrier a tile).  One pass: the softmax's reference exponent and sum are kept
// per query (fp32) and the output is scaled when the exponent moves.
//
// Long sequences are bound by the issue of matrix and vector instructions together: the two hardly overlap there (16384 tokens,
// 128 wide: matrix pipes busy 50 % of the time, vector pipes 47 %), and per 64 keys a wave needs 32 products of 32 cycles, 32
// exponentials of 16 and some 120 other instructions of 4.  Short ones leave the start and end of a workgroup, and uneven
// workgroups, in view: 16 prompts of up to 1024, 64 wide with a bias, 15 % and 41 % (the exponentials weigh twice as much at 64),
// 1.6 waves a SIMD where two and more fit; sequences up to 1999, 80 wide, 27 % and 35 %; fp32, 8 wide, bias by times, 28 % and
// 22 %.  Measured, on several cards: 16384 tokens, 16 heads of 128 over 2, causal, bf16 1027 to 1108 us (up to 1071 TFLOP/s; a
// library product of 8192^3 reaches 1105); lengths up to 1999, 12 heads of 80, both directions, fp16 113 to 121 us (558); 16
// prompts of up to 1024, 16 heads of 64 over 4, with a bias 49 to 55 us (401).
//
// 32 queries a wave: 64 would halve the LDS reads, but leave one wave a SIMD.  Tiles of 64 keys (fp32 at 128: 32) keep two
// workgroups' buffers in 160 KB.
template <typename T, int W>
struct FwdShape {
  static constexpr int DP = Tile<T, W, 32>::DP;
  static constexpr int WAVES = 4, ROWS = 32 * WAVES, KEYS = sizeof(T) == 4 && W > 64 ? 32 : 64;
  typedef Tile<T, W, KEYS> Tl;
  static constexpr int MOST = W > 64 ? 2 : 4;
  static constexpr int BUFFER = 2 * Tl::BYTES + 256;  // k, v, positions
  static int lds(bool bias, int max_distance) { return 2 * BUFFER + (bias ? table_places(max_distance) * 4 : 0); }
};

template <typename T, int W, bool BIAS, bool SAVE>
__global__ __launch_bounds__(256, 2) __attribute__((amdgpu_waves_per_eu(2, FwdShape<T, W>::MOST))) void pa_fwd_kernel(PaArgs a, long slots) {
  typedef FwdShape<T, W> S;
  typedef typename S::Tl Tl;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31,
            half = lane >> 5;
  long slot;
  int h, start;
  if (!tile_of(slots, a.heads, slot, h)) return;
  slot = slots - 1 - slot;  // the last tiles of a sequence -- with a causal mask the longest -- first
  const int span = pa_span(a.s.cu_q, a.s.batch, a.nq, 7, slot, start);
  const long row0 = start + ((slot - (start >> 7) - span) << 7);
  if (span == 0 || span > a.s.batch) {  // rows of no sequence
    const int end = (int)min(row0 + S::ROWS, (long)(span == 0 ? pa_clamp(a.s.cu_q[0], a.nq) : a.nq));
    for (long i = (row0 * a.dim) + threadIdx.x; i < (long)end * a.dim; i += 256) {
      const long to = (i / a.dim * a.heads + h) * a.dim + i % a.dim;
      if (a.zero_outside) ((T*)a.out)[to] = (T)0.0f;
      if (a.out32) a.out32[to] = 0.0f;
    }
    return;
  }
  const PaSeq w = pa_seq(a.s, a.nq, a.nk, span - 1);
  if (row0 >= w.q0 + w.lq) return;
  const int g = h / (a.heads / a.kv_heads);
  const int i0 = (int)(row0 - w.q0), iw = i0 + wave * 32, i = iw + col;  // first query of workgroup, wave; lane's own
  const bool valid = i < w.lq;
  const int ahead = w.lk - w.lq;  // keys before the query's own
  int keys = w.lk;                // keys that the workgroup's last query sees
  if (a.s.causal) keys = min(keys, min(i0 + S::ROWS, w.lq) + ahead);

  Loader<T, W, S::KEYS, S::WAVES> lk, lv;
  lk.init((const T*)a.k + (long)w.k0 * a.k_row + g * a.k_head, a.k_row, a.dim);
  lv.init((const T*)a.v + (long)w.k0 * a.v_row + g * a.v_head, a.v_row, a.dim);
  float* by_distance = (float*)(lds + 2 * S::BUFFER);
  const int far = a.s.max_distance;
  auto load = [&](int n) {
    char* b = lds + (n & 1) * S::BUFFER;
    lk.load(b, n * S::KEYS, keys);
    lv.load(b + Tl::BYTES, n * S::KEYS, keys);
    if (BIAS && a.s.pos_k) load_words(b + 2 * Tl::BYTES, a.s.pos_k + w.k0, n * S::KEYS, keys);
  };
  const int tiles = keys > 0 ? (keys + S::KEYS - 1) / S::KEYS : 0;
  if (tiles > 0) load(0);

  // a negative scale flips q's sign (exact), so that the largest product is the largest score
  const float sc = (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * PA_LOG2E;
  frag_t<T> q[Tl::STEPS];
  load_rows<T>(q, (const T*)a.q + (long)(w.q0 + i) * a.q_row + h * a.q_head, valid && a.scale != 0.0f, a.dim, half);
  if (a.scale < 0.0f)
#pragma unroll
    for (int s = 0; s < Tl::STEPS; ++s) q[s] = -q[s];
  if (BIAS) load_table(by_distance, a.s, a.table, h);
  const int pos_q = BIAS && valid ? pa_pos_q(a.s, w, i) : 0;

  f32x16 o[Tl::BLOCKS];
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b) o[b] = (f32x16)0.0f;
  float m = -INFINITY, l = 0.0f;  // the column's reference exponent; the lane's half of the sum

  // One tile.  MASK: some pairs may be hidden by their place; MODE: where the bias comes from.
  typename Tl::Lane at(lane);
  auto tile = [&](auto masked, auto mode, const char* kt, int j0) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(masked)::value;
    constexpr int MODE = decltype(mode)::value, BLOCKS = S::KEYS / 32;
    const char* vt = kt + Tl::BYTES;
    at.fresh();
    f32x16 x[BLOCKS];
#pragma unroll
    for (int kb = 0; kb < BLOCKS; ++kb) x[kb] = (f32x16)0.0f;
#pragma unroll
    for (int s = 0; s < Tl::STEPS; ++s)
#pragma unroll
      for (int kb = 0; kb < BLOCKS; ++kb) mma_step(x[kb], Tl::frag(kt, kb * 32, s, at), q[s]);
    // v's operands of the first 32 keys set out before the softmax, which hides their way
    constexpr bool EARLY = sizeof(T) == 2 && !(BIAS && SAVE);
    typename Tl::Turned early[EARLY ? Tl::BLOCKS : 1];
    if constexpr (EARLY) {
#pragma unroll
      for (int b = 0; b < Tl::BLOCKS; ++b) early[b] = Tl::turned(vt, 0, b, at);
      __builtin_amdgcn_sched_barrier(0);
    }
    const float one = MODE == ONE ? by_distance[j0 < iw + ahead ? 0 : 2 * (far + PAD)] : 0.0f;
    // the place of the tile's first row (clamped so far out that all rows' places are beyond max_distance)
    const float* near = by_distance + (min(max(j0 + 4 * half - pos_q, -far - 60), far) + far + PAD);
    const int last = a.s.causal ? min(keys, i + ahead + 1) : keys;  // keys the lane's query sees
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < BLOCKS; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = kb * 32 + acc_row(r, half);
        float y = x[kb][r];
        if (MODE == ONE) y = fmaf(y, sc, one);
        if (MODE == NEAR) y = fmaf(y, sc, near[kb * 32 + acc_row(r, 0)]);
        if (MODE == GIVEN)
          y = fmaf(y, sc, by_distance[PAD + pa_entry(pa_apart(((const int*)(vt + Tl::BYTES))[row], pos_q), far)]);
        if (MASK) y = j0 + row < last ? y : -INFINITY;
        x[kb][r] = y;
        top = fmaxf(top, y);
      }
    top = fmaxf(top, other_half(top));
    if (!BIAS) top *= sc;
    // The reference exponent moves only when a score passes it by 2^8: the sums stay far from overflow, and most tiles
    // rescale nothing.
    if (__any(top > m + 8.0f || m == -INFINITY)) {
      const float mn = fmaxf(m, top), fall = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= fall;
#pragma unroll
      for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] *= fall;
      m = mn;
    }
    const float ref = m == -INFINITY ? 0.0f : m - Lift<T>::FWD_LOG2;
#pragma unroll
    for (int kb = 0; kb < BLOCKS; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[kb][r] = __builtin_amdgcn_exp2f(BIAS ? x[kb][r] - ref : fmaf(x[kb][r], sc, -ref));
        l += x[kb][r];
      }
      // Rounding the probabilities to the type puts each off by at most half a step, independently: as much as rounding
      // the output once more.  The table's gradient is fp32, and delta = <dout, out> enters it: with a bias to train
      // what the rounding took away is multiplied too, until 22 bits (fp16, or 2^-32 where that is more) or 24 (bf16) of each
      // have been.
      Probs<T> p;
      if constexpr (BIAS && SAVE && sizeof(T) == 2) {
#pragma unroll
        for (int part = 0; part < (__is_same(T, f16_t) ? 2 : 3); ++part) {
          p.set_and_take(x[kb]);
#pragma unroll
          for (int b = 0; b < Tl::BLOCKS; ++b) Tl::mma_t(vt, kb * 32, b, at, p, o[b]);
        }
      } else {
        p.set(x[kb]);
#pragma unroll
        for (int b = 0; b < Tl::BLOCKS; ++b) {
          if constexpr (EARLY) {
            if (kb == 0) Tl::mma_turned(early[b], p, o[b]);
            else Tl::mma_t(vt, kb * 32, b, at, p, o[b]);
          } else {
            Tl::mma_t(vt, kb * 32, b, at, p, o[b]);
          }
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

  l += other_half(l);
  m -= Lift<T>::FWD_LOG2;  // what l is relative to (of a score of 2^27 the 7 is rounded away, here as there)
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
  float finite = l * 0.0f;
  const long to = ((long)(w.q0 + i) * a.heads + h) * a.dim;
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int d = b * 32 + 8 * t + 4 * half;
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
      f32x4 z;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[e] = o[b][4 * t + e] * inv;
        finite = fmaf(z[e], 0.0f, finite);
        y[e] = (T)z[e];
      }
      if (valid && d < a.dim) {
        *(t4*)((T*)a.out + to + d) = y;
        if (SAVE && sizeof(T) == 2 && a.out32) *(f32x4*)(a.out32 + to + d) = z;
      }
    }
  if (SAVE && valid && half == 0) {
    a.stats[(long)h * a.nq + w.q0 + i] = m == -INFINITY ? 0.0f : m;
    a.stats[(long)(a.heads + h) * a.nq + w.q0 + i] = m == -INFINITY ? INFINITY : log2f(l);
  }
  // A product of a hidden key's probability 0 with an infinity or NaN is NaN: rows that came out so are done again, pair
  // by pair, without the hidden ones.
  unsigned long long again = __ballot(valid && !(finite == 0.0f));
  for (unsigned rows = (unsigned)again | (unsigned)(again >> 32); rows; rows &= rows - 1)
    pa_row_fwd<T>(a, w, iw + __ffs(rows) - 1, h);
}

template <typename T, int W>
static bool launch_fwd(const PaArgs& a, hipStream_t st) {
  typedef FwdShape<T, W> S;
  const bool bias = a.table != nullptr, save = a.stats != nullptr;
  const long slots = (a.nq >> 7) + a.s.batch + 2;
  const int lds = S::lds(bias, a.s.max_distance);
  const dim3 grid(tile_grid(slots, a.heads));
#define PA_FWD(B, V)                                                                                \
  {                                                                                                 \
    static bool done[64];                                                                           \
    if (!i2r_lds_attr((const void*)pa_fwd_kernel<T, W, B, V>, S::lds(true, PA_MAX_DISTANCE), done)) return false; \
    hipLaunchKernelGGL((pa_fwd_kernel<T, W, B, V>), grid, dim3(256), lds, st, a, slots);   \
  }
  if (bias && save) PA_FWD(true, true)
  else if (bias) PA_FWD(true, false)
  else if (save) PA_FWD(false, true)
  else PA_FWD(false, false)
  return true;
}

bool pa_launch_fwd(int dtype, const PaArgs& a, hipStream_t st) {
#define PA_CALL(T, W) launch_fwd<T, W>(a, st)
  if (dtype == 0) PA_BY_WIDTH(float, PA_CALL);
  if (dtype == 1) PA_BY_WIDTH(f16_t, PA_CALL);
  PA_BY_WIDTH(bf16_t, PA_CALL);
}
