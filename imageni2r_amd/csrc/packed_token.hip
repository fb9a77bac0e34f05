// Packed attention of a few queries against many keys: tokens and their cache.
//
// Bound by reading k and v once.  The 32 columns of the products are (token, head of the group) pairs, so a key / value
// head is read once for all its query heads; the keys are split over workgroups (and over a workgroup's waves, each with
// its own tiles and no barrier), whose parts a second kernel joins in a fixed order.  Measured: 64 tokens against caches of
// up to 8192 rows, 32 heads of 128 over 8, bf16 285 us, joining included (5.3 TB/s; a large copy reaches 4.9, a fill 6.9);
// one token against 131072 rows, with a bias 126 us (4.3 TB/s, of which the join takes 11 us); one token against 40 rows
// 7 us, the start of a kernel.
#include "packed_tiles.h"

template <typename T, int W>
struct TokenShape {
  static constexpr int DP = Tile<T, W, 32>::DP;
  static constexpr int KEYS = 32, STAGE = 2 * KEYS * DP * (int)sizeof(T);  // k and v of 32 keys
  // 64 KiB of tiles a workgroup (two of them on a CU): as many waves as that feeds with two stages each
  static constexpr int WAVES = 65536 / (2 * STAGE) < 4 ? 65536 / (2 * STAGE) : 4;
  typedef Tile<T, W, KEYS> Tl;
  static constexpr int PER_WAVE = 2 * STAGE, PER_SIMD = WAVES == 1 ? 1 : 2;
  static_assert(32 * (DP + 4) * 4 <= PER_WAVE, "a wave's sums go where its tiles were");
  static constexpr int SMALL = WAVES * 32 * 8 + 32 * 4;  // m and l of the waves, marks
  static int lds(bool bias, int max_distance) {
    return WAVES * PER_WAVE + SMALL + (bias ? 32 * PA_MAX_BUCKETS * 4 + 2 * max_distance + 4 : 0);
  }
};

struct TokenPlan {
  int shift, heads, chunks, splits;  // log2 of the tokens a tile; heads of a group in a tile; tiles a group; splits
  float *o, *ml;                     // parts: (split, row, head, dim) and (split, {m, l}, row, head)
};

template <typename T, int W, bool BIAS>
__global__ __launch_bounds__((64 * TokenShape<T, W>::WAVES), (TokenShape<T, W>::PER_SIMD)) void pa_token_kernel(PaArgs a, TokenPlan p) {
  typedef TokenShape<T, W> S;
  typedef typename S::Tl Tl;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
  const int split = blockIdx.x % p.splits, rest = blockIdx.x / p.splits, chunk = rest % p.chunks;
  const int g = rest / p.chunks % a.kv_heads;
  const long slot = rest / p.chunks / a.kv_heads;
  int start;
  const int span = pa_span(a.s.cu_q, a.s.batch, a.nq, p.shift, slot, start);
  const int group = a.heads / a.kv_heads;
  const int row0 = start + (int)((slot - (start >> p.shift) - span) << p.shift);
  const int token = col / p.heads, hg = chunk * p.heads + col % p.heads, h = g * group + hg;  // the column's
  const bool column = token < 1 << p.shift && hg < group;
  const long parts = (long)a.nq * a.heads;
  if (span == 0 || span > a.s.batch) {  // rows of no sequence
    const int end = span == 0 ? pa_clamp(a.s.cu_q[0], a.nq) : a.nq;
    const int row = row0 + token;
    if (split || wave || half || !column || row >= end) return;
    const long to = ((long)row * a.heads + h) * a.dim;
    if (p.splits > 1) p.ml[parts + (long)row * a.heads + h] = -1.0f;  // l < 0: no sequence's
    for (int d = 0; d < a.dim; ++d) {
      if (a.zero_outside) ((T*)a.out)[to + d] = (T)0.0f;
      if (a.out32) a.out32[to + d] = 0.0f;
    }
    return;
  }
  const PaSeq w = pa_seq(a.s, a.nq, a.nk, span - 1);
  if (row0 >= w.q0 + w.lq) return;
  const int i0 = row0 - w.q0, i = i0 + token;
  const bool valid = column && i < w.lq;
  const int ahead = w.lk - w.lq;
  int keys = w.lk;
  if (a.s.causal) keys = min(keys, min(i0 + (1 << p.shift), w.lq) + ahead);
  const int blocks = keys > 0 ? (keys + 31) / 32 : 0;
  const int b0 = (int)((long)blocks * split / p.splits), b1 = (int)((long)blocks * (split + 1) / p.splits);

  char* tiles = lds + wave * S::PER_WAVE;
  float* small = (float*)(lds + S::WAVES * S::PER_WAVE);
  Loader<T, W, 32, 1> lk, lv;
  lk.init((const T*)a.k + (long)w.k0 * a.k_row + g * a.k_head, a.k_row, a.dim);
  lv.init((const T*)a.v + (long)w.k0 * a.v_row + g * a.v_head, a.v_row, a.dim);
  constexpr int LOADS = 2 * Loader<T, W, 32, 1>::LOADS;
  auto load = [&](int n, int b) {
    char* t = tiles + (n & 1) * S::STAGE;
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // what was there has been read
    lk.load(t, b * 32, keys);
    lv.load(t + Tl::BYTES, b * 32, keys);
  };
  if (b0 + wave < b1) load(0, b0 + wave);

  const float sc = (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * PA_LOG2E;
  frag_t<T> q[Tl::STEPS];
  load_rows<T>(q, (const T*)a.q + (long)(w.q0 + i) * a.q_row + h * a.q_head, valid && a.scale != 0.0f, a.dim, half);
  if (a.scale < 0.0f)
#pragma unroll
    for (int s = 0; s < Tl::STEPS; ++s) q[s] = -q[s];
  const int far = a.s.max_distance, nb = a.s.num_buckets;
  float* table = small + S::SMALL / 4;  // (head of the tile, bucket), log2 units
  unsigned char* lut = (unsigned char*)(table + 32 * PA_MAX_BUCKETS);
  int pos_q = 0;
  if (BIAS) {
    for (int n = threadIdx.x; n < p.heads * nb; n += 64 * S::WAVES) {
      const int head = chunk * p.heads + n / nb;
      table[n] = head < group ? pa_log2_units(a.table[(long)(g * group + head) * nb + n % nb]) : 0.0f;
    }
    for (int n = threadIdx.x; n <= 2 * far; n += 64 * S::WAVES) lut[n] = (unsigned char)min((int)a.s.lut[n], nb - 1);
    __syncthreads();
    pos_q = valid ? pa_pos_q(a.s, w, i) : 0;
  }
  const float* own = table + (col % p.heads) * nb;

  f32x16 o[Tl::BLOCKS];
#pragma unroll
  for (int b = 0; b < Tl::BLOCKS; ++b) o[b] = (f32x16)0.0f;
  float m = -INFINITY, l = 0.0f;
  const typename Tl::Lane at(lane);
  for (int n = 0, b = b0 + wave; b < b1; ++n, b += S::WAVES) {
    if (b + S::WAVES < b1) {
      load(n + 1, b + S::WAVES);
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory");  // all but the loads just asked for
    } else {
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    }
    const char* kt = tiles + (n & 1) * S::STAGE;
    const char* vt = kt + Tl::BYTES;
    const int jb = b * 32;
    f32x16 x = (f32x16)0.0f;
#pragma unroll
    for (int s = 0; s < Tl::STEPS; ++s) mma_step(x, Tl::frag(kt, 0, s, at), q[s]);
    if (BIAS) {
      const int hi = jb + 31 - (i0 + ahead);  // largest distance
      if (!a.s.pos_q && hi <= -far) {
        const float e = own[lut[0]];
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], sc, e);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = jb + acc_row(r, half);
          const int pos_k = !a.s.pos_k ? j : j < keys ? a.s.pos_k[w.k0 + j] : 0;
          x[r] = fmaf(x[r], sc, own[lut[pa_entry(pa_apart(pos_k, pos_q), far)]]);
        }
      }
    }
    const int last = a.s.causal ? min(keys, i + ahead + 1) : keys;
    if (jb + 32 > keys || (a.s.causal && jb + 31 > i0 + ahead)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = jb + acc_row(r, half) < last ? x[r] : -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top = fmaxf(top, other_half(top));
    if (!BIAS) top *= sc;
    if (__any(top > m + 8.0f || m == -INFINITY)) {
      const float mn = fmaxf(m, top), fall = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= fall;
#pragma unroll
      for (int t = 0; t < Tl::BLOCKS; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] *= fall;
      m = mn;
    }
    const float ref = m == -INFINITY ? 0.0f : m - Lift<T>::FWD_LOG2;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_amdgcn_exp2f(BIAS ? x[r] - ref : fmaf(x[r], sc, -ref));
      l += x[r];
    }
    // rounded to the type: half a step each, as much as rounding the output once more; with a table to train (delta enters
    // its fp32 gradient) what the rounding took away is multiplied too
    Probs<T> pr;
    if constexpr (BIAS && sizeof(T) == 2) {
      const int terms = !a.stats ? 1 : __is_same(T, f16_t) ? 2 : 3;
      for (int part = 0; part < terms; ++part) {
        pr.set_and_take(x);
#pragma unroll
        for (int t = 0; t < Tl::BLOCKS; ++t) Tl::mma_t(vt, 0, t, at, pr, o[t]);
      }
    } else {
      pr.set(x);
#pragma unroll
      for (int t = 0; t < Tl::BLOCKS; ++t) Tl::mma_t(vt, 0, t, at, pr, o[t]);
    }
  }
  l += other_half(l);
  m -= Lift<T>::FWD_LOG2;  // what l is relative to (of a score of 2^27 the 7 is rounded away, here as there)

  // join the waves
  float* wm = small;                    // [wave][col]
  float* wl = small + S::WAVES * 32;
  int* marks = (int*)(small + S::WAVES * 64);
  if (half == 0) wm[wave * 32 + col] = m, wl[wave * 32 + col] = l;
  if (threadIdx.x < 32) marks[threadIdx.x] = 0;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int v = 0; v < S::WAVES; ++v) top = fmaxf(top, wm[v * 32 + col]);
#pragma unroll
  for (int v = 0; v < S::WAVES; ++v)
    sum += wl[v * 32 + col] * (wm[v * 32 + col] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm[v * 32 + col] - top));
  // The largest of scores that are all NaN is -inf, as of none: that some were is left in the sum, and has to reach the join of
  // the splits.
  if (top == -INFINITY && sum != sum) top = NAN;
  const float fall = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
  float* mine = (float*)tiles;
#pragma unroll
  for (int t = 0; t < Tl::BLOCKS; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f32x4 z;
#pragma unroll
      for (int c = 0; c < 4; ++c) z[c] = o[t][4 * e + c] * fall;
      *(f32x4*)(mine + col * (S::DP + 4) + t * 32 + 8 * e + 4 * half) = z;
    }
  // (the sums of another column than the thread's own are needed below)
  __syncthreads();
  if (wave == 0 && half == 0) wm[col] = top, wl[col] = sum;
  __syncthreads();
  const int quads = a.dim / 4;
  for (int n = threadIdx.x; n < 32 * quads; n += 64 * S::WAVES) {
    const int c = n / quads, d = n % quads * 4;
    const int t = c / p.heads, hh = chunk * p.heads + c % p.heads;
    if (t >= 1 << p.shift || hh >= group || i0 + t >= w.lq) continue;
    f32x4 z = (f32x4)0.0f;
#pragma unroll
    for (int v = 0; v < S::WAVES; ++v) z += *(const f32x4*)((const float*)(lds + v * S::PER_WAVE) + c * (S::DP + 4) + d);
    const long rh = (long)(w.q0 + i0 + t) * a.heads + g * group + hh;
    if (p.splits > 1) {
      if (wm[c] != -INFINITY) *(f32x4*)(p.o + (split * parts + rh) * a.dim + d) = z;
      if (d == 0) {
        p.ml[(2 * split) * parts + rh] = wm[c];
        p.ml[(2 * split + 1) * parts + rh] = wl[c];
      }
    } else {
      const float inv = wm[c] == -INFINITY ? 0.0f : 1.0f / wl[c];
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
      float finite = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[e] *= inv;
        finite = fmaf(z[e], 0.0f, finite);
        y[e] = (T)z[e];
      }
      *(t4*)((T*)a.out + rh * a.dim + d) = y;
      if (a.out32) *(f32x4*)(a.out32 + rh * a.dim + d) = z;
      if (!(finite == 0.0f)) marks[c] = 1;
      if (a.stats && d == 0) {
        const long st = (long)(g * group + hh) * a.nq + w.q0 + i0 + t;
        a.stats[st] = wm[c] == -INFINITY ? 0.0f : wm[c];
        a.stats[st + (long)a.heads * a.nq] = wm[c] == -INFINITY ? INFINITY : log2f(wl[c]);
      }
    }
  }
  if (p.splits > 1) return;
  __syncthreads();
  for (int c = wave; c < 32; c += S::WAVES)  // rows that hidden infinities or NaN reached: pair by pair
    if (marks[c]) pa_row_fwd<T>(a, w, i0 + c / p.heads, g * group + chunk * p.heads + c % p.heads);
}

// One workgroup joins the splits of one (row, head): as many of them side by side as its threads (dim / 4 a split) allow, eight
// of a thread's at a time -- a chain of latencies is what this costs.
template <typename T>
__global__ __launch_bounds__(1024) void pa_token_join_kernel(PaArgs a, TokenPlan p) {
  __shared__ f32x4 sums[1024];
  __shared__ float ls[1024], tops[16];
  __shared__ int mark;
  const long parts = (long)a.nq * a.heads, rh = blockIdx.x;
  const int row = (int)(rh / a.heads), h = (int)(rh % a.heads);
  const int quads = a.dim / 4, lanes = blockDim.x / quads, t = threadIdx.x, q = t % quads, n = t / quads;
  if (p.ml[parts + rh] < 0.0f) return;  // no sequence's row: done before
  if (t == 0) mark = 0;
  float top = -INFINITY;
  for (int s = t; s < p.splits; s += blockDim.x) top = fmaxf(top, p.ml[2 * s * parts + rh]);
  f32x4 z = (f32x4)0.0f;
  float l = 0.0f, m[8];
  f32x4 o[8];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u * lanes;
      m[u] = n < lanes && s < p.splits ? p.ml[2 * s * parts + rh] : -INFINITY;
      o[u] = (f32x4)0.0f;
      if (m[u] != -INFINITY) o[u] = *(const f32x4*)(p.o + (s * parts + rh) * a.dim + 4 * q);
    }
  };
  load(n);
  top = wave_max(top);
  if ((t & 63) == 0) tops[t >> 6] = top;
  __syncthreads();
  top = tops[0];
  for (int v = 1; v < (int)blockDim.x / 64; ++v) top = fmaxf(top, tops[v]);
  for (int s0 = n;;) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float fall = m[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[u] - top);
      l = fmaf(m[u] == -INFINITY ? 0.0f : p.ml[(2 * (s0 + u * lanes) + 1) * parts + rh], fall, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = fmaf(o[u][e], fall, z[e]);
    }
    if ((s0 += 8 * lanes) >= p.splits) break;
    load(s0);
  }
  sums[t] = z;
  ls[t] = l;
  __syncthreads();
  for (int count = lanes; count > 1;) {
    const int keep = (count + 1) / 2;
    if (n + keep < count) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[t][e] += sums[t + keep * quads][e];
      ls[t] += ls[t + keep * quads];
    }
    __syncthreads();
    count = keep;
  }
  if (t < quads) {
    z = sums[t], l = ls[t];
    const float inv = top == -INFINITY ? 0.0f : 1.0f / l;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 y;
    float finite = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[e] *= inv;
      finite = fmaf(z[e], 0.0f, finite);
      y[e] = (T)z[e];
    }
    *(t4*)((T*)a.out + rh * a.dim + 4 * t) = y;
    if (a.out32) *(f32x4*)(a.out32 + rh * a.dim + 4 * t) = z;
    if (!(finite == 0.0f)) mark = 1;
    if (a.stats && t == 0) {
      a.stats[(long)h * a.nq + row] = top == -INFINITY ? 0.0f : top;
      a.stats[(long)(a.heads + h) * a.nq + row] = top == -INFINITY ? INFINITY : log2f(l);
    }
  }
  __syncthreads();
  if (mark && t < 64) {
    const PaSeq w = pa_seq(a.s, a.nq, a.nk, pa_seq_of(a.s.cu_q, a.s.batch, a.nq, row));
    if (row >= w.q0 && row < w.q0 + w.lq) pa_row_fwd<T>(a, w, row - w.q0, h);
  }
}

static TokenPlan token_plan(int batch, int nq, int nk, int heads, int kv_heads) {
  TokenPlan p = {};
  const int group = heads / kv_heads;
  p.heads = group < 32 ? group : 32;
  p.chunks = i2r_cdiv(group, p.heads);
  while ((2 << p.shift) * p.heads <= 32) ++p.shift;
  // 2048 workgroups: four for each of the two places on a CU, so that uneven caches level out; a split has at least 256
  // of a sequence's (average) keys
  const long busy = std::max((long)std::min(batch, nq), (long)i2r_cdiv(nq, 1 << p.shift)) * kv_heads * p.chunks;
  const long most = std::max(1L, (long)nk / std::max(batch, 1) / 256);
  p.splits = (int)std::max(1L, std::min({most, (2048 + busy - 1) / std::max(busy, 1L), 512L}));
  // (many sequences without queries are workgroups too)
  const long slots = ((long)(nq >> p.shift) + batch + 2) * kv_heads * p.chunks;
  p.splits = (int)std::max(1L, std::min((long)p.splits, (1L << 22) / slots));
  return p;
}

// Few queries a sequence: one tile of columns takes a sequence's rows of a key / value head.
bool pa_is_token(int batch, int nq, int heads, int kv_heads) {
  const long rows = (nq + batch - 1) / batch;
  return rows * std::min(heads / kv_heads, 32) <= 32;
}

long pa_token_ws_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dim) {
  const TokenPlan p = token_plan(batch, nq, nk, heads, kv_heads);
  return p.splits > 1 ? (long)p.splits * nq * heads * (dim + 2) * 4 : 0;
}

template <typename T, int W>
static bool launch_token(const PaArgs& a, const TokenPlan& p, hipStream_t st) {
  typedef TokenShape<T, W> S;
  const long slots = (a.nq >> p.shift) + a.s.batch + 2;
  const dim3 grid((unsigned)(slots * a.kv_heads * p.chunks * p.splits));
  static bool done[2][64];
  if (a.table) {
    if (!i2r_lds_attr((const void*)pa_token_kernel<T, W, true>, S::lds(true, PA_MAX_DISTANCE), done[1])) return false;
    hipLaunchKernelGGL((pa_token_kernel<T, W, true>), grid, dim3(64 * S::WAVES), S::lds(true, a.s.max_distance), st, a, p);
  } else {
    if (!i2r_lds_attr((const void*)pa_token_kernel<T, W, false>, S::lds(false, 0), done[0])) return false;
    hipLaunchKernelGGL((pa_token_kernel<T, W, false>), grid, dim3(64 * S::WAVES), S::lds(false, 0), st, a, p);
  }
  if (p.splits > 1) {
    const int threads = std::min(1024, (std::min(p.splits, 128) * (a.dim / 4) + 63) / 64 * 64);
    hipLaunchKernelGGL(pa_token_join_kernel<T>, dim3((unsigned)((long)a.nq * a.heads)), dim3(threads), 0, st, a, p);
  }
  return true;
}

bool pa_launch_token(int dtype, const PaArgs& a, void* ws, hipStream_t st) {
  TokenPlan p = token_plan(a.s.batch, a.nq, a.nk, a.heads, a.kv_heads);
  p.o = (float*)ws;
  p.ml = p.o + (long)p.splits * a.nq * a.heads * a.dim;
#define PA_CALL(T, W) launch_token<T, W>(a, p, st)
  if (dtype == 0) PA_BY_WIDTH(float, PA_CALL);
  if (dtype == 1) PA_BY_WIDTH(f16_t, PA_CALL);
  PA_BY_WIDTH(bf16_t, PA_CALL);
}
