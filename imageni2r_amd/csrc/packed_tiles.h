// Tiles of packed sequences on the matrix cores.
//
// Every product here has a 32-column operand B in registers (a column is a query row in the forward and dq kernels, a key
// in the dk / dv kernel) and its other operand A in a 32-row block of an LDS tile, so that a lane's 16 accumulators belong
// to ONE column: softmax statistics, masks and rescaling are per lane, and the accumulators of the first product, rounded
// to the type, ARE the second product's B operand -- they never pass through LDS or another lane.  That works because the
// order of the contracted index is free: accumulator r of lane half h belongs to row (r & 3) + 8 * (r >> 2) + 4 * h of its
// block, and A's transposed fragments are read from LDS in that same order.
#pragma once
#include "packed_rows.h"
#include <type_traits>

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// (the low half of a flat address is the place in LDS; the plain cast would test it for null.  The host's pass, whose
// pointers are 64 bits, warns of the width.)
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"
// (m0, where a load to LDS finds its place, is a register that the compiler keeps for itself: it obeys the clobber, and warns)
#pragma clang diagnostic ignored "-Winline-asm"
#define LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(unsigned)(uintptr_t)(p))

// row of the block that accumulator r of lane half h holds
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// 16 bytes of a row: the A or B operand of one step (32 bytes of a row, half h of the lanes the h-th 16)
template <typename T>
struct Frag {
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};
template <typename T>
using frag_t = typename Frag<T>::type;

__device__ __forceinline__ void mma_step(f32x16& c, frag_t<bf16_t> a, frag_t<bf16_t> b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma_step(f32x16& c, frag_t<f16_t> a, frag_t<f16_t> b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma_step(f32x16& c, frag_t<float> a, frag_t<float> b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
}

// Head dims are worked on in five widths W: one step of a product (32 bytes: 8 fp32 or 16 elements of 16 bits), 32, 64, 96 and
// 128; rows lie in LDS in 32, 64 or 128 elements.
#define PA_BY_WIDTH(T, CALL)                                                       \
  return a.dim <= 32 / (int)sizeof(T) ? CALL(T, 32 / (int)sizeof(T))               \
         : a.dim <= 32 ? CALL(T, 32)                                               \
         : a.dim <= 64 ? CALL(T, 64)                                               \
         : a.dim <= 96 ? CALL(T, 96)                                               \
                       : CALL(T, 128)

// A tile of ROWS rows of DP elements (the head dim padded with zeros), 16-byte chunks of a row exchanged by its number so
// that the 32 rows of a fragment read, and the 4 x 64 bytes of a transposed one, fall on different banks.
template <typename T, int W, int ROWS>
struct Tile {
  static constexpr int DP = W <= 32 ? 32 : W <= 64 ? 64 : 128;
  static constexpr int ROW_BYTES = DP * (int)sizeof(T), CHUNKS = ROW_BYTES / 16, BYTES = ROWS * ROW_BYTES;
  static constexpr int STEPS = W * (int)sizeof(T) / 32;  // steps of a product over the head dim
  static constexpr int BLOCKS = (W + 31) / 32;           // 32-wide blocks of the head dim

  // What a row's chunk numbers are exchanged by (exclusive or).  LDS has 64 banks of 4 bytes: of 16 rows' equal chunks, and of
  // the 4 x 64 bytes (fp32: 2 x 128) of a transposed read, each has to fall on 16 bytes, of 256, of its own.  Made of the
  // row's bits, so that what two disjoint sets of bits give is the exclusive or of both.
  __host__ __device__ static constexpr int swizzle(int row) {
    return CHUNKS >= 16 ? (sizeof(T) == 2 ? ((row & 3) << 2) | ((row >> 2) & 3)
                                          : ((row & 4) << 1) | ((row & 3) << 1) | ((row >> 3) & 1))
           : CHUNKS == 8 ? ((row & 2) << 1) | ((row >> 2) & 3)
                         : (row >> 2) & 3;
  }

  // A lane's two places in a block of 32 rows, from which every other differs by constants.  fresh() keeps the compiler
  // from holding all those sums in registers across tiles: at a head dim of 128 they are what would spill.
  struct Lane {
    int f, t;
    __device__ __forceinline__ explicit Lane(int lane) {
      const int half = lane >> 5, col = lane & 31;
      f = col * ROW_BYTES + ((half ^ swizzle(col)) << 4);
      if (sizeof(T) == 4) {
        t = 4 * half * ROW_BYTES + (((col >> 2) ^ swizzle(4 * half)) << 4) + (col & 3) * 4;
      } else {
        const int n = lane & 15, row = 4 * half + (n >> 2), chunk = ((lane >> 4) & 1) * 2 + ((n & 3) >> 1);
        t = row * ROW_BYTES + ((chunk ^ swizzle(row)) << 4) + (n & 1) * 8;
      }
    }
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(f), "+v"(t)); }
  };

  // the lane's row of the 32 from r0 on, step s
  __device__ static __forceinline__ frag_t<T> frag(const char* tile, int r0, int s, const Lane& at) {
    return *(const frag_t<T>*)(tile + r0 * ROW_BYTES + (at.f ^ (s << 5)));
  }

  // Transposed operands of rows r0 .. r0 + 32, 32 d of block db (16-bit types)
  struct Turned {
    s16x4 part[2][2];
  };
  __device__ static __forceinline__ Turned turned(const char* tile, int r0, int db, const Lane& at) {
    // ds_read_b64_tr_b16: of each 16 lanes, lane n addresses 4 elements of row n >> 2, and gets column n of the 4 rows
    Turned x;
    const unsigned base = (unsigned)(uintptr_t)tile;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 16 * c + 8 * e;
        typedef __attribute__((address_space(3))) char lds_char;
        lds_char* from = (lds_char*)(base + (at.t ^ (db << 6) ^ (swizzle(row) << 4))) + (r0 + row) * ROW_BYTES;
        x.part[c][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
      }
    return x;
  }
  template <typename P>
  __device__ static __forceinline__ void mma_turned(const Turned& x, const P& p, f32x16& acc) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const s16x8 a = __builtin_shufflevector(x.part[c][0], x.part[c][1], 0, 1, 2, 3, 4, 5, 6, 7);
      mma_step(acc, __builtin_bit_cast(frag_t<T>, a), p[c]);
    }
  }

  // acc[32 d of block db][columns] += tile(rows r0 .. r0 + 32)^T p, p the accumulators of those rows
  template <typename P>
  __device__ static __forceinline__ void mma_t(const char* tile, int r0, int db, const Lane& at, const P& p, f32x16& acc) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = acc_row(r, 0);
        const float a = *(const float*)(tile + (r0 + row) * ROW_BYTES + (at.t ^ (db << 7) ^ (swizzle(row) << 4)));
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc, 0, 0, 0);
      }
    } else {
      mma_turned(turned(tile, r0, db, at), p, acc);
    }
  }
};

// The accumulators of a 32-row block as B operands: two fragments of 8 in the 16-bit types, the accumulators in fp32.
template <typename T>
struct Probs {
  frag_t<T> f[2];
  __device__ __forceinline__ const frag_t<T>& operator[](int c) const { return f[c]; }
  __device__ __forceinline__ void set(const f32x16& x) {
#pragma unroll
    for (int r = 0; r < 16; ++r) f[r >> 3][r & 7] = (T)x[r];
  }
  // what the rounding took away is left in x
  __device__ __forceinline__ void set_and_take(f32x16& x) {
    set(x);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] -= (float)f[r >> 3][r & 7];
  }
};
template <>
struct Probs<float> {
  f32x16 f;
  __device__ __forceinline__ float operator[](int r) const { return f[r]; }
  __device__ __forceinline__ void set(const f32x16& x) { f = x; }
};

// Loads tiles of rows of one (sequence, head) into LDS without passing through registers, by WAVES waves together or (1)
// by each wave for itself.  Rows behind the last and
// columns behind the head dim are out of the descriptor's range and arrive as zeros.
template <typename T, int W, int ROWS, int WAVES>
struct Loader {
  typedef Tile<T, W, ROWS> Tl;
  static constexpr int LOADS = Tl::BYTES / (1024 * WAVES);  // 1 KiB for each wave and instruction
  static_assert(LOADS * 1024 * WAVES == Tl::BYTES, "a tile has to be whole instructions of all waves");
  const char* base;
  long step;   // bytes from one row to the next
  int width;   // bytes of a row that hold elements
  int offset[LOADS];

  __device__ __forceinline__ void init(const T* p, long row_stride, int dim) {
    base = (const char*)p, step = row_stride * (long)sizeof(T), width = dim * (int)sizeof(T);
    const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int chunk = (i * WAVES + wave) * 64 + lane, row = chunk / Tl::CHUNKS;
      const int c = (chunk % Tl::CHUNKS) ^ Tl::swizzle(row);
      offset[i] = c * 16 < width ? (int)(row * step) + c * 16 : 0x7fffffff;
    }
  }
  // rows first .. first + ROWS of `rows` into the tile (in flight until the next tiles_ready()).
  // Written out, not by builtin: the compiler would wait for these loads before it reads any other part of LDS.
  __device__ __forceinline__ void load(char* tile, int first, int rows) const {
    const int left = min(rows - first, ROWS);
    const unsigned long long at = (unsigned long long)(base + (long)first * step);
    i32x4 rs;
    rs[0] = __builtin_amdgcn_readfirstlane((int)at);
    rs[1] = __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff);
    rs[2] = __builtin_amdgcn_readfirstlane(left > 0 ? (int)((left - 1) * step) + width : 0);
    rs[3] = 0x00020000;
    const int to = __builtin_amdgcn_readfirstlane((int)(unsigned long)LDS_PTR(char, tile) + (WAVES == 1 ? 0 : (threadIdx.x >> 6) * 1024));
    asm volatile("s_nop 4" : : "s"(rs), "s"(to));  // a vector instruction may have written them just before
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "s"(to + i * WAVES * 1024), "v"(offset[i]), "s"(rs)
                   : "memory", "m0");
  }
};

// B operand of 32 rows, straight from memory: lane's row, zeros where it does not exist
template <typename T, int STEPS>
__device__ __forceinline__ void load_rows(frag_t<T> (&f)[STEPS], const T* row, bool valid, int dim, int h) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = (2 * s + h) * N;
    f[s] = (frag_t<T>)(T)0.0f;
    if (valid && d < dim) f[s] = *(const frag_t<T>*)(row + d);
  }
}

// the value of the lane with the other half of the same column
__device__ __forceinline__ float other_half(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// workgroup barrier after which the tiles that all waves have asked for are in LDS
__device__ __forceinline__ void tiles_ready() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 4 bytes for each of up to 64 rows into LDS, by wave 0 (in flight until the next tiles_ready()); rows behind the last: 0
__device__ __forceinline__ void load_words(void* to, const void* from, int first, int rows) {
  if (threadIdx.x >= 64) return;
  const int left = min(rows - first, 64);
  const unsigned long long at = (unsigned long long)((const int*)from + first);
  i32x4 rs;
  rs[0] = __builtin_amdgcn_readfirstlane((int)at);
  rs[1] = __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff);
  rs[2] = __builtin_amdgcn_readfirstlane(max(left, 0) * 4);
  rs[3] = 0x00020000;
  const int lds = __builtin_amdgcn_readfirstlane((int)(unsigned long)LDS_PTR(char, to));
  asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"((int)threadIdx.x * 4), "s"(rs)
               : "memory", "m0");
}

// Where a tile's bias comes from: there is none; all distances lie beyond max_distance on one side; places in the sequence;
// positions that the caller gave.
enum { NONE, ONE, NEAR, GIVEN };
template <int M>
using Mode = std::integral_constant<int, M>;
using True = std::true_type;
using False = std::false_type;

__device__ __forceinline__ int floor_div(int a, int b) { return a >= 0 ? a / b : -((b - 1 - a) / b); }

// The tiles of a pass over keys (or queries), as one wave meets them: [0, begin) none of its pairs; then in turn tiles
// whose distances are all beyond max_distance (one bias, nothing hidden) up to far0, others up to near0, and so again up to
// far1 and near1; behind that none.  One loop for each kind, so that the accumulators stay where they are; every wave passes every tile's
// barrier, whichever loop it is in.
struct Passage {
  int begin, far0, near0, far1, near1;
};
template <typename Step, typename Far, typename Near, typename Idle>
__device__ __forceinline__ void walk(const Passage& p, int tiles, Step step, Far far_tile, Near near_tile, Idle idle) {
  int n = 0;
#pragma unroll 1
  for (; n < p.begin; ++n) {
    step(n);
    idle();
  }
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
#pragma unroll 1
    for (; n < (k ? p.far1 : p.far0); ++n) {
      step(n);
      far_tile(n);
    }
#pragma unroll 1
    for (; n < (k ? p.near1 : p.near0); ++n) {
      step(n);
      near_tile(n);
    }
  }
#pragma unroll 1
  for (; n < tiles; ++n) {
    step(n);
    idle();
  }
}
template <typename Step, typename Far, typename Near>
__device__ __forceinline__ void walk(const Passage& p, int tiles, Step step, Far far_tile, Near near_tile) {
  walk(p, tiles, step, far_tile, near_tile, [] {});
}

// Order of the tiles: each of the 8 XCDs (workgroups go to them in turn) works through whole heads, so that what a head's
// workgroups all read stays in that XCD's L2.
__device__ __forceinline__ bool tile_of(long slots, int heads, long& slot, int& h) {
  const long per = (slots * heads + 7) / 8, w = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (w >= slots * heads || (long)(blockIdx.x >> 3) >= per) return false;
  h = (int)(w / slots);
  slot = w % slots;
  return true;
}
static inline unsigned tile_grid(long slots, int heads) { return (unsigned)((slots * heads + 7) / 8 * 8); }

// One head's bias by distance, in log2 units, and the bucket beside it where it is wanted.  64 places more on both sides
// hold what lies beyond max_distance, so that the places of a tile's pairs follow from one of them by constants.
constexpr int PAD = 64;
struct Entry {
  float bias;
  int bucket;
};
static __host__ __device__ constexpr int table_places(int max_distance) { return 2 * (max_distance + PAD) + 1; }
__device__ __forceinline__ void load_table(float* by_distance, const i2r_packed_seqs& s, const float* table, int h) {
  for (int n = threadIdx.x; n < table_places(s.max_distance); n += blockDim.x) {
    const int b = min((int)s.lut[min(max(n - PAD, 0), 2 * s.max_distance)], s.num_buckets - 1);
    by_distance[n] = pa_log2_units(table[(long)h * s.num_buckets + b]);
  }
}
__device__ __forceinline__ void load_table(Entry* by_distance, const i2r_packed_seqs& s, const float* table, int h) {
  for (int n = threadIdx.x; n < table_places(s.max_distance); n += blockDim.x) {
    const int b = min((int)s.lut[min(max(n - PAD, 0), 2 * s.max_distance)], s.num_buckets - 1);
    by_distance[n] = {pa_log2_units(table[(long)h * s.num_buckets + b]), b};
  }
}
