// The matrix products of the vocabulary losses (vocab.hip) on the 16-bit matrix pipe, fp32 accumulation:
//   logits   z  = W . x^T      rows = vocabulary, columns = tokens, contraction over D      (both operands contraction-contiguous)
//   d x^T       = W^T . dz^T   rows = features,   columns = tokens, contraction over V      (W contraction-strided)
//   d W^T       = x^T . dz     rows = features,   columns = vocabulary, contraction over tokens  (both contraction-strided)
// Rows sit in the accumulators' register direction (a lane of v_mfma_f32_16x16x32 holds four consecutive rows of one column),
// so the softmax sums run inside a lane and every store is of consecutive elements of a row-major result.
//
// Operands of 32 bits are two fp16 planes, x s = hi + lo (s a power of two that puts the tensor's largest magnitude in
// [2^13, 2^14)); a product is hi.hi + hi.lo + lo.hi, three passes ("segments") over the contraction into one accumulator.  What is
// dropped or rounded is below 3 x 2^-24 of |a||b|, plus 2^-39 of the tensors' largest magnitudes where lo is subnormal.
#pragma once
#include "common.hpp"
#include <type_traits>

typedef unsigned short u16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// vectors at the alignment of their elements (the hardware's global accesses of 16 bytes need no more)
typedef short s16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef short s16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// ---- element types ----------------------------------------------------------------------------------------------
struct Bf16T {
  static __device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u16 enc(float v) { return __builtin_bit_cast(u16, (__bf16)v); }
  static __device__ __forceinline__ float dec(u16 v) { return __uint_as_float((unsigned)v << 16); }
};
struct F16T {
  static __device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u16 enc(float v) { return __builtin_bit_cast(u16, (_Float16)v); }
  static __device__ __forceinline__ float dec(u16 v) { return (float)__builtin_bit_cast(_Float16, v); }
};
// a 32-bit value as the sum of two fp16
__device__ __forceinline__ void split_f16(float v, u16& hi, u16& lo) {
  hi = F16T::enc(v);
  lo = F16T::enc(v - F16T::dec(hi));
}

constexpr float LOG2E = 1.4426950408889634f;

// A launch has fewer than 2^32 threads along x: workgroups beyond GRID_ROW go to further rows of the grid (GRID_ROW is a multiple of 8: they are
// dealt to the XCDs as in one row).  The last row may hold workgroups without work.
constexpr int64_t GRID_ROW = 1 << 20;
inline dim3 grid_of(int64_t groups) {
  return groups <= GRID_ROW ? dim3((unsigned)groups) : dim3((unsigned)GRID_ROW, (unsigned)((groups + GRID_ROW - 1) / GRID_ROW));
}
__device__ __forceinline__ int64_t group_id() { return (int64_t)blockIdx.y * GRID_ROW + blockIdx.x; }

// What the preparation kernels find out on the device.
struct VocabMeta {
  int rows;            // tokens that count (compacted)
  float unscale_x;     // 1 / scale of the packed x (32-bit operands; else 1)
  float unscale_w;
  float unit_g;        // the stored dz is in units of unit_g 2^exp_g
  int exp_g;
};

// A product's sums times this are the logits.  The two tensors' scales may multiply to less or more than a float holds: kept normal, so that 0
// stays 0 and the -infinity of a row that does not exist stays that (sums are below 2^53: at the lower end the logits are 0 either way).
__device__ __forceinline__ float logit_scale(const VocabMeta& m, float inv_temp) {
  return fminf(fmaxf(inv_temp * (m.unscale_x * m.unscale_w), 1.17549435e-38f), 1.7e38f);
}
// one of them exactly scaled (the same value wherever the above is not at an end)
__device__ __forceinline__ float one_logit(float sum, const VocabMeta& m, float inv_temp) {
  return (float)((double)(sum * inv_temp) * ((double)m.unscale_x * m.unscale_w));
}

// A gradient from its sums: times unit_g 2^exp_g and the other operand's scale.  Of the two scales' product only the result's magnitude matters: the
// powers of two are put together as exponents, where their product may be far outside a float while the result is not.
struct GradScale { float by; int exp; };
__device__ __forceinline__ GradScale grad_scale(const VocabMeta& m, bool by_x) {
  int e;
  const float f = frexpf(m.unit_g, &e);
  return GradScale{f, e + m.exp_g + ilogbf(by_x ? m.unscale_x : m.unscale_w)};      // (unscale_x, unscale_w: powers of two)
}
__device__ __forceinline__ float unscale(float v, const GradScale& s) { return __builtin_amdgcn_ldexpf(v * s.by, s.exp); }

constexpr int VG_BK = 64;      // contraction elements of a stage; contractions are a multiple of it

struct VocabOperand {
  const u16* p;        // first element (of plane 0)
  int64_t ld;          // elements between rows as they lie in memory
  int64_t plane;       // elements between the two planes of a 32-bit operand
  int64_t rows;        // rows that may be read: a row index beyond is clamped to the last (its products are zero or not stored)
  int cols;            // elements of a row that may be read (a multiple of 8): a chunk beyond is replaced by the last (zeros of the other operand)
};

// A split contraction over columns that are tokens: the host plans for all tokens, the device knows how many count.  With fewer column tiles
// the contraction is split further, up to `most` ways, so that `slots` workgroups have work: dx of 833 of 1111 tokens x 50257 x 1024 113 us as
// planned and 99 us so, the sums behind it 7 and 9.
struct SplitFit { int slots, most, row_tiles, col_tiles, bn; };       // slots = 0: as planned
struct Splits { int splits, col_tiles; int64_t cols; };                // cols: columns of one split's partial sums
__host__ __device__ inline Splits fit_splits(const SplitFit& f, int planned, int64_t columns, int64_t out_cols) {
  Splits s;
  s.col_tiles = (int)((columns + f.bn - 1) / f.bn);
  if (s.col_tiles > f.col_tiles) s.col_tiles = f.col_tiles;
  s.cols = (int64_t)s.col_tiles * f.bn < out_cols ? (int64_t)s.col_tiles * f.bn : out_cols;
  const int fit = s.col_tiles ? f.slots / (f.row_tiles * s.col_tiles) : planned;
  s.splits = fit > f.most ? f.most : fit;
  if (s.splits < planned) s.splits = planned;
  return s;
}

struct VocabGemm {
  VocabOperand a, b;
  int64_t k;                   // contraction length, a multiple of VG_BK (k_from_meta: meta->rows rounded up)
  int k_from_meta;
  int cols_from_meta;          // columns are tokens: column tiles behind meta->rows are left out
  int row_tiles, col_tiles, splits;
  SplitFit fit;
  const VocabMeta* meta;
  // logits
  float inv_temp;
  int64_t valid_rows;          // vocabulary rows of this piece that exist
  int first_row_tile, all_row_tiles;
  int32_t first_row;           // of the piece, in the vocabulary
  const int32_t* label;        // per column: its one target, or NULL (several, see vocab_hits)
  float2* part;                // [column][all_row_tiles] maximum z and sum of exp(z - maximum) of a row tile
  float* hit;                  // per column: the logit of its label
  const float* lse; const float* gscale;   // per column
  const float* label_p;        // per column: softmax - 1 of the label (from the loss), or NULL: the difference
  u16* dz; int64_t ld_dz, plane_dz, dz_cols;
  // products
  float* slab; int64_t ld_slab, slab_stride; int accumulate;      // [split][column][ld_slab]
  const int32_t* row_of;       // the output row of a column (tokens that count), or NULL
  const int32_t* col_exp;      // two planes, with row_of: a column's sums are 2^col_exp times too large
  void* out; int64_t ld_out, out_rows, out_cols; int unscale_by_x;   // [column][row]
};

enum { EPI_PART = 0, EPI_DZ = 1, EPI_SLAB = 2, EPI_OUT = 3, EPI_DZ_ONE = 4 };      // EPI_DZ_ONE: the vocabulary is one row tile

// ---- staging of one operand tile, 16 bytes per lane straight into LDS ------------------------------------------------
// Contraction-contiguous (STRIDED = false): LDS [T rows][64 k], 128 bytes a row; the 16-byte chunk c of row r lies at position
// c ^ (r & 7), so that the rows a fragment read touches at once cover all banks.  (Rows of 32 k, loaded 64 bytes at a time, cost 5 %.)
// Contraction-strided: LDS [64 k][T columns]; the 32-byte granule g of row k lies at g ^ h(k), so that the rows a transposing
// read touches at once lie in different banks.  (h(k + 4) = h(k) for k < 4 modulo 8, h(k + 32) = h(k).)
template <int T> __device__ __forceinline__ int granule_swizzle(int k) {
  return T >= 256 ? ((k & 3) | ((k >> 1) & 12)) : ((k & 3) | ((k >> 1) & 4));
}

// 64 lanes x 16 bytes from base + off (bytes, per lane) to 1 KB of LDS.  As a statement of its own: the compiler would order the builtin's
// LDS write against every later LDS read with a wait for all loads, and with it end the overlap of one step's loads with the step
// before.  It has no register result; the waits are in vocab_gemm's loop; nothing else in the kernel uses M0.
__device__ __forceinline__ void load_to_lds(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds(const char* from, unsigned lds) {      // every lane's own address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// A wave's share of one operand's stages: N loads of 1 KB, their lanes' byte offsets from the tile's first row (contraction-contiguous)
// or the stage's first row (contraction-strided) kept in registers.  (Fewer kilobytes than waves: some are loaded twice, so that
// every wave has the same number of loads on the way.)
template <int T, bool STRIDED, int WAVES> struct Stager {
  static constexpr int OPS = T * VG_BK * 2 / 1024, N = OPS < WAVES ? 1 : OPS / WAVES, CH = T / 8;      // CH: 16-byte chunks a strided row
  static_assert(OPS % WAVES == 0 || WAVES % OPS == 0, "whole kilobytes");
  const char* base;
  unsigned off[N];
  int64_t step_bytes, rows;
  unsigned row_bytes;
  int cols;

  static __device__ __forceinline__ int op(int u, int wave) { return (u * WAVES + wave) % OPS; }
  __device__ __forceinline__ void init(const VocabOperand& o, int64_t t0, int64_t k0, int wave, int lane) {
    row_bytes = (unsigned)(o.ld * 2);
    rows = o.rows;
    cols = o.cols;
    if (!STRIDED) {
      base = (const char*)(o.p + t0 * o.ld + k0);
      step_bytes = VG_BK * 2;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int r = op(u, wave) * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
        off[u] = (unsigned)min((int64_t)r, rows - 1 - t0) * row_bytes + c * 16;
      }
    } else {
      base = (const char*)(o.p + k0 * o.ld);
      step_bytes = VG_BK * o.ld * 2;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int idx = op(u, wave) * 64 + lane, r = idx / CH, p = idx % CH;
        const int c = (((p >> 1) ^ granule_swizzle<T>(r)) << 1) | (p & 1);
        off[u] = r * row_bytes + (unsigned)min(t0 + c * 8, (int64_t)o.cols - 8) * 2;
      }
    }
  }
  // stage s counted from k0, whose contraction index is k, `plane` bytes further on; CLAMP: the contraction may end inside or in front of it
  template <bool CLAMP> __device__ __forceinline__ void load(unsigned lds, int s, int64_t k, int64_t plane, int wave, int lane) const {
    const char* from = base + s * step_bytes + plane;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const unsigned to = lds + op(u, wave) * 1024;
      if (!CLAMP) { load_to_lds(from, off[u], to); continue; }
      // (contraction-strided: rows beyond the last; contraction-contiguous: elements beyond a row's)
      const int64_t beyond = STRIDED ? (k + (op(u, wave) * 64 + lane) / CH - (rows - 1)) * row_bytes : (k + ((lane & 7) ^ (lane >> 3)) * 8 - (cols - 8)) * 2;
      load_to_lds(from + off[u] - max(beyond, (int64_t)0), to);
    }
  }
};

// 16 x 32 fragments: lane l gets row t + (l & 15), contraction elements 32 half + 8 (l >> 4) .. + 7 of the stage, t = 16 (first + i).
template <int T, bool STRIDED, int F> struct Fragments {
  int at[STRIDED ? F : 2];
  __device__ __forceinline__ void init(int first, int lane) {
    const int i = lane & 15, quad = lane >> 4;
    if (!STRIDED) {
#pragma unroll
      for (int half = 0; half < 2; ++half) at[half] = (first * 16 + i) * (VG_BK * 2) + (((half * 4 + quad) ^ (i & 7)) << 4);
    } else {
      const int k = quad * 8 + (i >> 2);
#pragma unroll
      for (int f = 0; f < F; ++f) at[f] = k * (T * 2) + (((first + f) ^ granule_swizzle<T>(k)) << 5) + (i & 3) * 8;
    }
  }
  __device__ __forceinline__ s16x8 read(const char* lds, int f, int half) const {
    if (!STRIDED) return *reinterpret_cast<const s16x8*>(lds + at[half] + f * 16 * VG_BK * 2);
    typedef __attribute__((address_space(3))) s16x4* Lds;
    const char* p = lds + at[f] + half * 32 * T * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * T * 2));
    return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};

// A tile's 16-bit results as rows of a row-major matrix, through LDS: a lane's four rows of one column are 8 bytes of an output row,
// stored directly they reach memory in pieces of 32; rearranged they leave as whole runs of BM elements, 16 bytes a lane.  (Chunk c of output
// row v lies at c ^ v: sixteen columns' pieces go to different banks.)  value(i, j, r) is the result of row 16 i + 4 quad + r of the wave's.
template <int BM, int BN, int WM, int WN, class F, class S> __device__ __forceinline__ void store_tile(char* lds, int tid, const F& value, const S& store) {
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16, CHUNKS = BM / 8, MASK = CHUNKS - 1;
  static_assert(CHUNKS <= 32 && (CHUNKS & MASK) == 0, "chunks of a row");
  const int lane = tid & 63, wm = (tid >> 6) / WN, wn = (tid >> 6) % WN, quad = lane >> 4;
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int v = (wn * FN + j) * 16 + (lane & 15);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int c = (wm * FM + i) * 2 + (quad >> 1);
      *reinterpret_cast<s16x4*>(lds + v * (BM * 2) + ((c ^ (v & MASK)) << 4) + (quad & 1) * 8) =
          s16x4{(short)value(i, j, 0), (short)value(i, j, 1), (short)value(i, j, 2), (short)value(i, j, 3)};
    }
  }
  __syncthreads();
#pragma unroll 4
  for (int n = tid; n < BN * CHUNKS; n += 64 * WM * WN) {
    const int v = n / CHUNKS, c = n % CHUNKS;
    store(v, c * 8, *reinterpret_cast<const s16x8*>(lds + v * (BM * 2) + ((c ^ (v & MASK)) << 4)));
  }
}

// Workgroups are dealt to the eight XCDs in turn: give every XCD a contiguous share of the n tiles, and within it run through four
// row tiles at a time, so that the 32 workgroups that an XCD works on at once share four row panels and eight column panels in its L2.
// What is left of a share behind whole rounds of `at_once` tiles, if it fills half a round at most, is worked on as half tiles (of half the
// columns), so that the last round takes little more than half as long: the logits of 738 x 32001 x 768 fp32, 378 tiles on 256 CUs,
// 137 us whole and 120 us so.
// False: nothing left for this workgroup.  half: -1 whole, else which.
__device__ __forceinline__ bool tile_of(int id, int row_tiles, int col_tiles, int splits, int at_once, int& rt, int& ct, int& split, int& half) {
  const int n = row_tiles * col_tiles * splits, x = id & 7, q = n >> 3, r = n & 7;
  const int share = q + (x < r), rest = share % at_once;
  int l = id >> 3;
  half = -1;
  if (2 * rest <= at_once && l >= share - rest) {
    const int h = l - (share - rest);
    half = h & 1;
    l = share - rest + (h >> 1);
  }
  if (l >= share) return false;
  int t = x * q + min(x, r) + l;
  split = t / (row_tiles * col_tiles);
  t -= split * row_tiles * col_tiles;
  const int group = t / (4 * col_tiles), left = t - group * 4 * col_tiles, h = min(4, row_tiles - 4 * group);
  ct = left / h;
  rt = group * 4 + (left - ct * h);
  return true;
}

// The pipeline, per stage of 64 contraction elements in two halves: the products of a half run from registers while the next half is
// read from LDS into the other set of registers, and while the following stages are on their way from memory.  One barrier a stage, in its
// middle: behind it the next stage is there for every wave, and nobody reads this stage any more, whose place is loaded next.
template <class T, int BM, int BN, int WM, int WN, int STAGES, bool A_STRIDED, bool B_STRIDED, int EPI, int PLANES>
__device__ __forceinline__ void vocab_tile(const VocabGemm& g, char* const lds, const int rows, const int rt, const int64_t c0, const int split, const int splits, const int64_t slab_stride) {
  constexpr int WAVES = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, STAGE = (BM + BN) * VG_BK * 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int64_t r0 = (int64_t)rt * BM;
  const int64_t k_all = g.k_from_meta ? (int64_t)((rows + VG_BK - 1) / VG_BK) * VG_BK : g.k;
  const int64_t steps = k_all / VG_BK, k0 = steps * split / splits * VG_BK, k1 = steps * (split + 1) / splits * VG_BK;
  const int per_segment = (int)((k1 - k0) / VG_BK), n = per_segment * (PLANES == 1 ? 1 : 3);

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  Stager<BM, A_STRIDED, WAVES> sa;
  Stager<BN, B_STRIDED, WAVES> sb;
  sa.init(g.a, r0, k0, wave, lane);
  sb.init(g.b, c0, k0, wave, lane);
  Fragments<BM, A_STRIDED, FM> ra;
  Fragments<BN, B_STRIDED, FN> rb;
  ra.init(wm * FM, lane);
  rb.init(wn * FN, lane);
  const unsigned lds0 = lds_address(lds);
  constexpr int LOADS = Stager<BM, A_STRIDED, WAVES>::N + Stager<BN, B_STRIDED, WAVES>::N;        // a wave's, per stage
  int place = 0, loaded = 0;                           // where the next stage goes, and which one it is
  auto load = [&](auto clamp) {
    const unsigned to = lds0 + place * STAGE;
    // segments: lo.hi, hi.lo, hi.hi (in integers: selects by a condition end up in vector registers)
    const int first = PLANES == 1 ? -1 : (loaded - per_segment) >> 31, second = PLANES == 1 ? -1 : (loaded - 2 * per_segment) >> 31;
    const int s = PLANES == 1 ? loaded : loaded - (per_segment & ~first) - (per_segment & ~second);
    const int64_t k = k0 + (int64_t)s * VG_BK;
    sa.template load<decltype(clamp)::value>(to, s, k, PLANES == 1 ? 0 : g.a.plane * 2 & (int64_t)first, wave, lane);
    sb.template load<decltype(clamp)::value>(to + BM * VG_BK * 2, s, k, PLANES == 1 ? 0 : g.b.plane * 2 & (int64_t)(second & ~first), wave, lane);
    place = place + 1 == STAGES ? 0 : place + 1;
    ++loaded;
  };
  // The wave's LDS reads have returned (as a builtin, which the compiler counts); at most `stages` stages' loads are still on their way;
  // everybody is here.  With a memory clobber, so that the compiler moves no LDS access across it; it keeps no loads of its own in
  // flight here.
  auto sync = [&](auto stages) {
    __builtin_amdgcn_s_waitcnt(0xC07F);                // lgkmcnt(0)
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LOADS * decltype(stages)::value) : "memory");
  };
  typedef std::integral_constant<int, STAGES - 1> Others;
  typedef std::integral_constant<int, STAGES - 2> Later;
  typedef std::integral_constant<int, 0> None;
  s16x8 fa[2][FM], fb[2][FN];
  int from = 0;
  auto read = [&](int half) {
    const char* const la = lds + from * STAGE;
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[half][j] = rb.read(la + BM * VG_BK * 2, j, half);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[half][i] = ra.read(la, i, half);
  };
  auto multiply = [&](int h) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = T::mma(fa[h][i], fb[h][j], acc[i][j]);
    // the next half's LDS reads go between the first products, one by one
    constexpr int READS = FM * (A_STRIDED ? 2 : 1) + FN * (B_STRIDED ? 2 : 1), EACH = (READS + FM * FN - 1) / (FM * FN), GROUPS = (READS + EACH - 1) / EACH;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, FM * FN - GROUPS, 0);
  };
  auto next = [&] { from = from + 1 == STAGES ? 0 : from + 1; };
  if (n > 0) {
    for (int i = 0; i < STAGES && i < n; ++i) load(std::true_type());
    if (n < STAGES) sync(None()); else sync(Others());       // stage 0 is there
    read(0);
    int it = 0;
    for (; it + STAGES + 1 < n; ++it) {                      // (the last stage of the contraction may end early: not loaded here)
      read(1);
      multiply(0);
      sync(Later());
      load(std::false_type());
      next();
      read(0);
      multiply(1);
    }
    for (; it < n; ++it) {
      read(1);
      multiply(0);
      if (it + STAGES < n) { sync(Later()); load(std::true_type()); } else sync(None());
      next();
      read(0);                                               // (behind the last stage: of no use, and of no harm)
      multiply(1);
    }
  }
  __syncthreads();                                 // the epilogue uses the LDS

  const int col16 = lane & 15, quad = lane >> 4;
  // a column's label as a row of this wave's FM * 16 (outside: not here); a lane holds rows i * 16 + quad * 4 + r
  auto label_row = [&](int64_t c) {
    return g.label && c < rows ? (int64_t)g.label[c] - g.first_row - r0 - wm * FM * 16 - quad * 4 : (int64_t)-1;
  };
  // rows of the lane's that exist; in all but the last row tile every one does
  const bool whole = g.valid_rows - r0 >= (wm + 1) * FM * 16;
  const int left = (int)min(g.valid_rows - r0 - wm * FM * 16 - quad * 4, (int64_t)BM);
  auto beyond = [&](float v) {
    if (whole) return;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = i * 16 + r < left ? acc[i][j][r] : v;
  };
  // The tile's maximum and sum of exp(z - maximum) of each column (token): every wave's share into `red`, then put together by column.
  // The difference is taken before the change to base 2: z itself (exact at temperature 1) stays what the backward pass forms again, and
  // no rounding is relative to a large z.  z = acc f is formed in the difference's own instruction: an epilogue is bound by its vector
  // instructions, four cycles each (dz, all but the steps of a tile: 14.6 us with masks and selects for every element, 11.4 so; the maximum and sum 8.2 and 6.9).
  float2* const red = reinterpret_cast<float2*>(lds);        // [WM][BN]
  auto wave_stats = [&](int j, float f) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32)) * f;
    const float base = m == -INFINITY ? 0.f : m;             // nothing here: exp(-inf - 0) = 0
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) l += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], f, -base) * LOG2E);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (quad == 0) red[wm * BN + (wn * FN + j) * 16 + col16] = make_float2(m, l);
  };
  auto tile_stats = [&](int c) {
    float m = red[c].x;
#pragma unroll
    for (int w = 1; w < WM; ++w) m = fmaxf(m, red[w * BN + c].x);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < WM; ++w) l += red[w * BN + c].y * __builtin_amdgcn_exp2f((red[w * BN + c].x - base) * LOG2E);
    return make_float2(m, l);
  };
  if constexpr (EPI == EPI_PART) {
    const float f = logit_scale(*g.meta, g.inv_temp);
    beyond(-INFINITY);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t c = c0 + (wn * FN + j) * 16 + col16;
      const int64_t label = label_row(c);
      if (__any(label >= 0 && label < FM * 16)) {
        float z = 0.f;
        bool mine = false;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) { const bool is = label == i * 16 + r; z = is ? acc[i][j][r] : z; mine |= is; }
        if (mine) g.hit[c] = one_logit(z, *g.meta, g.inv_temp);
      }
      wave_stats(j, f);
    }
    __syncthreads();
    for (int c = tid; c < BN; c += 64 * WAVES)
      if (c0 + c < rows) g.part[(size_t)(c0 + c) * g.all_row_tiles + g.first_row_tile + rt] = tile_stats(c);
  } else if constexpr (EPI == EPI_DZ || EPI == EPI_DZ_ONE) {
    // dz is rounded to the operands' 16 bits here (two fp16 for 32-bit ones): the two products behind it run on the 16-bit pipe, a second plane
    // for it would be two more products of four (4096 x 131072 x 4096: 13 ms would become 20).  It is all that the gradients are off beyond their own rounding:
    // 833 x 50257 x 1024 bf16 dx 0.00208 of its norm against 0.00166, and 0.00208 with exact products of the rounded dz; 48 x 32000 x 2048 fp16 0.00028
    // against 0.00021.  A caller who needs more passes fp32.
    // softmax - 1 of a label: lse is off by half a step of its own magnitude, more than what is left in a confident row.  It comes from the
    // loss, where the caller has it (label_p), and in a vocabulary of one tile from the sum, which is formed here again.
    const float f = logit_scale(*g.meta, g.inv_temp);
    if constexpr (EPI == EPI_DZ_ONE) {
      beyond(-INFINITY);
#pragma unroll
      for (int j = 0; j < FN; ++j) wave_stats(j, f);
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t c = c0 + (wn * FN + j) * 16 + col16;
      const bool some = c < rows;
      float lse = some ? g.lse[c] : 0.f, over = 1.f;
      if constexpr (EPI == EPI_DZ_ONE) { const float2 s = tile_stats((wn * FN + j) * 16 + col16); lse = s.x; over = 1.f / s.y; }
      const float gs = some ? g.gscale[c] : 0.f, at_label = some && g.label_p ? g.label_p[c] : 0.f;      // a token that does not exist is zero (its logits are finite): it takes part in the products
      const int64_t label = label_row(c);
      auto column = [&](auto here) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float p = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], f, -lse) * LOG2E);
            if (EPI == EPI_DZ_ONE) p *= over;
            if (here && label == i * 16 + r) p = g.label_p ? at_label : p - 1.f;
            acc[i][j][r] = p * gs;
          }
      };
      if (__any(label >= 0 && label < FM * 16)) column(std::true_type()); else column(std::false_type());
    }
    beyond(0.f);                                             // and so is a vocabulary row that does not exist
    if (EPI == EPI_DZ_ONE) __syncthreads();
    if constexpr (PLANES == 1) {
      store_tile<BM, BN, WM, WN>(lds, tid, [&](int i, int j, int r) { return T::enc(acc[i][j][r]); },
                                 [&](int v, int d, s16x8 x) { if (c0 + v < g.dz_cols) *reinterpret_cast<s16x8*>(g.dz + (c0 + v) * g.ld_dz + r0 + d) = x; });
    } else {
      // (two planes: twice through LDS takes longer than storing 8 bytes a lane, 100 against 78 us at 777 x 16128 x 768)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int64_t c = c0 + (wn * FN + j) * 16 + col16;
        if (c >= g.dz_cols) continue;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          u16 hi[4], lo[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) split_f16(acc[i][j][r], hi[r], lo[r]);
          u16* to = g.dz + c * g.ld_dz + r0 + (wm * FM + i) * 16 + quad * 4;
          *reinterpret_cast<s16x4*>(to) = s16x4{(short)hi[0], (short)hi[1], (short)hi[2], (short)hi[3]};
          *reinterpret_cast<s16x4*>(to + g.plane_dz) = s16x4{(short)lo[0], (short)lo[1], (short)lo[2], (short)lo[3]};
        }
      }
    }
    if (BN < VG_BK)          // one column tile: the rest of the contraction's step over tokens
      for (int n = tid; n < (VG_BK - BN) * (BM / 8); n += 64 * WAVES)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          *reinterpret_cast<s16x8*>(g.dz + p * g.plane_dz + (BN + n / (BM / 8)) * g.ld_dz + r0 + n % (BM / 8) * 8) = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
  } else if constexpr (EPI == EPI_SLAB) {
    float* slab = g.slab + split * slab_stride;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t c = c0 + (wn * FN + j) * 16 + col16;
      if (c >= g.out_cols) continue;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int64_t row = r0 + (wm * FM + i) * 16 + quad * 4;
        if (row >= g.ld_slab) continue;                  // ld_slab is a multiple of 64
        f32x4* p = reinterpret_cast<f32x4*>(slab + c * g.ld_slab + row);
        f32x4 v = acc[i][j];
        if (g.accumulate) v += *p;
        *p = v;
      }
    }
  } else {
    const GradScale f = grad_scale(*g.meta, g.unscale_by_x);
    const int64_t cols = g.row_of ? (int64_t)rows : g.out_cols;
    if constexpr (PLANES == 2) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int64_t c = c0 + (wn * FN + j) * 16 + col16;
        if (c >= cols) continue;
        float* out = (float*)g.out + (g.row_of ? g.row_of[c] : c) * g.ld_out;
        const GradScale own = {f.by, f.exp - (g.row_of ? g.col_exp[c] : 0)};
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const int64_t row = r0 + (wm * FM + i) * 16 + quad * 4;
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = unscale(acc[i][j][r], own);
          if (row + 4 <= g.out_rows) *reinterpret_cast<f32x4u*>(out + row) = v;
          else
#pragma unroll
            for (int r = 0; r < 4; ++r) if (row + r < g.out_rows) out[row + r] = v[r];
        }
      }
    } else {
      store_tile<BM, BN, WM, WN>(lds, tid, [&](int i, int j, int r) { return T::enc(unscale(acc[i][j][r], f)); }, [&](int v, int d, s16x8 x) {
        const int64_t c = c0 + v, row = r0 + d;
        if (c >= cols) return;
        u16* p = (u16*)g.out + (g.row_of ? g.row_of[c] : c) * g.ld_out + row;
        if (row + 8 <= g.out_rows) *reinterpret_cast<s16x8u*>(p) = x;
        else
#pragma unroll
          for (int r = 0; r < 8; ++r) if (row + r < g.out_rows) p[r] = (u16)x[r];
      });
    }
  }
}

// half tiles: 128 columns of 256 (a contraction-strided operand needs that many), 64 of 128
template <int BN, bool B_STRIDED> constexpr bool vocab_halves() { return BN >= 256 || (BN == 128 && !B_STRIDED); }
template <int BM> constexpr int vocab_at_once() { return BM >= 256 ? 32 : 64; }        // workgroups of an XCD: one or two a CU
template <class T, int BM, int BN, int WM, int WN, int STAGES, bool A_STRIDED, bool B_STRIDED, int EPI, int PLANES>
__global__ void __launch_bounds__(64 * WM * WN, 2) vocab_gemm(const VocabGemm g) {
  __shared__ __attribute__((aligned(16))) char lds[STAGES * (BM + BN) * VG_BK * 2];
  const int rows = g.meta->rows;
  // (the last step of a contraction over tokens reads dz up to the next multiple of its length)
  const int most = (rows + VG_BK - 1) & ~(VG_BK - 1);
  const int col_tiles = g.cols_from_meta ? min(g.col_tiles, (most + BN - 1) / BN) : g.col_tiles;
  int splits = g.splits;
  int64_t slab_stride = g.slab_stride;
  if (EPI == EPI_SLAB && g.fit.slots) {
    const Splits f = fit_splits(g.fit, splits, most, g.out_cols);
    splits = f.splits;
    slab_stride = f.cols * g.ld_slab;
  }
  constexpr bool HALVES = vocab_halves<BN, B_STRIDED>();
  int rt, ct, split, half;
  if (!tile_of(blockIdx.x, g.row_tiles, col_tiles, splits, HALVES ? vocab_at_once<BM>() : 1, rt, ct, split, half)) return;
  if constexpr (HALVES)
    if (half >= 0) {
      const int64_t c0 = (int64_t)ct * BN + half * (BN / 2);
      if (g.cols_from_meta && c0 >= most) return;
      return vocab_tile<T, BM, BN / 2, 4, WM * WN / 4, STAGES, A_STRIDED, B_STRIDED, EPI, PLANES>(g, lds, rows, rt, c0, split, splits, slab_stride);
    }
  vocab_tile<T, BM, BN, WM, WN, STAGES, A_STRIDED, B_STRIDED, EPI, PLANES>(g, lds, rows, rt, (int64_t)ct * BN, split, splits, slab_stride);
}
