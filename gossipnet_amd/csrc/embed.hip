// Rows of a vocabulary table for token ids, scaled, and the table's gradient summed in token order.
//   forward    y[m] = scale * s[m] * table[id[m]]                 (zero where the id is outside [0, V))
//   backward   d table[v] = scale * sum over the tokens m with id[m] = v, ascending, of s[m] * dy[m]
//              d s[m] = scale * dy[m] . table[id[m]]
// Every kernel here moves bytes: M rows in, M rows out; the backward pass reads M rows of dy and writes the V rows of the table's
// gradient once, the rows without a token included.
//   embed_sort    keys (id << 32 | token), distinct, sorted per 4096 tokens; embed_merge joins 16 sorted runs at a time by binary
//                 searches (no atomics: the order of every sum is fixed)
//   embed_sums    four kinds of workgroups in one launch: sums of the runs of equal ids (a wave starts where a run starts), partial sums
//                 of the runs of more than HOT tokens per HOT sorted tokens, zeros for the rows without a token, d s
//   embed_hot_rows  adds a long run's partial sums
// or, for few tokens and a small table, embed_few alone, and for at most 64 tokens embed_wave.
#include "vocab_gemm.hpp"

namespace {

typedef unsigned long long u64;
constexpr unsigned NONE = 0xffffffffu;      // id of a token that is left out: sorted behind all others
constexpr int RUN = 4096;          // tokens sorted by one workgroup: 32 KB of keys
constexpr int WAY = 16;            // runs joined by one merge pass
constexpr int HOT = 16;            // tokens a row's own wave adds up
constexpr int BLOCKS = 2;          // column blocks of 64 * VEC elements a wave keeps sums of
constexpr int FILL_ROWS = 64;      // table rows a workgroup looks for and fills with zeros

template <int DT> struct Elem { typedef u16 type; };
template <> struct Elem<GNET_F32> { typedef float type; };
template <int DT> __device__ __forceinline__ float dec(typename Elem<DT>::type v) {
  if constexpr (DT == GNET_F32) return v;
  else if constexpr (DT == GNET_BF16) return Bf16T::dec(v);
  else return F16T::dec(v);
}
template <int DT> __device__ __forceinline__ typename Elem<DT>::type enc(float v) {
  if constexpr (DT == GNET_F32) return v;
  else if constexpr (DT == GNET_BF16) return Bf16T::enc(v);
  else return F16T::enc(v);
}
// VEC elements of a row at once, at the alignment of an element; what is left behind the last whole VEC one by one
template <class E, int VEC> struct Pack {
  typedef E V __attribute__((ext_vector_type(VEC)));
  typedef E U __attribute__((ext_vector_type(VEC), aligned(sizeof(E))));
  V v;
};
template <class E, int VEC> __device__ __forceinline__ Pack<E, VEC> load_pack(const E* p, int64_t left) {
  Pack<E, VEC> o;
  if (left >= VEC) o.v = *reinterpret_cast<const typename Pack<E, VEC>::U*>(p);
  else
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = i < left ? p[i] : (E)0;
  return o;
}
template <class E, int VEC> __device__ __forceinline__ void store_pack(E* p, const Pack<E, VEC>& o, int64_t left) {
  if (left >= VEC) *reinterpret_cast<typename Pack<E, VEC>::U*>(p) = o.v;
  else
#pragma unroll
    for (int i = 0; i < VEC; ++i) if (i < left) p[i] = o.v[i];
}

__device__ __forceinline__ int64_t load_id(const void* p, int64_t i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// ---- forward ------------------------------------------------------------------------------------------------------
struct ForwardArgs {
  const void* ids; int ids64; int64_t M, V, D;
  const void* table; int64_t ld; float scale; const float* token_scale;
  void* y; int blocks;                 // column blocks of 64 * VEC elements a row
};
template <int DT, int VEC> __global__ void __launch_bounds__(256) embed_rows_out(const ForwardArgs a) {
  typedef typename Elem<DT>::type E;
  const int64_t w = group_id() * 4 + (threadIdx.x >> 6);
  const int64_t m = w / a.blocks, d = ((w % a.blocks) * 64 + (threadIdx.x & 63)) * VEC;
  if (m >= a.M || d >= a.D) return;
  const int64_t id = load_id(a.ids, m, a.ids64);
  Pack<E, VEC> o;
  if (id >= 0 && id < a.V) {
    const Pack<E, VEC> t = load_pack<E, VEC>((const E*)a.table + id * a.ld + d, a.D - d);
    const float s = a.token_scale ? a.scale * a.token_scale[m] : a.scale;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = enc<DT>(dec<DT>(t.v[i]) * s);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = enc<DT>(0.f);
  }
  store_pack<E, VEC>((E*)a.y + m * a.D + d, o, a.D - d);
}

// ---- the order of the tokens ------------------------------------------------------------------------------------------
// Bitonic sort of one run, four consecutive keys a thread: partners up to 2 apart are the thread's own, up to 128 apart the wave's (lane
// exchanges), the rest go through LDS -- 10 of the 78 steps.  KEY = 32 bits, id << 12 | place in the run, where ids fit into 20 bits,
// else 64.  Keys are distinct, so the result is the stable order.
template <int X> __device__ __forceinline__ unsigned lane_xor(unsigned v) {
  if constexpr (X == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true);
  else if constexpr (X == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true);
  else if constexpr (X == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);       // a rotation by 8 within 16
  else if constexpr (X == 32) return __shfl_xor(v, 32);
  else return __builtin_amdgcn_ds_swizzle(v, (X << 10) | 0x1f);
}
template <int X> __device__ __forceinline__ u64 lane_xor(u64 v) {
  return (u64)lane_xor<X>((unsigned)(v >> 32)) << 32 | lane_xor<X>((unsigned)v);
}
template <class KEY> __device__ __forceinline__ void order(KEY& a, KEY& b, bool up) {
  const KEY lo = a < b ? a : b, hi = a < b ? b : a;
  a = up ? lo : hi;
  b = up ? hi : lo;
}
template <class KEY, int X> __device__ __forceinline__ void lane_step(KEY (&v)[4], bool up) {
  const bool low = !(threadIdx.x & X);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const KEY o = lane_xor<X>(v[i]);
    v[i] = (v[i] < o) == (low == up) ? v[i] : o;
  }
}
template <class KEY> __global__ void __launch_bounds__(RUN / 4) embed_sort(const void* ids, int ids64, int64_t M, int64_t V, int n, u64* __restrict__ keys) {
  __shared__ __attribute__((aligned(16))) KEY s[RUN];
  constexpr int PLACE = sizeof(KEY) == 4 ? 12 : 32;
  constexpr KEY OUT = sizeof(KEY) == 4 ? (KEY)0xfffff : (KEY)NONE;            // behind every id: no token
  const int64_t base = (int64_t)blockIdx.x * RUN;
  const int t0 = threadIdx.x * 4;
  KEY v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    KEY id = OUT;
    if (base + t0 + i < M) {
      const int64_t x = load_id(ids, base + t0 + i, ids64);
      if (x >= 0 && x < V) id = (KEY)x;
    }
    v[i] = id << PLACE | (KEY)(t0 + i);
  }
  for (int k = 2; k <= n; k <<= 1) {
    for (int j = k >> 1; j >= 256; j >>= 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t0 + i] = v[i];
      __syncthreads();
      const bool keep_low = !(t0 & j) == !(t0 & k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const KEY o = s[(t0 ^ j) + i];
        v[i] = (v[i] < o) == keep_low ? v[i] : o;
      }
    }
    const bool up = !(t0 & k);
    if (k > 128) lane_step<KEY, 32>(v, up);
    if (k > 64) lane_step<KEY, 16>(v, up);
    if (k > 32) lane_step<KEY, 8>(v, up);
    if (k > 16) lane_step<KEY, 4>(v, up);
    if (k > 8) lane_step<KEY, 2>(v, up);
    if (k > 4) lane_step<KEY, 1>(v, up);
    if (k > 2) { order(v[0], v[2], up); order(v[1], v[3], up); order(v[0], v[1], up); order(v[2], v[3], up); }
    else { order(v[0], v[1], true); order(v[2], v[3], false); }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const KEY id = v[i] >> PLACE;
    const int64_t m = base + (int64_t)(v[i] & (((KEY)1 << PLACE) - 1));
    // (places behind the last token of a short run sort behind the tokens that are left out: they came later)
    if (base + t0 + i < M) keys[base + t0 + i] = (id == OUT ? (u64)NONE : (u64)id) << 32 | (u64)m;
  }
}

// keys of [lo, hi) below `key`
__device__ __forceinline__ int64_t lower_bound(const u64* __restrict__ keys, int64_t lo, int64_t hi, u64 key) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}
// WAY lanes a key: each counts the smaller keys of one run; their sum is the key's place
__global__ void __launch_bounds__(256) embed_merge(const u64* __restrict__ in, u64* __restrict__ out, int64_t M, int64_t run) {
  const int64_t i = (int64_t)blockIdx.x * (256 / WAY) + threadIdx.x / WAY;
  const bool some = i < M;
  const u64 key = some ? in[i] : 0;
  const int64_t own = i / run, first = own / WAY * WAY, r = first + threadIdx.x % WAY;
  int n = 0;
  if (some && r * run < M) n = r == own ? (int)(i - own * run) : (int)(lower_bound(in, r * run, min(M, (r + 1) * run), key) - r * run);
#pragma unroll
  for (int o = WAY / 2; o; o >>= 1) n += __shfl_xor(n, o);
  if (some && threadIdx.x % WAY == 0) out[first * run + n] = key;
}

// ---- backward ------------------------------------------------------------------------------------------------------
struct BackwardArgs {
  const u64* keys; int64_t M, V, D;
  const void* dy; int64_t ld; float scale; const float* token_scale;
  void* out; int64_t ld_out; int accumulate;
  float* part; int64_t ld_part;        // [segment][2][D rounded up to 8]
  unsigned hot_groups, run_groups, scale_groups, fill_groups;     // workgroups of each kind, in this order
  const void* ids; int ids64; const void* table; int64_t ld_table; float* dscale;
};

// Sums over tokens held by the wave's lanes [lo, hi), in order, for `blocks` <= NB column blocks `step` elements apart from column d on;
// U tokens' rows are on the way at a time.
template <int DT, int VEC, int U, int NB> __device__ __forceinline__ void add_tokens(float (&sum)[NB][VEC], const BackwardArgs& a, int token, int lo, int hi, int64_t d, int step, int blocks) {
  typedef typename Elem<DT>::type E;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[b][i] = 0.f;
  for (int j = lo; j < hi; j += U) {
    Pack<E, VEC> g[U][NB];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= hi) continue;
      const int64_t m = __builtin_amdgcn_readlane(token, j + u);
      s[u] = a.token_scale ? a.token_scale[m] : 1.f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (b < blocks && d + b * step < a.D) g[u][b] = load_pack<E, VEC>((const E*)a.dy + m * a.ld + d + b * step, a.D - d - b * step);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= hi) continue;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (b < blocks && d + b * step < a.D)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[b][i] = fmaf(dec<DT>(g[u][b].v[i]), s[u], sum[b][i]);
    }
  }
}
template <int DT, int VEC> __device__ __forceinline__ void store_row(const float (&sum)[VEC], const BackwardArgs& a, int64_t v, int64_t d) {
  typedef typename Elem<DT>::type E;
  E* p = (E*)a.out + v * a.ld_out + d;
  Pack<E, VEC> o;
  if (a.accumulate) o = load_pack<E, VEC>(p, a.D - d);
#pragma unroll
  for (int i = 0; i < VEC; ++i) o.v[i] = enc<DT>(a.accumulate ? dec<DT>(o.v[i]) + sum[i] * a.scale : sum[i] * a.scale);
  store_pack<E, VEC>(p, o, a.D - d);
}

// 64 consecutive keys from place p on, one a lane: id (NONE outside the order) and token
__device__ __forceinline__ void load_keys(const BackwardArgs& a, int64_t p, unsigned& id, int& token) {
  const int64_t i = p + (threadIdx.x & 63);
  const u64 key = i >= 0 && i < a.M ? a.keys[i] : ~0ull;
  id = (unsigned)(key >> 32);
  token = (int)(unsigned)key;
}

// A wave per place of the sorted order: where a run of at most HOT tokens starts, its sum.
template <int DT, int VEC> __device__ __forceinline__ void run_sums(const BackwardArgs& a, int64_t p) {
  if (p >= a.M) return;
  unsigned ids;
  int token;
  load_keys(a, p - 1, ids, token);                           // lane 0: the place in front
  const unsigned id = __builtin_amdgcn_readlane(ids, 1);
  if (id == NONE || (p > 0 && (unsigned)__builtin_amdgcn_readlane(ids, 0) == id)) return;
  const int n = __popcll(__ballot(ids == id));               // (equal ids are next to each other)
  if (n > HOT) return;
  const int lane = threadIdx.x & 63;
  for (int64_t d0 = 0; d0 < a.D; d0 += BLOCKS * 64 * VEC) {
    const int blocks = (int)min((int64_t)BLOCKS, (a.D - d0 + 64 * VEC - 1) / (64 * VEC));
    const int64_t d = d0 + lane * VEC;
    float sum[BLOCKS][VEC];
    add_tokens<DT, VEC, 4, BLOCKS>(sum, a, token, 1, 1 + n, d, 64 * VEC, blocks);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
      if (b < blocks && d + b * 64 * VEC < a.D) store_row<DT, VEC>(sum[b], a, id, d + b * 64 * VEC);
  }
}

// The runs of more than HOT equal ids: a segment of HOT sorted tokens meets at most two, one that comes in over its first token
// (slot 0: also a run that starts right there and leaves) and one that leaves over its last (slot 1).  A run that crosses a border of
// the segment has more than HOT tokens if the HOT places on either side of it hold that many.
static_assert(3 * HOT <= 64, "a segment and its neighbours are a wave's keys");
template <int DT, int VEC> __device__ __forceinline__ void hot_sums(const BackwardArgs& a, int64_t seg) {
  const int64_t lo = seg * HOT;
  unsigned ids;
  int token;
  load_keys(a, lo - HOT, ids, token);                        // lanes HOT .. 2 HOT - 1: the segment
  const int end = (int)min((int64_t)HOT, a.M - lo) + HOT;
  const unsigned first = __builtin_amdgcn_readlane(ids, HOT), last = __builtin_amdgcn_readlane(ids, end - 1);
  const bool in = first != NONE && (unsigned)__builtin_amdgcn_readlane(ids, HOT - 1) == first;
  const bool leaves = last != NONE && (unsigned)__builtin_amdgcn_readlane(ids, end) == last;
  for (int slot = 0; slot < 2; ++slot) {
    const unsigned id = slot ? last : first;
    if (slot ? !(leaves && first != last) : !(in || (leaves && first == last))) continue;
    const u64 run = __ballot(ids == id);                     // the run as far as these keys show it
    if (__popcll(run) <= HOT) continue;
    const int b = max(HOT, (int)__builtin_ctzll(run)), e = min(end, 64 - (int)__builtin_clzll(run));
    for (int64_t d = (int64_t)threadIdx.x * VEC; d < a.D; d += 256 * VEC) {
      float sum[1][VEC];
      add_tokens<DT, VEC, 8, 1>(sum, a, token, b, e, d, 0, 1);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a.part[(seg * 2 + slot) * a.ld_part + d + i] = sum[0][i];
    }
  }
}

// Zeros for those of FILL_ROWS rows that no token has (each row's tokens by binary search).
template <int DT, int VEC> __device__ __forceinline__ void fill_rows(const BackwardArgs& a, int64_t group, int64_t* start) {
  typedef typename Elem<DT>::type E;
  const int64_t v0 = group * FILL_ROWS;
  if (threadIdx.x <= FILL_ROWS) start[threadIdx.x] = lower_bound(a.keys, 0, a.M, (u64)(v0 + threadIdx.x) << 32);
  __syncthreads();
  Pack<E, VEC> zero;
#pragma unroll
  for (int i = 0; i < VEC; ++i) zero.v[i] = enc<DT>(0.f);
  for (int r = threadIdx.x >> 6; r < FILL_ROWS && v0 + r < a.V; r += 4)
    if (start[r] == start[r + 1])
      for (int64_t d = (int64_t)(threadIdx.x & 63) * VEC; d < a.D; d += 64 * VEC) store_pack<E, VEC>((E*)a.out + (v0 + r) * a.ld_out + d, zero, a.D - d);
}

template <int DT, int VEC> __device__ __forceinline__ void scale_gradient(const BackwardArgs& a, int64_t m) {
  typedef typename Elem<DT>::type E;
  if (m >= a.M) return;
  const int64_t id = load_id(a.ids, m, a.ids64);
  float dot = 0.f;
  if (id >= 0 && id < a.V) {
#pragma unroll 4
    for (int64_t d = (int64_t)(threadIdx.x & 63) * VEC; d < a.D; d += 64 * VEC) {
      const Pack<E, VEC> t = load_pack<E, VEC>((const E*)a.table + id * a.ld_table + d, a.D - d);
      const Pack<E, VEC> g = load_pack<E, VEC>((const E*)a.dy + m * a.ld + d, a.D - d);
#pragma unroll
      for (int i = 0; i < VEC; ++i) dot = fmaf(dec<DT>(t.v[i]), dec<DT>(g.v[i]), dot);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
  }
  if ((threadIdx.x & 63) == 0) a.dscale[m] = dot * a.scale;
}

template <int DT, int VEC> __global__ void __launch_bounds__(256) embed_sums(const BackwardArgs a) {
  __shared__ int64_t start[FILL_ROWS + 1];
  int64_t g = group_id();
  const int wave = threadIdx.x >> 6;
  if (g < a.hot_groups) return hot_sums<DT, VEC>(a, g);
  g -= a.hot_groups;
  if (g < a.run_groups) return run_sums<DT, VEC>(a, g * 4 + wave);
  g -= a.run_groups;
  if (g < a.scale_groups) return scale_gradient<DT, VEC>(a, g * 4 + wave);
  g -= a.scale_groups;
  if (g < a.fill_groups) fill_rows<DT, VEC>(a, g, start);
}

// The segment in which a hot run starts adds the run's partial sums, a workgroup per column block: each wave a quarter of them in order,
// then the quarters in order.
template <int DT, int VEC> __global__ void __launch_bounds__(256) embed_hot_rows(const BackwardArgs a) {
  __shared__ float quarter[3][64 * VEC];
  const int64_t seg = blockIdx.x, lo = seg * HOT, hi = lo + HOT;
  if (hi >= a.M) return;
  unsigned ids;
  int token;
  load_keys(a, lo - HOT, ids, token);
  const unsigned id = __builtin_amdgcn_readlane(ids, 2 * HOT - 1);
  if (id == NONE || (unsigned)__builtin_amdgcn_readlane(ids, 2 * HOT) != id) return;         // no run leaves this segment
  const bool whole = (unsigned)__builtin_amdgcn_readlane(ids, HOT) == id;
  if (whole && (unsigned)__builtin_amdgcn_readlane(ids, HOT - 1) == id) return;              // it started earlier
  if (__popcll(__ballot(ids == id)) <= HOT) return;                                          // run_sums has it
  const int64_t n = (lower_bound(a.keys, hi, a.M, ((u64)id + 1) << 32) - 1) / HOT - seg;      // segments behind this one
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t s0 = seg + 1 + n * wave / 4, s1 = seg + 1 + n * (wave + 1) / 4;
  const int64_t d = ((int64_t)blockIdx.y * 64 + lane) * VEC;
  float sum[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
  if (d < a.D) {
    if (wave == 0)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] = a.part[(seg * 2 + (whole ? 0 : 1)) * a.ld_part + d + i];
#pragma unroll 4
    for (int64_t s = s0; s < s1; ++s)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] += a.part[s * 2 * a.ld_part + d + i];
  }
  if (wave)
#pragma unroll
    for (int i = 0; i < VEC; ++i) quarter[wave - 1][lane * VEC + i] = sum[i];
  __syncthreads();
  if (wave == 0 && d < a.D) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = ((sum[i] + quarter[0][lane * VEC + i]) + quarter[1][lane * VEC + i]) + quarter[2][lane * VEC + i];
    store_row<DT, VEC>(sum, a, id, d);
  }
}

// A small table and few tokens: no order is needed.  A workgroup per row of the table and column block looks through all ids, its 16 waves
// a share of the tokens each, and adds up those of its row; more workgroups for d s.  One launch for three.
constexpr int FEW = 2048, FEW_WAVES = 16;          // tokens at most
template <int DT, int VEC> __global__ void __launch_bounds__(64 * FEW_WAVES) embed_few(const BackwardArgs a) {
  __shared__ int list[FEW_WAVES][FEW / FEW_WAVES];
  __shared__ float sums[FEW_WAVES][64 * VEC];
  __shared__ int found[FEW_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x < a.scale_groups) {
    if (blockIdx.y == 0) scale_gradient<DT, VEC>(a, (int64_t)blockIdx.x * FEW_WAVES + wave);
    return;
  }
  const int64_t v = blockIdx.x - a.scale_groups, d0 = (int64_t)blockIdx.y * 64 * VEC, d = d0 + lane * VEC;
  const int share = (int)((a.M + 64 * FEW_WAVES - 1) / (64 * FEW_WAVES)) * 64, first = wave * share;
  bool mine[FEW / FEW_WAVES / 64];
#pragma unroll
  for (int i = 0; i < FEW / FEW_WAVES / 64; ++i) {
    const int m = first + i * 64 + lane;
    mine[i] = i * 64 < share && m < a.M && load_id(a.ids, m, a.ids64) == v;
  }
  int n = 0;
#pragma unroll
  for (int i = 0; i < FEW / FEW_WAVES / 64; ++i) {
    const u64 all = __ballot(mine[i]);
    if (mine[i]) list[wave][n + __popcll(all & ((1ull << lane) - 1))] = first + i * 64 + lane;
    n += __popcll(all);
  }
  if (lane == 0) found[wave] = n;
  float sum[1][VEC], more[1][VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[0][i] = 0.f;
  for (int j = 0; j < n; j += 64) {                  // (a wave reads what it wrote itself)
    const int token = j + lane < n ? list[wave][j + lane] : 0;
    add_tokens<DT, VEC, 8, 1>(more, a, token, 0, min(64, n - j), d, 0, 1);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[0][i] += more[0][i];
  }
  if (n)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[wave][lane * VEC + i] = sum[0][i];
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < FEW_WAVES; ++w) total += found[w];
  const int c = threadIdx.x;
  if (c >= 64 * VEC || d0 + c >= a.D || (a.accumulate && !total)) return;
  float all[1] = {0.f};
#pragma unroll
  for (int w = 0; w < FEW_WAVES; ++w)
    if (found[w]) all[0] += sums[w][c];
  store_row<DT, 1>(all, a, v, d0 + c);
}
// Measured against the sorted order: 2000 tokens, a table of 81 x 128 8 and 18 us, of 2048 x 64 10 and 18; 16 tokens, 4096 x 64 (not taken)
// 12 and 9.  The worst case, all tokens of one row, is bound by what one CU can fetch: 2000 tokens 28 and 21 us, 4096 (not taken) 53 and 28.
bool few(int64_t M, int64_t V, int64_t column_blocks) { return M <= FEW && V * column_blocks <= 2048; }

// At most a wave of tokens: every wave holds all ids and finds the tokens of one by a ballot.  Workgroups as in embed_sums, without the
// long runs: sums (a wave per token and column block, at work where the token is its row's first), d s, rows without a token.  One launch
// for two or three: 64 tokens, 5000 x 512 bf16 5.6 and 11.8 us, 40000 x 4096 60 and 63.
constexpr int WAVE = 64;
template <int DT, int VEC> __global__ void __launch_bounds__(256) embed_wave(const BackwardArgs a) {
  typedef typename Elem<DT>::type E;
  __shared__ int have[FILL_ROWS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t g = group_id();
  if (g >= a.run_groups && g - a.run_groups < a.scale_groups) return scale_gradient<DT, VEC>(a, (g - a.run_groups) * 4 + wave);
  int64_t id = -1;
  if (lane < a.M) id = load_id(a.ids, lane, a.ids64);
  if (id < 0 || id >= a.V) id = -1;
  if (g < a.run_groups) {
    const int64_t blocks = (a.D + 64 * VEC - 1) / (64 * VEC), w = g * 4 + wave, m = w / blocks, d = (w % blocks * 64 + lane) * VEC;
    if (m >= a.M) return;
    const int64_t row = __shfl(id, (int)m);
    const u64 mine = __ballot(id == row);
    if (row < 0 || __builtin_ctzll(mine) != m) return;
    int token = 0;                                    // lane k: the row's token number k
    if (id == row) token = lane;
    token = __builtin_amdgcn_ds_permute((id == row ? __popcll(mine & ((1ull << lane) - 1)) : 63 - __popcll(~mine & ((1ull << lane) - 1))) * 4, token);
    float sum[1][VEC];
    add_tokens<DT, VEC, 8, 1>(sum, a, token, 0, __popcll(mine), d, 0, 1);
    if (d < a.D) store_row<DT, VEC>(sum[0], a, row, d);
    return;
  }
  const int64_t v0 = (g - a.run_groups - a.scale_groups) * FILL_ROWS;
  if (v0 >= (int64_t)a.fill_groups * FILL_ROWS) return;
  if (threadIdx.x < FILL_ROWS) have[threadIdx.x] = 0;
  __syncthreads();
  if (wave == 0 && id >= v0 && id < v0 + FILL_ROWS) have[id - v0] = 1;
  __syncthreads();
  Pack<E, VEC> zero;
#pragma unroll
  for (int i = 0; i < VEC; ++i) zero.v[i] = enc<DT>(0.f);
  for (int k = wave; k < FILL_ROWS && v0 + k < a.V; k += 4)
    if (!have[k])
      for (int64_t d = (int64_t)lane * VEC; d < a.D; d += 64 * VEC) store_pack<E, VEC>((E*)a.out + (v0 + k) * a.ld_out + d, zero, a.D - d);
}

// Elements a lane takes at once: 16 bytes, or as many as still give every lane of a wave something to do.
int pick_vec(int dtype, int64_t D) {
  int v = dtype == GNET_F32 ? 4 : 8;
  while (v > 1 && D < 64 * v) v >>= 1;
  return v;
}
template <template <int, int> class F, class A> void launch(int dtype, int vec, const A& a, dim3 grid, hipStream_t s) {
#define GO(DT)                                                  \
  switch (vec) {                                                \
    case 1: F<DT, 1>::go(a, grid, s); break;                    \
    case 2: F<DT, 2>::go(a, grid, s); break;                    \
    case 4: F<DT, 4>::go(a, grid, s); break;                    \
    default: F<DT, DT == GNET_F32 ? 4 : 8>::go(a, grid, s);     \
  }
  if (dtype == GNET_F32) { GO(GNET_F32) } else if (dtype == GNET_BF16) { GO(GNET_BF16) } else { GO(GNET_F16) }
#undef GO
}
#define KERNEL_OF(name, kernel, args, threads) \
  template <int DT, int VEC> struct name { static void go(const args& a, dim3 grid, hipStream_t s) { kernel<DT, VEC><<<grid, threads, 0, s>>>(a); } }
KERNEL_OF(GoForward, embed_rows_out, ForwardArgs, 256);
KERNEL_OF(GoSums, embed_sums, BackwardArgs, 256);
KERNEL_OF(GoHotRows, embed_hot_rows, BackwardArgs, 256);
KERNEL_OF(GoWave, embed_wave, BackwardArgs, 256);
KERNEL_OF(GoFew, embed_few, BackwardArgs, 64 * FEW_WAVES);

int check(int64_t M, int64_t V, int64_t D, int64_t ld, int dtype) {
  if (dtype != GNET_F32 && dtype != GNET_BF16 && dtype != GNET_F16) return GNET_ERR_INVALID;
  if (M < 0 || V < 1 || D < 1 || ld < D) return GNET_ERR_INVALID;
  if (M > (1 << 24) || V > (1ll << 30) || D > (1 << 16) || M * D > (1ll << 38) || V * D > (1ll << 38)) return GNET_ERR_UNSUPPORTED;
  return GNET_OK;
}
size_t keys_bytes(int64_t M) { return ((size_t)M * 8 + 255) & ~(size_t)255; }

}  // namespace

extern "C" int gnet_embed_forward(const void* ids, int32_t ids64, const void* table, int64_t ld_table, float scale, const float* token_scale,
                                  int64_t M, int64_t V, int64_t D, int32_t dtype, void* y, gnet_stream_t stream) {
  clear_hip_error();
  if (const int e = check(M, V, D, ld_table, dtype)) return e;
  if (M == 0) return GNET_OK;
  if (!ids || !table || !y) return GNET_ERR_INVALID;
  ForwardArgs a{ids, ids64, M, V, D, table, ld_table, scale, token_scale, y, 1};
  const int vec = pick_vec(dtype, D);
  a.blocks = (int)((D + 64 * vec - 1) / (64 * vec));
  launch<GoForward>(dtype, vec, a, grid_of((M * a.blocks + 3) / 4), (hipStream_t)stream);
  return launch_status();
}

extern "C" size_t gnet_embed_workspace_bytes(int64_t M, int64_t D) {
  if (M <= WAVE || D <= 0 || M > (1 << 24) || D > (1 << 16)) return 0;
  return 2 * keys_bytes(M) + (size_t)((M + HOT - 1) / HOT) * 2 * ((D + 7) & ~7ll) * 4;
}

extern "C" int gnet_embed_backward(const void* ids, int32_t ids64, const void* dy, int64_t ld_dy, float scale, const float* token_scale,
                                   int64_t M, int64_t V, int64_t D, int32_t dtype, void* dtable, int32_t accumulate, const void* table,
                                   int64_t ld_table, float* dscale, void* workspace, size_t workspace_bytes, gnet_stream_t stream) {
  clear_hip_error();
  if (const int e = check(M, V, D, ld_dy, dtype)) return e;
  if (!dtable || (M && (!ids || !dy)) || (dscale && M && (!table || ld_table < D))) return GNET_ERR_INVALID;
  if (M > WAVE && (!workspace || workspace_bytes < gnet_embed_workspace_bytes(M, D) || ((uintptr_t)workspace & 255))) return GNET_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  u64* keys = (u64*)workspace;
  u64* other = (u64*)((char*)workspace + keys_bytes(M));
  float* part = (float*)((char*)workspace + 2 * keys_bytes(M));
  BackwardArgs a{keys, M, V, D, dy, ld_dy, scale, token_scale, dtable, D, accumulate, part, (D + 7) & ~7ll, 0, 0, 0, 0, ids, ids64, table, ld_table, dscale};
  const int vec = pick_vec(dtype, D);
  const unsigned column_blocks = (unsigned)((D + 64 * vec - 1) / (64 * vec));
  if (M && few(M, V, column_blocks)) {
    a.scale_groups = dscale ? (unsigned)((M + FEW_WAVES - 1) / FEW_WAVES) : 0;
    launch<GoFew>(dtype, vec, a, dim3(a.scale_groups + (unsigned)V, column_blocks), s);
    return launch_status();
  }
  a.fill_groups = accumulate ? 0 : (unsigned)((V + FILL_ROWS - 1) / FILL_ROWS);
  if (M && M <= WAVE) {
    a.run_groups = (unsigned)((M * column_blocks + 3) / 4);
    a.scale_groups = dscale ? (unsigned)((M + 3) / 4) : 0;
    launch<GoWave>(dtype, vec, a, grid_of((int64_t)a.run_groups + a.scale_groups + a.fill_groups), s);
    return launch_status();
  }
  if (M) {
    int n = 256;                                      // a whole wave
    while (n < RUN && n < M) n <<= 1;
    const unsigned runs = (unsigned)((M + RUN - 1) / RUN);
    if (V < (1 << 20) - 1) embed_sort<unsigned><<<runs, n / 4, 0, s>>>(ids, ids64, M, V, n, keys);
    else embed_sort<u64><<<runs, n / 4, 0, s>>>(ids, ids64, M, V, n, keys);
    if (const int e = launch_status()) return e;      // (nothing runs on keys that are not there)
    for (int64_t run = RUN; run < M; run *= WAY) {
      embed_merge<<<(unsigned)((M + 256 / WAY - 1) / (256 / WAY)), 256, 0, s>>>(keys, other, M, run);
      if (const int e = launch_status()) return e;
      u64* t = keys; keys = other; other = t;
    }
  }
  a.keys = keys;
  const unsigned segments = (unsigned)((M + HOT - 1) / HOT);
  a.hot_groups = M > HOT ? segments : 0;
  a.run_groups = (unsigned)((M + 3) / 4);
  a.scale_groups = dscale ? a.run_groups : 0;
  const int64_t groups = (int64_t)a.hot_groups + a.run_groups + a.scale_groups + a.fill_groups;
  if (groups) launch<GoSums>(dtype, vec, a, grid_of(groups), s);
  if (const int e = launch_status()) return e;
  if (M > HOT) launch<GoHotRows>(dtype, vec, a, dim3(segments, column_blocks), s);
  return launch_status();
}
