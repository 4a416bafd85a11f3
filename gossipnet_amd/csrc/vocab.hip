// Softmax losses over a large vocabulary, straight from the features: the logits z = x . W^T / temperature are never laid out.
//   cross entropy   loss = lse(z) - z[label]                               (gnet_xent_*)
//   distillation    loss = sum_k q_k (log q_k - z[id_k] + lse(z)),  q = softmax(teacher's logits / temperature)   (gnet_distill_*)
// Cross entropy is distillation with one target of weight 1, so both run the same kernels:
//   forward    vocab_targets  which tokens count, the targets' weights      vocab_pack   the tokens that count, moved together
//              vocab_gemm<EPI_PART>  maximum and sum of 2^z per vocabulary tile         vocab_join   lse, the targets' logits, loss
//   backward   the first two, then for one piece of the vocabulary after the other
//              vocab_gemm<EPI_DZ>  dz = g softmax(z) from recomputed logits       vocab_hits   dz at the targets, from fp32
//              vocab_gemm<EPI_SLAB>  dx += dz . W (fp32)     vocab_gemm<EPI_OUT>  dW = dz^T . x     and at last vocab_finish  dx
// A token whose targets are all outside [0, V) is left out of everything, whatever its row of x holds: it is not read again after
// vocab_targets, its dx is zero.
#include "vocab_gemm.hpp"

namespace {

constexpr int TILE = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ int64_t load_id(const void* p, int64_t i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
template <int DT> __device__ __forceinline__ float load_elem(const void* p, int64_t i) {
  if (DT == GNET_F32) return ((const float*)p)[i];
  if (DT == GNET_BF16) return Bf16T::dec(((const u16*)p)[i]);
  return F16T::dec(((const u16*)p)[i]);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
// the power of two that brings a magnitude into [2^top, 2^(top+1)); 1 for 0, infinities and NaN
__device__ __forceinline__ int scale_exponent(float a, int top) {
  if (!(a > 0.f) || !(a < INFINITY)) return 0;
  return max(-126, min(126, top - ilogbf(a)));
}

struct Targets {
  const void* ids; int ids64;          // [M,K]
  const float* logits;                 // [M,K] teacher's logits, or NULL (one target of weight 1)
  int64_t M; int K; int64_t V;
  float to_log2;                       // log2(e) / temperature
  float inv_temp;
};
__device__ __forceinline__ bool target_counts(const Targets& t, int64_t i, int64_t& id) {
  id = load_id(t.ids, i, t.ids64);
  return id >= 0 && id < t.V && !(t.logits && t.logits[i] == -INFINITY);
}

// One wave per token (and per padding byte of the flags): does it count; its targets' weights; in the backward pass weights of
// equal ids added up in each of their slots.  Two passes over K logits, K <= 1024: latency.
struct TargetsArgs {
  Targets t;
  int64_t flags_n;                     // M rounded up to 16
  uint8_t* flag; float* q; float* q_sum; float* entropy;       // q_sum: backward pass; entropy: forward pass
  const void* x; int64_t ldx, D; float* row_x;   // 32-bit x: the row's largest magnitude
  const float* dloss; float* row_g;              // backward only
};
__global__ void __launch_bounds__(256) vocab_targets(const TargetsArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.flags_n) return;
  bool counts = false;
  if (m < a.t.M) {
    const int K = a.t.K;
    float top = -INFINITY;
    bool any = false;
    for (int k = lane; k < K; k += 64) {
      int64_t id;
      if (target_counts(a.t, m * K + k, id)) { any = true; if (a.t.logits) top = fmaxf(top, a.t.logits[m * K + k]); }
    }
    counts = __any(any);
    top = wave_max(top);
    float sum = 0.f;
    for (int k = lane; k < K; k += 64) {
      int64_t id;
      float e = 0.f;
      if (target_counts(a.t, m * K + k, id)) e = a.t.logits ? exp2f((a.t.logits[m * K + k] - top) * a.t.to_log2) : 1.f;
      a.q[m * K + k] = e;
      sum += e;
    }
    sum = wave_sum(sum);
    float ent = 0.f;
    for (int k = lane; k < K; k += 64) {
      const float e = a.q[m * K + k], q = counts ? e / sum : 0.f;
      a.q[m * K + k] = q;
      if (a.t.logits && q > 0.f) ent += q * ((a.t.logits[m * K + k] - top) * a.t.inv_temp - logf(sum));
    }
    if (a.entropy) { ent = wave_sum(ent); if (lane == 0) a.entropy[m] = ent; }
    if (a.dloss && a.t.logits) {
      // the same id twice in a row: each of its slots stands for the sum (read back what the wave itself wrote)
      __threadfence_block();
      for (int kb = 0; kb < K; kb += 64) {
        const int k = kb + lane;
        int64_t id = -1;
        const bool c = k < K && target_counts(a.t, m * K + k, id);
        float s = 0.f;
        for (int j = 0; j < K; ++j)
          if (c && load_id(a.t.ids, m * K + j, a.t.ids64) == id) s += a.q[m * K + j];
        if (k < K) a.q_sum[m * K + k] = s;             // (an array of its own: later slots still read the single weights)
      }
    }
    if (a.row_x) {
      float mx = 0.f;
      if (counts) for (int64_t d = lane; d < a.D; d += 64) mx = fmaxf(mx, fabsf(((const float*)a.x)[m * a.ldx + d]));
      mx = wave_max(mx);
      if (lane == 0) a.row_x[m] = mx;
    }
    if (a.row_g && lane == 0) a.row_g[m] = counts ? fabsf(a.dloss[m] * a.t.inv_temp) : 0.f;
  }
  if (lane == 0) a.flag[m] = counts;
}

// largest magnitude of a 32-bit matrix, one partial result per workgroup
__global__ void __launch_bounds__(256) vocab_absmax(const float* __restrict__ w, int64_t ld, int64_t rows, int64_t D, float* __restrict__ part) {
  __shared__ float red[4];
  float mx = 0.f;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int64_t d = threadIdx.x; d < D; d += 256) mx = fmaxf(mx, fabsf(w[r * ld + d]));
  mx = wave_max(mx);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

__device__ __forceinline__ int block_sum(int v, int* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

template <int DT> __device__ __forceinline__ void pack_row(const void* src, int64_t first, int64_t D, u16* dst, int64_t Dp, int64_t plane, float scale, int lane) {
  for (int64_t d = lane; d < Dp; d += 64) {
    if (DT == GNET_F32) {
      u16 hi = 0, lo = 0;
      if (d < D) split_f16(((const float*)src)[first + d] * scale, hi, lo);
      dst[d] = hi; dst[plane + d] = lo;
    } else {
      dst[d] = d < D ? ((const u16*)src)[first + d] : (u16)0;
    }
  }
}

// The tokens that count moved together, in order, rows padded to a multiple of 64 elements, zero rows behind them up to Mp.
// Every workgroup counts the flags in front of its own rows: M bytes out of L2 instead of a scan in a launch of its own.
constexpr int PACK_ROWS = 16;
struct PackArgs {
  const uint8_t* flag; int64_t flags_n, M, Mp;
  const void* x; int64_t ldx, D, Dp; u16* xp; int64_t plane;
  const float* row_x; const float* w_part; int w_parts;
  const float* row_g; const float* dloss; const float* lse; float inv_temp; int top_g;
  int32_t* pos; float* lse2; float* gscale;
  VocabMeta* meta;
};
template <int DT> __global__ void __launch_bounds__(256) vocab_pack(const PackArgs a) {
  __shared__ int ired[4];
  __shared__ float fred[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * PACK_ROWS;
  int before = 0, all = 0;
  for (int64_t i = (int64_t)threadIdx.x * 4; i < a.flags_n; i += 1024) {
    const int n = __popc(*reinterpret_cast<const unsigned*>(a.flag + i));      // flags are 0 or 1
    all += n;
    if (i < r0) before += n;                                                   // r0 is a multiple of 16
  }
  before = block_sum(before, ired);
  all = block_sum(all, ired);
  float mx = 0.f, mw = 0.f, mg = 0.f;
  if (DT == GNET_F32) {
    for (int64_t i = threadIdx.x; i < a.M; i += 256) mx = fmaxf(mx, a.row_x[i]);
    for (int i = threadIdx.x; i < a.w_parts; i += 256) mw = fmaxf(mw, a.w_part[i]);
    mx = block_max(mx, fred);
    mw = block_max(mw, fred);
  }
  if (a.row_g) {
    for (int64_t i = threadIdx.x; i < a.M; i += 256) mg = fmaxf(mg, a.row_g[i]);
    mg = block_max(mg, fred);
  }
  const int ex = DT == GNET_F32 ? scale_exponent(mx, 13) : 0, eg = a.row_g ? scale_exponent(mg, a.top_g) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.meta->rows = all;
    a.meta->unscale_x = ldexpf(1.f, -ex);
    a.meta->unscale_w = DT == GNET_F32 ? ldexpf(1.f, -scale_exponent(mw, 13)) : 1.f;
    a.meta->unscale_g = ldexpf(1.f, -eg);
  }
  const float sx = ldexpf(1.f, ex);
  for (int j = wave; j < PACK_ROWS; j += 4) {
    const int64_t r = r0 + j;
    if (r >= a.Mp) continue;
    int f = 0;                                    // flags of this workgroup's rows in front of r; r's own
    bool own = false;
    for (int i = 0; i <= j; ++i) { const bool b = r0 + i < a.M && a.flag[r0 + i]; if (i < j) f += b; else own = b; }
    const int64_t rank = before + f;              // tokens that count in front of r
    if (r < a.M && lane == 0) a.pos[r] = own ? (int32_t)rank : -1;
    const int64_t to = own ? rank : all + (r - rank);        // the others' places behind them are zeroed
    u16* dst = a.xp + to * a.Dp;
    if (own) pack_row<DT>(a.x, r * a.ldx, a.D, dst, a.Dp, a.plane, sx, lane);
    else pack_row<DT>(a.x, 0, 0, dst, a.Dp, a.plane, sx, lane);
    if (own && a.row_g && lane == 0) {
      a.lse2[to] = a.lse[r] * LOG2E;
      a.gscale[to] = ldexpf(a.dloss[r] * a.inv_temp, eg);
    }
  }
}

// Rows of W that the matrix products cannot read where they lie (32 bits; widths that are no multiple of 64; alignment).
template <int DT> __global__ void __launch_bounds__(256) vocab_pack_w(const void* w, int64_t ldw, int64_t rows, int64_t D, u16* dst, int64_t Dp, int64_t plane, const VocabMeta* meta) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const float s = DT == GNET_F32 ? 1.f / meta->unscale_w : 1.f;
  pack_row<DT>(w, r * ldw, r < rows ? D : 0, dst + r * Dp, Dp, plane, s, threadIdx.x & 63);
}

// One workgroup per token: lse from the vocabulary tiles' sums, the targets' logits as fp32 dot products, the loss.
struct JoinArgs {
  Targets t;
  const int32_t* pos; const float2* part; int tiles;
  const void* x; int64_t ldx; const void* w; int64_t ldw; int64_t D;
  const float* q; const float* entropy;
  float* loss; float* lse; float* hit;
};
template <int DT> __global__ void __launch_bounds__(256) vocab_join(const JoinArgs a) {
  __shared__ float red[4], red2[4];
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = a.t.K;
  const int p = a.pos[m];
  if (p < 0) {
    for (int k = threadIdx.x; k < K; k += 256) a.hit[m * K + k] = 0.f;
    if (threadIdx.x == 0) { a.loss[m] = 0.f; a.lse[m] = 0.f; }
    return;
  }
  const float2* part = a.part + (int64_t)p * a.tiles;
  float mx = -INFINITY, sum = 0.f;
  for (int i = threadIdx.x; i < a.tiles; i += 256) {
    const float2 v = part[i];
    const float n = fmaxf(mx, v.x), b = n == -INFINITY ? 0.f : n;
    sum = sum * exp2f(mx - b) + v.y * exp2f(v.x - b);
    mx = n;
  }
  const float top = wave_max(mx);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  const float all = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), base = all == -INFINITY ? 0.f : all;
  sum = wave_sum(sum * exp2f(mx - base));
  if (lane == 0) red2[wave] = sum;
  __syncthreads();
  sum = (red2[0] + red2[1]) + (red2[2] + red2[3]);
  const float lse = (base + log2f(sum)) * LN2;
  float loss = 0.f;
  for (int k = wave; k < K; k += 4) {
    int64_t id;
    const bool c = target_counts(a.t, m * K + k, id);
    float dot = 0.f;
    if (c) {
      for (int64_t d = lane; d < a.D; d += 64) dot = fmaf(load_elem<DT>(a.x, m * a.ldx + d), load_elem<DT>(a.w, id * a.ldw + d), dot);
      dot = wave_sum(dot) * a.t.inv_temp;
      const float q = a.q[m * K + k];
      if (q != 0.f) loss += q * (lse - dot);       // (an infinite logit of a target without weight stays out)
    }
    if (lane == 0) a.hit[m * K + k] = dot;
  }
  __syncthreads();
  if (lane == 0) red[wave] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    loss = (red[0] + red[1]) + (red[2] + red[3]) + (a.t.logits ? a.entropy[m] : 0.f);
    // cross entropy is >= 0: what is below comes from rounding (NaN stays).  Distillation with an id in two slots may be below 0.
    a.loss[m] = !a.t.logits && loss < 0.f ? 0.f : loss;
    a.lse[m] = lse;
  }
}

// dz at the targets of one piece of the vocabulary: (softmax - weight) g from the forward pass's fp32 logits, over what
// vocab_gemm<EPI_DZ> stored there.  Slots with the same id store the same value.
struct HitsArgs {
  Targets t;
  const int32_t* pos; const float* lse; const float* hit; const float* q; const float* gscale;
  u16* dz; int64_t ld_dz, plane; int64_t v0, v1;
};
template <class T, int PLANES> __global__ void __launch_bounds__(256) vocab_hits(const HitsArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.t.M * a.t.K) return;
  const int64_t m = i / a.t.K;
  int64_t id;
  if (!target_counts(a.t, i, id) || id < a.v0 || id >= a.v1) return;
  const int p = a.pos[m];
  const float d = (exp2f((a.hit[i] - a.lse[m]) * LOG2E) - a.q[i]) * a.gscale[p];
  u16* to = a.dz + p * a.ld_dz + (id - a.v0);
  if (PLANES == 1) *to = T::enc(d);
  else { u16 hi, lo; split_f16(d, hi, lo); to[0] = hi; to[a.plane] = lo; }
}

// out[r][:] = unscale * sum over the splits' partial sums (ascending), zero for a row whose place is -1
struct FinishArgs {
  const float* slab; int64_t ld, stride; int splits;
  const int32_t* pos;                                // NULL: row r of the slab
  int64_t rows, D; void* out; int64_t ld_out;
  const VocabMeta* meta; int by_x;
};
template <int DT> __global__ void __launch_bounds__(256) vocab_finish(const FinishArgs a) {
  const float f = a.meta->unscale_g * (a.by_x ? a.meta->unscale_x : a.meta->unscale_w);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / a.D, d = i % a.D;
  if (r >= a.rows) return;
  const int64_t p = a.pos ? a.pos[r] : r;
  float v = 0.f;
  if (p >= 0) {
    for (int s = 0; s < a.splits; ++s) v += a.slab[s * a.stride + p * a.ld + d];
    v *= f;
  }
  if (DT == GNET_F32) ((float*)a.out)[r * a.ld_out + d] = v;
  else if (DT == GNET_BF16) ((u16*)a.out)[r * a.ld_out + d] = Bf16T::enc(v);
  else ((u16*)a.out)[r * a.ld_out + d] = F16T::enc(v);
}

// ---- the plan: sizes, pieces and where everything lies in the workspace ------------------------------------------------
inline int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Plan {
  int64_t Mp, Dp, flags_n, piece, pieces, w_tiles;
  int planes, pack_w, dx_splits, dw_splits;
  int64_t flag, q, entropy, row_x, row_g, w_part, meta, pos, lse2, gscale, xp, wp, part, dz, dx_slab, dw_slab, bytes;
};
constexpr int W_PARTS = 512;

// One pass over the chip is 256 workgroups: a product with fewer tiles splits its contraction, down to eight steps a split.
int pick_splits(int64_t tiles, int64_t steps) {
  int s = 1;
  while (tiles * s < 256 && steps / (2 * s) >= 8 && s < 64) s *= 2;
  return s;
}

Plan make_plan(int64_t M, int64_t V, int64_t D, int64_t K, int dtype, int pack_w, int backward) {
  Plan p = {};
  p.planes = dtype == GNET_F32 ? 2 : 1;
  p.pack_w = pack_w;
  p.Mp = up(M, TILE); p.Dp = up(D, 64); p.flags_n = up(M, 16);
  // A piece's dz and packed rows of W stay within the last-level cache (256 MB) for the products that read them again.
  const int64_t per_row = (int64_t)p.planes * 2 * ((backward ? p.Mp : 0) + (pack_w ? p.Dp : 0));
  const int64_t Vp = up(V, TILE);
  int64_t piece = per_row ? (128ll << 20) / per_row / TILE * TILE : Vp;
  if (piece < 8 * TILE) piece = 8 * TILE;
  p.pieces = (Vp + piece - 1) / piece;
  p.piece = up((Vp + p.pieces - 1) / p.pieces, TILE);
  p.pieces = (Vp + p.piece - 1) / p.piece;
  p.w_tiles = Vp / TILE;
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o = up(o + bytes, 256); return at; };
  p.flag = take(p.flags_n);
  p.q = take(M * K * 4 * 2);
  p.meta = take(sizeof(VocabMeta));
  p.pos = take(M * 4);
  p.xp = take(p.planes * p.Mp * p.Dp * 2);
  if (p.planes == 2) { p.row_x = take(M * 4); p.w_part = take(W_PARTS * 4); }
  if (pack_w) p.wp = take(p.planes * p.piece * p.Dp * 2);
  if (!backward) {
    p.entropy = take(M * 4);
    p.part = take(p.Mp * p.w_tiles * 8);
  } else {
    p.row_g = take(M * 4); p.lse2 = take(p.Mp * 4); p.gscale = take(p.Mp * 4);
    p.dz = take(p.planes * p.Mp * p.piece * 2);
    p.dx_splits = pick_splits(up(p.Dp, TILE) / TILE * (p.Mp / TILE), p.piece / VG_BK);
    p.dx_slab = take((int64_t)p.dx_splits * p.Mp * p.Dp * 4);
    p.dw_splits = pick_splits(up(p.Dp, TILE) / TILE * (p.piece / TILE), p.Mp / VG_BK);
    if (p.dw_splits > 1) p.dw_slab = take((int64_t)p.dw_splits * p.piece * p.Dp * 4);
  }
  p.bytes = o;
  return p;
}

int needs_pack(const void* w, int64_t ldw, int64_t D, int dtype) {
  return dtype == GNET_F32 || (D & 63) || (ldw & 7) || ldw > (1 << 22) || ((uintptr_t)w & 15);      // (2^22: 32-bit offsets in a tile)
}

struct Problem {
  const void* x; int64_t ldx; const void* w; int64_t ldw; Targets t; int64_t D; int dtype;
};

int check(const Problem& q) {
  if (q.dtype != GNET_F32 && q.dtype != GNET_BF16 && q.dtype != GNET_F16) return GNET_ERR_INVALID;
  if (q.t.M < 0 || q.t.V < 1 || q.D < 1 || q.t.K < 1 || q.ldx < q.D || q.ldw < q.D) return GNET_ERR_INVALID;
  if (q.t.M > (1 << 24) || q.t.V > (1ll << 30) || q.t.M * q.t.V > (1ll << 44) || q.D > (1 << 16) || q.t.K > 1024) return GNET_ERR_UNSUPPORTED;
  if (!(q.t.inv_temp > 0.f) || !(q.t.inv_temp < INFINITY)) return GNET_ERR_INVALID;
  if (!q.w || (q.t.M && (!q.x || !q.t.ids))) return GNET_ERR_INVALID;
  return GNET_OK;
}

template <int DT, class T, int PLANES> struct Run {
  template <bool AS, bool BS, int EPI> static void gemm(const VocabGemm& g, hipStream_t s) {
    vocab_gemm<T, TILE, TILE, 2, 4, AS, BS, EPI, PLANES><<<(unsigned)((int64_t)g.row_tiles * g.col_tiles * g.splits), 512, 0, s>>>(g);
  }

  // targets, packing: everything in front of the first matrix product
  static void prepare(const Problem& q, const Plan& p, char* ws, const float* dloss, const float* lse, hipStream_t s) {
    TargetsArgs a = {};
    a.t = q.t; a.flags_n = p.flags_n;
    a.flag = (uint8_t*)(ws + p.flag); a.q = (float*)(ws + p.q); a.q_sum = a.q + q.t.M * q.t.K; a.entropy = dloss ? nullptr : (float*)(ws + p.entropy);
    a.x = q.x; a.ldx = q.ldx; a.D = q.D;
    a.row_x = PLANES == 2 ? (float*)(ws + p.row_x) : nullptr;
    a.dloss = dloss; a.row_g = dloss ? (float*)(ws + p.row_g) : nullptr;
    vocab_targets<<<(unsigned)((p.flags_n + 3) / 4), 256, 0, s>>>(a);
    if (PLANES == 2) vocab_absmax<<<W_PARTS, 256, 0, s>>>((const float*)q.w, q.ldw, q.t.V, q.D, (float*)(ws + p.w_part));
    PackArgs k = {};
    k.flag = a.flag; k.flags_n = p.flags_n; k.M = q.t.M; k.Mp = p.Mp;
    k.x = q.x; k.ldx = q.ldx; k.D = q.D; k.Dp = p.Dp; k.xp = (u16*)(ws + p.xp); k.plane = p.Mp * p.Dp;
    k.row_x = a.row_x; k.w_part = PLANES == 2 ? (float*)(ws + p.w_part) : nullptr; k.w_parts = W_PARTS;
    k.row_g = a.row_g; k.dloss = dloss; k.lse = lse; k.inv_temp = q.t.inv_temp; k.top_g = DT == GNET_BF16 ? 0 : 14;
    k.pos = (int32_t*)(ws + p.pos); k.lse2 = (float*)(ws + p.lse2); k.gscale = (float*)(ws + p.gscale);
    k.meta = (VocabMeta*)(ws + p.meta);
    vocab_pack<DT><<<(unsigned)((p.Mp + PACK_ROWS - 1) / PACK_ROWS), 256, 0, s>>>(k);
  }

  // W rows v0 .. of one piece as an operand (packed first where needed)
  static VocabOperand piece_of_w(const Problem& q, const Plan& p, char* ws, int64_t v0, hipStream_t s) {
    VocabOperand o = {};
    if (p.pack_w) {
      const int64_t rows = q.t.V - v0 < p.piece ? q.t.V - v0 : p.piece;
      const char* from = (const char*)q.w + v0 * q.ldw * (DT == GNET_F32 ? 4 : 2);
      vocab_pack_w<DT><<<(unsigned)(p.piece / 4), 256, 0, s>>>(from, q.ldw, rows, q.D, (u16*)(ws + p.wp), p.Dp, p.piece * p.Dp, (const VocabMeta*)(ws + p.meta));
      o.p = (const u16*)(ws + p.wp); o.ld = p.Dp; o.plane = p.piece * p.Dp; o.rows = p.piece;
    } else {
      o.p = (const u16*)q.w + v0 * q.ldw; o.ld = q.ldw; o.plane = 0; o.rows = q.t.V - v0;
    }
    o.cols = (int)p.Dp;
    return o;
  }
  static VocabOperand packed_x(const Plan& p, char* ws) {
    VocabOperand o = {};
    o.p = (const u16*)(ws + p.xp); o.ld = p.Dp; o.plane = p.Mp * p.Dp; o.rows = p.Mp; o.cols = (int)p.Dp;
    return o;
  }
  static VocabGemm logits(const Problem& q, const Plan& p, char* ws, const VocabOperand& w, int64_t v0) {
    VocabGemm g = {};
    g.a = w; g.b = packed_x(p, ws);
    g.k = p.Dp; g.cols_from_meta = 1; g.segments = PLANES == 2 ? 3 : 1;
    const int64_t rows = up(q.t.V - v0 < p.piece ? q.t.V - v0 : p.piece, TILE);
    g.row_tiles = (int)(rows / TILE); g.col_tiles = (int)(p.Mp / TILE); g.splits = 1;
    g.meta = (const VocabMeta*)(ws + p.meta);
    g.to_log2 = q.t.to_log2; g.valid_rows = q.t.V - v0;
    g.first_row_tile = (int)(v0 / TILE); g.all_row_tiles = (int)p.w_tiles;
    return g;
  }

  static int forward(const Problem& q, const Plan& p, char* ws, float* loss, float* lse, float* hit, hipStream_t s) {
    prepare(q, p, ws, nullptr, nullptr, s);
    for (int64_t v0 = 0; v0 < q.t.V; v0 += p.piece) {
      VocabGemm g = logits(q, p, ws, piece_of_w(q, p, ws, v0, s), v0);
      g.part = (float2*)(ws + p.part);
      gemm<false, false, EPI_PART>(g, s);
    }
    JoinArgs j = {};
    j.t = q.t; j.pos = (const int32_t*)(ws + p.pos); j.part = (const float2*)(ws + p.part); j.tiles = (int)p.w_tiles;
    j.x = q.x; j.ldx = q.ldx; j.w = q.w; j.ldw = q.ldw; j.D = q.D;
    j.q = (const float*)(ws + p.q); j.entropy = (const float*)(ws + p.entropy);
    j.loss = loss; j.lse = lse; j.hit = hit;
    vocab_join<DT><<<(unsigned)q.t.M, 256, 0, s>>>(j);
    return launch_status();
  }

  static int backward(const Problem& q, const Plan& p, char* ws, const float* lse, const float* hit, const float* dloss, void* dx, void* dw, hipStream_t s) {
    prepare(q, p, ws, dloss, lse, s);
    const VocabMeta* meta = (const VocabMeta*)(ws + p.meta);
    const int elem = DT == GNET_F32 ? 4 : 2;
    for (int64_t v0 = 0; v0 < q.t.V; v0 += p.piece) {
      const int64_t rows = q.t.V - v0 < p.piece ? q.t.V - v0 : p.piece, rows64 = up(rows, VG_BK);
      const VocabOperand w = piece_of_w(q, p, ws, v0, s);
      VocabGemm g = logits(q, p, ws, w, v0);
      g.lse2 = (const float*)(ws + p.lse2); g.gscale = (const float*)(ws + p.gscale);
      g.dz = (u16*)(ws + p.dz); g.ld_dz = p.piece; g.plane_dz = p.Mp * p.piece;
      gemm<false, false, EPI_DZ>(g, s);
      HitsArgs h = {};
      h.t = q.t; h.pos = (const int32_t*)(ws + p.pos); h.lse = lse; h.hit = hit;
      h.q = (const float*)(ws + p.q) + (q.t.logits ? q.t.M * q.t.K : 0);
      h.gscale = g.gscale; h.dz = g.dz; h.ld_dz = g.ld_dz; h.plane = g.plane_dz; h.v0 = v0; h.v1 = v0 + rows;
      vocab_hits<T, PLANES><<<(unsigned)((q.t.M * q.t.K + 255) / 256), 256, 0, s>>>(h);
      VocabOperand dz = {};
      dz.p = g.dz; dz.ld = p.piece; dz.plane = g.plane_dz; dz.rows = p.Mp; dz.cols = (int)p.piece;
      if (dx) {
        VocabGemm d = {};
        d.a = w; d.b = dz; d.k = rows64; d.cols_from_meta = 1; d.segments = g.segments;
        d.row_tiles = (int)(up(p.Dp, TILE) / TILE); d.col_tiles = (int)(p.Mp / TILE); d.splits = p.dx_splits; d.meta = meta;
        d.slab = (float*)(ws + p.dx_slab); d.ld_slab = p.Dp; d.slab_stride = p.Mp * p.Dp; d.accumulate = v0 > 0; d.out_cols = p.Mp;
        gemm<true, false, EPI_SLAB>(d, s);
      }
      if (dw) {
        VocabGemm d = {};
        d.a = packed_x(p, ws); d.b = dz; d.k_from_meta = 1; d.segments = g.segments;
        d.row_tiles = (int)(up(p.Dp, TILE) / TILE); d.col_tiles = (int)(up(rows, TILE) / TILE); d.splits = p.dw_splits; d.meta = meta;
        d.out_cols = rows;
        void* out = (char*)dw + v0 * q.D * elem;
        if (p.dw_splits == 1) {
          d.out = out; d.ld_out = q.D; d.out_rows = q.D; d.unscale_by_x = 1;
          d.out_vec = (q.D & 3) == 0 && ((uintptr_t)dw & 7) == 0;
          gemm<true, true, EPI_OUT>(d, s);
        } else {
          d.slab = (float*)(ws + p.dw_slab); d.ld_slab = p.Dp; d.slab_stride = p.piece * p.Dp;
          gemm<true, true, EPI_SLAB>(d, s);
          FinishArgs f = {};
          f.slab = d.slab; f.ld = p.Dp; f.stride = d.slab_stride; f.splits = d.splits;
          f.rows = rows; f.D = q.D; f.out = out; f.ld_out = q.D; f.meta = meta; f.by_x = 1;
          vocab_finish<DT><<<(unsigned)((rows * q.D + 255) / 256), 256, 0, s>>>(f);
        }
      }
    }
    if (dx) {
      FinishArgs f = {};
      f.slab = (const float*)(ws + p.dx_slab); f.ld = p.Dp; f.stride = p.Mp * p.Dp; f.splits = p.dx_splits;
      f.pos = (const int32_t*)(ws + p.pos); f.rows = q.t.M; f.D = q.D; f.out = dx; f.ld_out = q.D; f.meta = meta;
      vocab_finish<DT><<<(unsigned)((q.t.M * q.D + 255) / 256), 256, 0, s>>>(f);
    }
    return launch_status();
  }
};

__global__ void __launch_bounds__(256) vocab_zero(unsigned* p, int64_t words, u16* tail) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) p[i] = 0;
  if (tail && blockIdx.x == 0 && threadIdx.x == 0) *tail = 0;
}

int run_forward(const Problem& q, float* loss, float* lse, float* hit, void* ws, size_t ws_bytes, hipStream_t s) {
  clear_hip_error();
  if (const int e = check(q)) return e;
  if (q.t.M == 0) return GNET_OK;
  if (!loss || !lse || !hit) return GNET_ERR_INVALID;
  const Plan p = make_plan(q.t.M, q.t.V, q.D, q.t.K, q.dtype, needs_pack(q.w, q.ldw, q.D, q.dtype), 0);
  if (!ws || ws_bytes < (size_t)p.bytes || ((uintptr_t)ws & 255)) return GNET_ERR_WORKSPACE;
  switch (q.dtype) {
    case GNET_F32: return Run<GNET_F32, F16T, 2>::forward(q, p, (char*)ws, loss, lse, hit, s);
    case GNET_BF16: return Run<GNET_BF16, Bf16T, 1>::forward(q, p, (char*)ws, loss, lse, hit, s);
    default: return Run<GNET_F16, F16T, 1>::forward(q, p, (char*)ws, loss, lse, hit, s);
  }
}

int run_backward(const Problem& q, const float* lse, const float* hit, const float* dloss, void* dx, void* dw, void* ws, size_t ws_bytes, hipStream_t s) {
  clear_hip_error();
  if (const int e = check(q)) return e;
  if (q.t.M == 0) {
    if (dw) {
      const int64_t bytes = q.t.V * q.D * (q.dtype == GNET_F32 ? 4 : 2);
      vocab_zero<<<1024, 256, 0, s>>>((unsigned*)dw, bytes / 4, bytes & 2 ? (u16*)((char*)dw + bytes - 2) : nullptr);
    }
    return launch_status();
  }
  if (!lse || !hit || !dloss) return GNET_ERR_INVALID;
  const Plan p = make_plan(q.t.M, q.t.V, q.D, q.t.K, q.dtype, needs_pack(q.w, q.ldw, q.D, q.dtype), 1);
  if (!ws || ws_bytes < (size_t)p.bytes || ((uintptr_t)ws & 255)) return GNET_ERR_WORKSPACE;
  switch (q.dtype) {
    case GNET_F32: return Run<GNET_F32, F16T, 2>::backward(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
    case GNET_BF16: return Run<GNET_BF16, Bf16T, 1>::backward(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
    default: return Run<GNET_F16, F16T, 1>::backward(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
  }
}

Problem problem(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* ids, int ids64, const float* logits, float temperature,
                int64_t M, int64_t V, int64_t D, int64_t K, int dtype) {
  Problem q;
  q.x = x; q.ldx = ldx; q.w = w; q.ldw = ldw; q.D = D; q.dtype = dtype;
  q.t.ids = ids; q.t.ids64 = ids64; q.t.logits = logits; q.t.M = M; q.t.K = (int)(K > 1 << 20 ? 1 << 20 : K); q.t.V = V;
  q.t.inv_temp = 1.f / temperature; q.t.to_log2 = LOG2E / temperature;
  return q;
}

}  // namespace

// ------------------------------------------------------------------------------------------
extern "C" size_t gnet_vocab_workspace_bytes(const void* w, int64_t ldw, int64_t M, int64_t V, int64_t D, int64_t K, int32_t dtype, int32_t backward) {
  if (M <= 0 || V < 1 || D < 1 || K < 1 || M > (1 << 24) || V > (1ll << 30) || D > (1 << 16) || K > 1024) return 0;
  return (size_t)make_plan(M, V, D, K, dtype, needs_pack(w, ldw, D, dtype), backward).bytes;
}

extern "C" int gnet_xent_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* labels, int32_t labels64, int64_t M,
                                 int64_t V, int64_t D, int32_t dtype, float* loss, float* lse, float* hit, void* workspace,
                                 size_t workspace_bytes, gnet_stream_t stream) {
  return run_forward(problem(x, ldx, w, ldw, labels, labels64, nullptr, 1.f, M, V, D, 1, dtype), loss, lse, hit, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int gnet_xent_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* labels, int32_t labels64,
                                  const float* lse, const float* hit, const float* dloss, int64_t M, int64_t V, int64_t D, int32_t dtype,
                                  void* dx, void* dw, void* workspace, size_t workspace_bytes, gnet_stream_t stream) {
  return run_backward(problem(x, ldx, w, ldw, labels, labels64, nullptr, 1.f, M, V, D, 1, dtype), lse, hit, dloss, dx, dw, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int gnet_distill_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* top_ids, int32_t ids64,
                                    const float* top_logits, float temperature, int64_t M, int64_t V, int64_t D, int64_t K, int32_t dtype,
                                    float* loss, float* lse, float* hit, void* workspace, size_t workspace_bytes, gnet_stream_t stream) {
  if (!top_logits && M > 0) return GNET_ERR_INVALID;
  return run_forward(problem(x, ldx, w, ldw, top_ids, ids64, top_logits, temperature, M, V, D, K, dtype), loss, lse, hit, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int gnet_distill_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* top_ids, int32_t ids64,
                                     const float* top_logits, float temperature, const float* lse, const float* hit, const float* dloss,
                                     int64_t M, int64_t V, int64_t D, int64_t K, int32_t dtype, void* dx, void* dw, void* workspace,
                                     size_t workspace_bytes, gnet_stream_t stream) {
  if (!top_logits && M > 0) return GNET_ERR_INVALID;
  return run_backward(problem(x, ldx, w, ldw, top_ids, ids64, top_logits, temperature, M, V, D, K, dtype), lse, hit, dloss, dx, dw, workspace, workspace_bytes, (hipStream_t)stream);
}
