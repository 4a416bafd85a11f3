// Softmax losses over a large vocabulary, straight from the features: the logits z = x . W^T / temperature are never laid out.
//   cross entropy   loss = lse(z) - z[label]                               (gnet_xent_*)
//   distillation    loss = sum_k q_k (log q_k - z[id_k] + lse(z)),  q = softmax(teacher's logits / temperature)   (gnet_distill_*)
// Cross entropy is distillation with one target of weight 1, so both run the same kernels:
//   forward    vocab_targets  which tokens count, the teacher's weights      vocab_pack   the tokens that count, moved together;
//              the logits at the teacher's ids
//              vocab_gemm<EPI_PART>  maximum and sum of 2^z per vocabulary tile, the label's logit
//              vocab_join   lse, loss
//   backward   the first two, then for one piece of the vocabulary after the other
//              vocab_gemm<EPI_DZ>  dz = g (softmax(z) - label) from recomputed logits       vocab_hits   dz at the teacher's ids
//              vocab_gemm<EPI_SLAB>  dx += dz . W (fp32)     vocab_gemm<EPI_OUT>  dW = dz^T . x     and at last vocab_finish  dx
// A token whose targets are all outside [0, V) is left out of everything, whatever its row of x holds, and its dx is zero.
// A small vocabulary takes other kernels (vocab_small.hpp), and so do few tokens on a W that would have to be laid out (vocab_few.hpp) or on little of it; few
// tiles of logits take another softmax (logits_splits).
#include "vocab_gemm.hpp"
#include <algorithm>

namespace {

__device__ __forceinline__ int64_t load_id(const void* p, int64_t i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
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
__device__ __forceinline__ int wave_isum(int v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
// |v|, or 0 for what is not finite: an infinity in one token's values must not set the scale of all others'
__device__ __forceinline__ float finite_abs(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.f; }
// the exponent of the power of two that brings a magnitude into [2^top, 2^(top+1)); 0 for 0, infinities and NaN
__device__ __forceinline__ int scale_exponent(float a, int top) {
  if (!(a > 0.f) || !(a < INFINITY)) return 0;
  return max(-126, min(126, top - ilogbf(a)));
}

struct Targets {
  const void* ids; int ids64;          // [M,K]
  const float* logits;                 // [M,K] teacher's logits, or NULL (one target of weight 1: K = 1)
  int64_t M; int K; int64_t V;
  float to_log2;                       // log2(e) / temperature
  float inv_temp;
};
__device__ __forceinline__ bool target_counts(const Targets& t, int64_t i, int64_t& id) {
  id = load_id(t.ids, i, t.ids64);
  return id >= 0 && id < t.V && !(t.logits && t.logits[i] == -INFINITY);
}

#include "vocab_small.hpp"
#include "vocab_few.hpp"

// ---- what is known before the first product ------------------------------------------------------------------------
// Token workgroups, one wave per token (and per padding byte of the flags): does it count; its targets' weights; in the backward pass
// the weights of equal ids added up in each of their slots.  Two passes over K <= 1024 logits: latency.
// The remaining W_PARTS workgroups, 32-bit operands only: the largest magnitude of W, one partial result each.
constexpr int W_PARTS = 1024;
struct TargetsArgs {
  Targets t;
  int64_t flags_n;                     // M rounded up to 16
  unsigned token_groups;
  uint8_t* flag; float* q; float* q_sum; float* entropy;       // q, entropy: distillation; q_sum: its backward pass
  const float* x; int64_t ldx, D; float* row_x;                // 32-bit x: the row's largest magnitude
  const float* dloss; float* row_g;                            // backward only
  const float* w; int64_t ldw; float* w_part;
};
// the largest finite magnitude of a thread's share of n consecutive values
__device__ __forceinline__ float magnitude(const float* p, int64_t n, int64_t t, int64_t threads) {
  float mx = 0.f;
#pragma unroll 4
  for (int64_t i = t; i < n / 4; i += threads) {
    const f32x4 v = *reinterpret_cast<const f32x4u*>(p + i * 4);
    mx = fmaxf(mx, fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3]))));
  }
  for (int64_t i = n / 4 * 4 + t; i < n; i += threads) mx = fmaxf(mx, finite_abs(p[i]));
  return mx;
}
__global__ void __launch_bounds__(256) vocab_targets(const TargetsArgs a) {
  const int lane = threadIdx.x & 63;
  if (blockIdx.x >= a.token_groups) {
    __shared__ float red[4];
    const unsigned part = blockIdx.x - a.token_groups;
    float mx = 0.f;
    if (a.ldw == a.D) mx = magnitude(a.w, a.t.V * a.D, (int64_t)part * 256 + threadIdx.x, W_PARTS * 256ll);
    else for (int64_t r = part; r < a.t.V; r += W_PARTS) mx = fmaxf(mx, magnitude(a.w + r * a.ldw, a.D, threadIdx.x, 256));
    mx = block_max(mx, red);
    if (threadIdx.x == 0) a.w_part[part] = mx;
    return;
  }
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.flags_n) return;
  bool counts = false;
  if (m < a.t.M) {
    const int K = a.t.K;
    if (!a.t.logits) {
      int64_t id;
      counts = target_counts(a.t, m, id);
    } else {
      float top = -INFINITY;
      bool any = false;
      for (int k = lane; k < K; k += 64) {
        int64_t id;
        if (target_counts(a.t, m * K + k, id)) { any = true; top = fmaxf(top, a.t.logits[m * K + k]); }
      }
      counts = __any(any);
      top = wave_max(top);
      float sum = 0.f;
      for (int k = lane; k < K; k += 64) {
        int64_t id;
        const float e = target_counts(a.t, m * K + k, id) ? exp2f((a.t.logits[m * K + k] - top) * a.t.to_log2) : 0.f;
        a.q[m * K + k] = e;
        sum += e;
      }
      sum = wave_sum(sum);
      float ent = 0.f;
      for (int k = lane; k < K; k += 64) {
        const float e = a.q[m * K + k], q = counts ? e / sum : 0.f;
        a.q[m * K + k] = q;
        if (q != 0.f) ent += q * ((a.t.logits[m * K + k] - top) * a.t.inv_temp - logf(sum));
      }
      if (a.entropy) { ent = wave_sum(ent); if (lane == 0) a.entropy[m] = ent; }
      if (a.dloss) {
        __threadfence_block();                             // the wave reads back what its other lanes wrote
        auto slot = [&](int k, int& id32, float& q) {      // (an id that counts is below 2^30)
          int64_t id = -1;
          const bool c = k < K && target_counts(a.t, m * K + k, id);
          id32 = c ? (int)id : -1;
          q = c ? a.q[m * K + k] : 0.f;
        };
        for (int kb = 0; kb < K; kb += 64) {
          int id, other;
          float q, s = 0.f;
          slot(kb + lane, id, q);
          for (int jb = 0; jb < K; jb += 64) {
            slot(jb + lane, other, q);
            for (int l = 0; l < min(64, K - jb); ++l)
              if (__builtin_amdgcn_readlane(other, l) == id) s += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q), l));
          }
          if (kb + lane < K) a.q_sum[m * K + kb + lane] = s;       // (an array of its own: later slots still read the single weights)
        }
      }
    }
    if (a.row_x) {
      float mx = 0.f;
      if (counts) mx = magnitude(a.x + m * a.ldx, a.D, lane, 64);
      mx = wave_max(mx);
      if (lane == 0) a.row_x[m] = mx;
    }
    if (a.row_g && lane == 0) a.row_g[m] = counts ? finite_abs(a.dloss[m] * a.t.inv_temp) : 0.f;
  }
  if (lane == 0) a.flag[m] = counts;
}

// Rows copied to the matrix products' layout: Dp elements (a multiple of 64), zeros behind D; 32 bits as two fp16 planes, if asked for (dst2)
// twice, the second time at a scale of its own.
struct RowCopy { int64_t D, Dp, plane; float scale; };
template <int DT> __device__ __forceinline__ void copy_row(const void* src, int64_t first, bool zero, u16* dst, const RowCopy& c, int t, int threads, u16* dst2 = nullptr, float scale2 = 0.f) {
  for (int64_t d = (int64_t)t * 8; d < c.Dp; d += (int64_t)threads * 8) {
    s16x8 hi = {0, 0, 0, 0, 0, 0, 0, 0}, lo = hi, hi2 = hi, lo2 = hi;
    if (!zero) {
      if (DT == GNET_F32) {
        const float* p = (const float*)src + first + d;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (d + 8 <= c.D) {
          const f32x4 v0 = *reinterpret_cast<const f32x4u*>(p), v1 = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = i < 4 ? v0[i & 3] : v1[i & 3];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) if (d + i < c.D) v[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          u16 h, l;
          split_f16(v[i] * c.scale, h, l);
          hi[i] = (short)h; lo[i] = (short)l;
        }
        if (dst2)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u16 h, l;
            split_f16(v[i] * scale2, h, l);
            hi2[i] = (short)h; lo2[i] = (short)l;
          }
      } else {
        const u16* p = (const u16*)src + first + d;
        if (d + 8 <= c.D) hi = *reinterpret_cast<const s16x8u*>(p);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) if (d + i < c.D) hi[i] = (short)p[i];
      }
    }
    *reinterpret_cast<s16x8*>(dst + d) = hi;
    if (DT == GNET_F32) *reinterpret_cast<s16x8*>(dst + c.plane + d) = lo;
    if (DT == GNET_F32 && dst2) {
      *reinterpret_cast<s16x8*>(dst2 + d) = hi2;
      *reinterpret_cast<s16x8*>(dst2 + c.plane + d) = lo2;
    }
  }
}
template <int DT> __device__ __forceinline__ void zero_row(void* out, int64_t first, int64_t D, int t, int threads) {
  for (int64_t d = t; d < D; d += threads) {
    if (DT == GNET_F32) ((float*)out)[first + d] = 0.f;
    else ((u16*)out)[first + d] = 0;
  }
}
// Rows of W that the matrix products cannot read where they lie (32 bits; widths that are no multiple of 8; alignment).
struct PackW { const void* w; int64_t ldw, rows, rows_out; u16* dst; int each; RowCopy c; };      // each: rows of a workgroup, a multiple of 4
template <int DT> __device__ __forceinline__ void pack_w_rows(const PackW& a, int64_t group, float scale) {
  RowCopy c = a.c;
  c.scale = scale;
  for (int64_t r = group * a.each + (threadIdx.x >> 6); r < min(a.rows_out, (group + 1) * a.each); r += 4)
    copy_row<DT>(a.w, r * a.ldw, r >= a.rows, a.dst + r * c.Dp, c, threadIdx.x & 63, 64);
}
template <int DT> __global__ void __launch_bounds__(256) vocab_pack_w(const PackW a, const VocabMeta* meta) {
  pack_w_rows<DT>(a, blockIdx.x, DT == GNET_F32 ? 1.f / meta->unscale_w : 1.f);
}

// The student's logits at the teacher's ids, distillation's forward pass: fp32 dot products, four slots of a token a wave.
template <int DT> __device__ __forceinline__ void dot8(const s16x8 (&x)[DT == GNET_F32 ? 2 : 1], const void* w, float& s) {
  if constexpr (DT == GNET_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 a = __builtin_bit_cast(f32x4, x[h]), b = ((const f32x4u*)w)[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) s = fmaf(a[i], b[i], s);
    }
  } else {
    const s16x8 b = *(const s16x8u*)w;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      s = DT == GNET_BF16 ? fmaf(Bf16T::dec((u16)x[0][i]), Bf16T::dec((u16)b[i]), s) : fmaf(F16T::dec((u16)x[0][i]), F16T::dec((u16)b[i]), s);
  }
}
template <int DT> __device__ __forceinline__ float load_elem(const void* p, int64_t i) {
  if (DT == GNET_F32) return ((const float*)p)[i];
  if (DT == GNET_BF16) return Bf16T::dec(((const u16*)p)[i]);
  return F16T::dec(((const u16*)p)[i]);
}
struct DotArgs { const void* x; int64_t ldx; const void* w; int64_t ldw, D; float* hit; int per_token; };      // per_token: waves
template <int DT> __device__ __forceinline__ void target_dots(const Targets& t, const DotArgs& a, int64_t unit) {
  constexpr int SIZE = DT == GNET_F32 ? 4 : 2, U = 4;
  const int64_t m = unit / a.per_token;
  if (m >= t.M) return;
  const int lane = threadIdx.x & 63, k0 = (int)(unit - m * a.per_token) * U;
  const char* x = (const char*)a.x + m * a.ldx * SIZE;
  const char* w[U];
  bool c[U];
  float dot[U];
  bool some = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int64_t id = 0;
    c[u] = k0 + u < t.K && target_counts(t, m * t.K + k0 + u, id);
    w[u] = (const char*)a.w + (c[u] ? id : 0) * a.ldw * SIZE;
    dot[u] = 0.f;
    some |= c[u];
  }
  if (some) {                                        // (a token that does not count: its x is not read)
#pragma unroll 2
    for (int64_t d = (int64_t)lane * 8; d + 8 <= a.D; d += 512) {
      s16x8 xv[DT == GNET_F32 ? 2 : 1];
#pragma unroll
      for (int h = 0; h < (DT == GNET_F32 ? 2 : 1); ++h) xv[h] = ((const s16x8u*)(x + d * SIZE))[h];
#pragma unroll
      for (int u = 0; u < U; ++u) dot8<DT>(xv, w[u] + d * SIZE, dot[u]);
    }
    const int64_t d = (a.D & ~7ll) + lane;           // what is left of eight
    if (d < a.D) {
      const float v = load_elem<DT>(x, d);
#pragma unroll
      for (int u = 0; u < U; ++u) dot[u] = fmaf(v, load_elem<DT>(w[u], d), dot[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float z = wave_sum(dot[u]) * t.inv_temp;
    if (lane == 0 && k0 + u < t.K) a.hit[m * t.K + k0 + u] = c[u] ? z : 0.f;
  }
}

// Token workgroups: the tokens that count moved together, in order, zero rows behind them up to Mp.  Every workgroup counts the tokens
// in front of its own rows: M bytes (or labels) out of L2 instead of a scan in a launch of its own.
// Then workgroups that pack the first piece of W, and those of the targets' logits.
struct PackArgs {
  Targets t;
  const uint8_t* flag;                 // NULL: cross entropy's labels are looked at directly
  int64_t flags_n, Mp; int rows;       // rows of a workgroup, a multiple of 4
  unsigned token_groups;
  const void* x; int64_t ldx; u16* xp; RowCopy c;
  const float* row_x; const float* w_part;
  const float* row_g; const float* dloss; const float* loss; const float* lse; int top_exp;       // dz is stored in units of the largest |dloss| / 2^top_exp
  int32_t* pos; int32_t* label; int32_t* row_of; float* lse_c; float* gscale; float* label_p;      // label_p: with loss
  u16* xg; int32_t* exp_c;             // two planes, backward: x as dW's operand, and the tokens' own exponents
  void* dx;                            // its rows of tokens that do not count are zeroed here; NULL: later
  VocabMeta* meta;
  PackW w; unsigned w_groups;
  DotArgs dots;
};
template <int DT, bool BACKWARD> __global__ void __launch_bounds__(256) vocab_pack(const PackArgs a) {
  __shared__ int ired[2][4];
  __shared__ float fred[3][4];
  __shared__ int place[256], own_exp[DT == GNET_F32 && BACKWARD ? 256 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t group = group_id();
  if (group >= a.token_groups + a.w_groups) {
    if (!BACKWARD && a.dots.hit) target_dots<DT>(a.t, a.dots, (group - a.token_groups - a.w_groups) * 4 + (threadIdx.x >> 6));
    return;
  }
  const bool packs_w = group >= a.token_groups;
  const int64_t r0 = group * a.rows, M = a.t.M;
  auto counts = [&](int64_t i) { int64_t id; return a.flag ? a.flag[i] != 0 : target_counts(a.t, i, id); };
  // all that is looked through first, then one exchange between the waves
  int before = 0, all = 0;
  float mw = 0.f, mg = 0.f, mx = 0.f;
  if (DT == GNET_F32)
    for (int i = threadIdx.x; i < W_PARTS; i += 256) mw = fmaxf(mw, a.w_part[i]);
  if (!packs_w) {
    if (a.flag) {
#pragma unroll 4
      for (int64_t i = (int64_t)threadIdx.x * 4; i < a.flags_n; i += 1024) {
        const int n = __popc(*reinterpret_cast<const unsigned*>(a.flag + i));      // flags are 0 or 1
        all += n;
        if (i < r0) before += n;                                                   // r0 is a multiple of 4
      }
      if (BACKWARD)
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < M; i += 256) mg = fmaxf(mg, a.row_g[i]);
      if (DT == GNET_F32)
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < M; i += 256) mx = fmaxf(mx, a.row_x[i]);
    } else {
#pragma unroll 4
      for (int64_t i = threadIdx.x; i < M; i += 256) {
        const bool c = counts(i);
        all += c;
        if (i < r0) before += c;
        if (BACKWARD && c) mg = fmaxf(mg, finite_abs(a.dloss[i] * a.t.inv_temp));
      }
    }
  }
  before = wave_isum(before);
  all = wave_isum(all);
  if (DT == GNET_F32) { mw = wave_max(mw); mx = wave_max(mx); }
  if (BACKWARD) mg = wave_max(mg);
  if (lane == 0) { ired[0][wave] = before; ired[1][wave] = all; fred[0][wave] = mw; fred[1][wave] = mx; fred[2][wave] = mg; }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < 4; ++w) { before += ired[0][w]; all += ired[1][w]; mw = fmaxf(mw, fred[0][w]); mx = fmaxf(mx, fred[1][w]); mg = fmaxf(mg, fred[2][w]); }
  const int ew = DT == GNET_F32 ? scale_exponent(mw, 13) : 0;
  if (packs_w) { pack_w_rows<DT>(a.w, group - a.token_groups, ldexpf(1.f, ew)); return; }
  const int ex = DT == GNET_F32 ? scale_exponent(mx, 13) : 0;
  // dz is stored in units of the largest |dloss|, not of a power of two: with one dloss for all tokens what is rounded to 16 bits is
  // softmax - target itself, and the -1 of a label and the rest of its row are not off by different shares (fp16: 2^15 times that)
  const float unit_g = mg >= 1.17549435e-38f && mg < INFINITY ? mg : 1.f;
  if (group == 0 && threadIdx.x == 0) {
    a.meta->rows = all;
    a.meta->unscale_x = ldexpf(1.f, -ex);
    a.meta->unscale_w = ldexpf(1.f, -ew);
    a.meta->unit_g = unit_g;
    a.meta->exp_g = -a.top_exp;
  }
  RowCopy c = a.c;
  c.scale = ldexpf(1.f, ex);
  const int wide = c.Dp >= 2048;                  // a whole workgroup a row, or a wave
  const int t = wide ? threadIdx.x : lane;
  // 256 rows of the group at a time: place[] = how many that count are in front of a row, or ~ of it for a row that does not
  for (int j0 = 0; j0 < a.rows; j0 += 256) {
    const int64_t base = r0 + j0, mine = base + threadIdx.x;
    const bool c256 = threadIdx.x < a.rows - j0 && mine < M && counts(mine);
    const unsigned long long mask = __ballot(c256);
    __syncthreads();
    if (lane == 0) ired[0][wave] = __popcll(mask);
    __syncthreads();
    int rank = before + __popcll(mask & ((1ull << lane) - 1));
    for (int w = 0; w < wave; ++w) rank += ired[0][w];
    place[threadIdx.x] = c256 ? rank : ~rank;
    if (mine < M && threadIdx.x < a.rows - j0) a.pos[mine] = c256 ? rank : -1;
    // Two fp16 end at 2^-40 of the unit: a token whose |dloss| is far below the largest has its dz in a unit 2^e smaller, taken back from
    // dx's sums and, for dW, from its row of x.  (16-bit operands: one unit for all; x times a power of two would leave fp16's range.)
    int e = 0;
    if (c256) {
      if (a.label) a.label[rank] = (int32_t)load_id(a.t.ids, mine, a.t.ids64);
      if (BACKWARD && a.row_of) a.row_of[rank] = (int32_t)mine;
      if (BACKWARD) {
        const float gs = a.dloss[mine] * a.t.inv_temp / unit_g;
        if (DT == GNET_F32 && gs != 0.f && fabsf(gs) < INFINITY) e = min(max(-1 - ilogbf(gs), 0), 100);      // (below 2^15, as the largest is: fp16 ends at 65504)
        a.lse_c[rank] = a.lse[mine];
        if (a.loss) a.label_p[rank] = expm1f(-a.loss[mine]);
        a.gscale[rank] = ldexpf(gs, a.top_exp + e);
        if (DT == GNET_F32) a.exp_c[rank] = e;
      }
    }
    if (DT == GNET_F32 && BACKWARD) own_exp[threadIdx.x] = e;
    before += ired[0][0] + ired[0][1] + ired[0][2] + ired[0][3];
    __syncthreads();
    const int n = (int)min((int64_t)min(256, a.rows - j0), a.Mp - base);
    for (int j = wide ? 0 : wave; j < n; j += wide ? 1 : 4) {
      const int64_t r = base + j;
      const int at = place[j];
      const bool own = at >= 0;
      const int64_t to = own ? at : all + (r - ~at);           // the others' places behind them are zeroed
      copy_row<DT>(a.x, r * a.ldx, !own, a.xp + to * c.Dp, c, t, wide ? 256 : 64, DT == GNET_F32 && BACKWARD ? a.xg + to * c.Dp : nullptr,
                   DT == GNET_F32 && BACKWARD ? ldexpf(1.f, ex - own_exp[j]) : 0.f);
      if (BACKWARD && a.dx && !own && r < M) zero_row<DT>(a.dx, r * c.D, c.D, t, wide ? 256 : 64);
    }
  }
}

// ---- behind the products ---------------------------------------------------------------------------------------------
struct JoinArgs {
  Targets t;
  const int32_t* pos; const float2* part; int tiles; const float* hit_c;     // hit_c: cross entropy's label logits, compacted
  const float* q; const float* entropy;
  float* loss; float* lse; float* hit;                                       // hit: distillation's comes from vocab_pack
};
// a token's largest logit and the log of the sum over the vocabulary of exp(z - largest), from its tiles', by one wave
__device__ __forceinline__ void join_tiles(const float2* part, int tiles, int lane, float& top, float& log_sum) {
  float mx = -INFINITY, sum = 0.f;
#pragma unroll 8
  for (int i = lane; i < tiles; i += 64) mx = fmaxf(mx, part[i].x);
  mx = wave_max(mx);
  top = mx == -INFINITY ? 0.f : mx;
#pragma unroll 8
  for (int i = lane; i < tiles; i += 64) sum += part[i].y * exp2f((part[i].x - top) * LOG2E);
  log_sum = logf(wave_sum(sum));
}
// one wave per token
__global__ void __launch_bounds__(256) vocab_join(const JoinArgs a) {
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.t.M) return;
  const int p = a.pos[m], lane = threadIdx.x & 63, K = a.t.K;
  float top = 0.f, log_sum = 0.f, loss = 0.f;
  if (p >= 0) join_tiles(a.part + (int64_t)p * a.tiles, a.tiles, lane, top, log_sum);
  const float lse = top + log_sum;
  if (!a.t.logits) {
    const float hit = p >= 0 ? a.hit_c[p] : 0.f;
    loss = (top - hit) + log_sum;                  // both from the same products: where the label takes nearly everything nothing cancels
    if (loss < 0.f) loss = 0.f;                    // (below 0 from rounding only; NaN stays)
    if (lane == 0) a.hit[m] = hit;
  } else if (p >= 0) {
    for (int k = lane; k < K; k += 64) {
      const float q = a.q[m * K + k];
      if (q != 0.f) loss += q * (lse - a.hit[m * K + k]);      // (an infinite logit of a target without weight stays out)
    }
    loss = wave_sum(loss) + a.entropy[m];
  }
  if (lane == 0) { a.loss[m] = loss; a.lse[m] = lse; }
}

// Few tiles and a long contraction: the logits' product is split along its contraction, and what fits into 64 MB of partial sums goes
// on by rows, a workgroup a token: its logits are the splits' sums, and the whole row's maximum and sum are at hand in both directions.
// forward: loss, lse, hit in place of the tiles' sums and vocab_join;  backward: dz, normalised by the row itself.
struct RowsArgs {
  Targets t;
  const float* slab; int64_t ld, stride; int splits;
  const VocabMeta* meta;
  const int32_t* pos; const float* q; const float* entropy; float* loss; float* lse; float* hit;       // forward
  const int32_t* label; const float* gscale; const float* label_p; u16* dz; int64_t ld_dz, plane;      // backward
};
template <class T, int PLANES, bool BACKWARD> __global__ void __launch_bounds__(256) vocab_rows(const RowsArgs a) {
  __shared__ float red[4];
  const int64_t m = blockIdx.x;                        // forward: token; backward: place
  const int rows = a.meta->rows, K = a.t.K;
  const int p = BACKWARD ? (m < rows ? (int)m : -1) : a.pos[m];
  if (p < 0) {
    if (BACKWARD) {
      for (int64_t v = threadIdx.x * 4; v < a.ld; v += 1024)
#pragma unroll
        for (int i = 0; i < PLANES; ++i) *reinterpret_cast<s16x4*>(a.dz + i * a.plane + m * a.ld_dz + v) = s16x4{0, 0, 0, 0};
    } else {
      if (!a.t.logits && threadIdx.x == 0) a.hit[m] = 0.f;
      if (threadIdx.x == 0) { a.loss[m] = 0.f; a.lse[m] = 0.f; }
    }
    return;
  }
  const float f = logit_scale(*a.meta, a.t.inv_temp);
  auto sums = [&](int64_t v) {                         // of rows v .. v + 3
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) z += *reinterpret_cast<const f32x4*>(a.slab + s * a.stride + p * a.ld + v);
    return z;
  };
  auto logit = [&](int64_t v) {
    f32x4 z = sums(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = v + i < a.t.V ? z[i] * f : -INFINITY;
    return z;
  };
  const f32x4 own = threadIdx.x * 4 < a.t.V ? logit(threadIdx.x * 4) : f32x4{0.f, 0.f, 0.f, 0.f};      // the first of the thread's, kept
  float top = -INFINITY, sum = 0.f;
  for (int64_t v = threadIdx.x * 4; v < a.t.V; v += 1024) {
    const f32x4 z = v < 1024 ? own : logit(v);
    top = fmaxf(top, fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
  }
  top = block_max(top, red);
  if (top == -INFINITY) top = 0.f;
  for (int64_t v = threadIdx.x * 4; v < a.t.V; v += 1024) {
    const f32x4 z = v < 1024 ? own : logit(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += exp2f((z[i] - top) * LOG2E);
  }
  sum = block_sum(sum, red);
  if constexpr (BACKWARD) {
    const float over = 1.f / sum, gs = a.gscale[p];
    const int64_t label = a.label ? a.label[p] : -1;
    for (int64_t v = threadIdx.x * 4; v < a.ld; v += 1024) {
      u16 hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
      if (v < a.t.V) {
        const f32x4 z = v < 1024 ? own : logit(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float d = exp2f((z[i] - top) * LOG2E) * over;                      // (behind V: exp(-inf) = 0)
          if (v + i == label) d = a.label_p ? a.label_p[p] : d - 1.f;
          d *= gs;
          if (PLANES == 1) hi[i] = T::enc(v + i < a.t.V ? d : 0.f); else split_f16(v + i < a.t.V ? d : 0.f, hi[i], lo[i]);
        }
      }
      *reinterpret_cast<s16x4*>(a.dz + m * a.ld_dz + v) = s16x4{(short)hi[0], (short)hi[1], (short)hi[2], (short)hi[3]};
      if (PLANES == 2) *reinterpret_cast<s16x4*>(a.dz + a.plane + m * a.ld_dz + v) = s16x4{(short)lo[0], (short)lo[1], (short)lo[2], (short)lo[3]};
    }
  } else {
    const float log_sum = logf(sum), lse = top + log_sum;
    float loss = 0.f;
    if (!a.t.logits) {
      const int64_t label = load_id(a.t.ids, m, a.t.ids64);
      const float hit = one_logit(sums(label & ~3ll)[label & 3], *a.meta, a.t.inv_temp);
      loss = (top - hit) + log_sum;
      if (loss < 0.f) loss = 0.f;
      if (threadIdx.x == 0) a.hit[m] = hit;
    } else {
      for (int k = threadIdx.x; k < K; k += 256) {
        const float q = a.q[m * K + k];
        if (q != 0.f) loss += q * (lse - a.hit[m * K + k]);
      }
      loss = block_sum(loss, red) + a.entropy[m];
    }
    if (threadIdx.x == 0) { a.loss[m] = loss; a.lse[m] = lse; }
  }
}

// dz at the teacher's ids of one piece of the vocabulary: (softmax - weight) g from the forward pass's fp32 logits, over what
// vocab_gemm<EPI_DZ> stored there.  Slots with the same id store the same value.
struct HitsArgs {
  Targets t;
  const int32_t* pos; const float* lse; const float* hit; const float* q; const float* gscale;
  u16* dz; int64_t ld_dz, plane; int64_t v0, v1;
};
template <class T, int PLANES> __global__ void __launch_bounds__(256) vocab_hits(const HitsArgs a) {
  const int64_t i = group_id() * 256 + threadIdx.x;
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

// out[r][:] = unscale * sum over the splits' partial sums (ascending), zero for a row whose place is -1; four elements a thread
struct FinishArgs {
  const float* slab; int64_t ld, stride; int splits;
  const int32_t* pos;                                // NULL: row r of the slab
  int64_t rows, D; unsigned quads; void* out;                 // quads: groups of four a row
  const VocabMeta* meta; int by_x;
  const int32_t* exp_c;                              // dx of two planes: by place
  SplitFit fit; int64_t out_cols;                    // dx: how often the contraction was split (vocab_gemm)
};
template <int DT> __global__ void __launch_bounds__(64) vocab_finish(const FinishArgs a) {
  GradScale f = grad_scale(*a.meta, a.by_x);
  const int64_t i = group_id() * 64 + threadIdx.x;
  const int64_t r = i / a.quads, d = (i - r * a.quads) * 4;
  if (r >= a.rows) return;
  const int64_t p = a.pos ? a.pos[r] : r;
  int splits = a.splits;
  int64_t stride = a.stride;
  if (a.fit.slots) {
    const Splits n = fit_splits(a.fit, splits, (a.meta->rows + VG_BK - 1) & ~(VG_BK - 1), a.out_cols);
    splits = n.splits;
    stride = n.cols * a.ld;
  }
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (p >= 0) {
    if (DT == GNET_F32 && a.exp_c) f.exp -= a.exp_c[p];
#pragma unroll 8
    for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(a.slab + s * stride + p * a.ld + d);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = unscale(v[k], f);
  }
  const int64_t at = r * a.D + d;
  if (DT == GNET_F32) {
    float* o = (float*)a.out + at;
    if (d + 4 <= a.D) *reinterpret_cast<f32x4u*>(o) = v;
    else for (int k = 0; k < 4; ++k) if (d + k < a.D) o[k] = v[k];
  } else {
    u16* o = (u16*)a.out + at;
    s16x4 e;
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = (short)(DT == GNET_BF16 ? Bf16T::enc(v[k]) : F16T::enc(v[k]));
    if (d + 4 <= a.D) *reinterpret_cast<s16x4u*>(o) = e;
    else for (int k = 0; k < 4; ++k) if (d + k < a.D) o[k] = (u16)e[k];
  }
}

// ---- the plan: tiles, pieces and where everything lies in the workspace ------------------------------------------------
inline int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
inline int64_t tiles(int64_t v, int64_t a) { return (v + a - 1) / a; }

// Tile shapes of the products.  A contraction step of 64 takes 256 x 256 tiles 1.5 us (one workgroup a CU: 1.4 PFLOP/s) and 128 x 128
// tiles 0.9 us (two a CU: 1.2), and every tile 6 or 3.5 us before and behind its steps (fitted to 4096 x 131072 x 4096, 833 x 50257 x 1024 and
// 464 x 65537 x 1536).  A last round that fills half of the chip at most is worked on as half tiles (vocab_gemm.hpp).  128 x 64 and 128 x 32 are for products with that few tokens, which wait for W: they only have to keep
// loads in flight.
enum Shape { S256, S128, S64, S32 };
struct ShapeInfo { int bm, bn; };
constexpr ShapeInfo SHAPE[] = {{256, 256}, {128, 128}, {128, 64}, {128, 32}};
struct Product { int shape, splits; };

double product_us(int shape, int splits, int64_t rows, int64_t cols, int64_t steps, bool halves) {
  const int64_t n = tiles(rows, SHAPE[shape].bm) * tiles(cols, SHAPE[shape].bn) * splits;
  const double round = shape == S256 ? tiles(steps, splits) * 1.5 + 6 : tiles(steps, splits) * 0.9 + 3.5;
  const int64_t at_once = shape == S256 ? 256 : 512, rest = n % at_once;
  const double rounds = (double)(n / at_once) + (!rest ? 0. : halves && 2 * rest <= at_once ? 0.65 : 1.);
  const double joined = splits > 1 ? 5 + (double)rows * cols * 4 * (2 * splits) / 4e6 : 0;       // partial sums out and in at 4 TB/s
  return rounds * round + joined;
}
// few_cols: the columns are tokens, for which the narrow shapes exist
Product pick_product(int64_t rows, int64_t cols, int64_t steps, bool few_cols, bool may_split) {
  Product best = {few_cols && cols <= 32 ? S32 : few_cols && cols <= 64 ? S64 : S256, 1};
  if (best.shape == S256) {
    double least = 1e30;
    for (int shape = S256; shape <= S128; ++shape)
      for (int splits = 1; splits <= (may_split ? 16 : 1) && (splits == 1 || steps / splits >= 4); ++splits) {
        const double us = product_us(shape, splits, rows, cols, steps, shape == S256 || few_cols);
        if (us < least) { least = us; best.shape = shape; best.splits = splits; }
      }
  } else if (may_split) {
    const int64_t n = tiles(rows, SHAPE[best.shape].bm);
    while (best.splits < 64 && n * best.splits < 768 && steps / (best.splits + 1) >= 8) ++best.splits;      // three workgroups a CU
  }
  return best;
}

// Splits of the logits' contraction where the tiles leave more than half of the chip idle.  A tile alone on its CU takes 0.6 us a step of
// 64; the partial sums are then read twice by one workgroup a token, about 20 bytes a nanosecond.  The forward
// product and the kernel behind it, in one and split: 165 x 2283 x 2240 fp32 67 and 29 us, 40 x 1000 x 4096 fp16 39 and 15 us, 5 x 154 x 3088 bf16
// 30 and 14 us, 700 x 512 x 1024 bf16 19 and 15 us; 31 x 16278 x 1183 fp16 17 us in one, where the second kernel alone took 20 us.
int logits_splits(int shape, int64_t V, int64_t M, int64_t steps, int64_t slab_bytes) {
  const int64_t n = tiles(V, SHAPE[shape].bm) * tiles(M, SHAPE[shape].bn);
  int best = 1;
  double least = steps * 0.6;
  for (int s = 2; n * s <= 256 && steps / s >= 8 && slab_bytes * s <= 64ll << 20; ++s) {
    const double us = tiles(steps, s) * 0.6 + 4 + (double)V * s * 8 / 20e3 * (M > 1024 ? M / 1024. : 1.);
    if (us < least) { least = us; best = s; }
  }
  return best;
}

// Where the small vocabulary's kernels run (vocab_small.hpp).  A workgroup reads all of W and computes its tokens' logits on the fp32
// matrix pipe, at a sixteenth of the 16-bit rate and a fifth of two fp16 planes': past some V D and M V D the general path is faster.
// Forward and backward together, here and there: fp32 2000 x 81 x 128 26 and 68 us, 4096 x 256 x 256 69 and 88, 2000 x 256 x 512 (not
// taken) 105 and 84; bf16 2000 x 81 x 128 28 and 48, 4096 x 128 x 256 47 and 58, 2000 x 256 x 256 (not taken) 60 and 51; distillation with
// K = 32, 2000 x 81 x 128: fp32 30 and 85, bf16 32 and 67.
bool small(int64_t M, int64_t V, int64_t D, int64_t K, int dtype) {
  const int64_t most = dtype == GNET_F32 ? 1 << 16 : 1 << 15;
  return V <= 256 && K <= SMALL_K && M <= 8192 && V * D <= most && M * V * D <= 4096 * most;
}
size_t small_bytes(int64_t M, int64_t V) { return (size_t)up(M, 16) * (up(V, 16) + 1) * 4; }

// Whether a product's workgroups make one launch (half tiles add 16 or 32 to each XCD's)
bool launchable(const Product& p, int64_t rows, int64_t cols) {
  return (tiles(rows, SHAPE[p.shape].bm) * tiles(cols, SHAPE[p.shape].bn) * p.splits + 512) * (p.shape == S256 ? 512 : 256) < 1ll << 32;
}

struct Plan {
  int64_t Mp, Dp, flags_n, piece, pieces, w_tiles;
  int planes, pack_w, direct, dx_direct, launchable;
  Product logits, dx, dw;
  SplitFit dx_fit;
  int64_t flag, q, entropy, row_x, row_g, w_part, meta, pos, label, row_of, hit_c, lse_c, gscale, label_p, exp_c, xp, xg, wp, part, z_slab, dz, dx_slab, dw_slab, bytes;
};

Plan make_plan(int64_t M, int64_t V, int64_t D, int64_t K, int dtype, int distill, int pack_w, int backward) {
  Plan p = {};
  p.planes = dtype == GNET_F32 ? 2 : 1;
  const int segments = p.planes == 2 ? 3 : 1;
  p.pack_w = pack_w;
  // cross entropy on 16 bits needs nothing of its tokens but the labels: up to 8192 of them the packing looks at them itself
  p.direct = !distill && p.planes == 1 && M <= 8192;
  p.Mp = up(M, VG_BK); p.Dp = up(D, 64); p.flags_n = up(M, 16);
  // A piece's dz and packed rows of W take at most 256 MB: that is what the last-level cache holds for the products that read them
  // again, though larger pieces measured the same (2048 x 100352 x 2048: 2.25 ms; 64 MB 2.22, 512 MB 2.17; 4096 x 131072 x 4096: 9.85, 9.77, 9.79).
  // But 2048 rows at least, since every piece reads and writes dx's fp32 sums: past 65536 tokens in 16 bits (32768 in 32) dz takes 4 KB (8 KB)
  // a token.  A floor of 2 D rows: 131072 x 50304 x 256 17.1 and 19.1 ms, 524288 x 8192 x 128 8.5 and 25.2, 131072 x 16384 x 256 fp32 13.9 and 21.0.
  const int64_t per_row = (int64_t)p.planes * 2 * ((backward ? p.Mp : 0) + (pack_w ? p.Dp : 0));
  const int64_t Vp = up(V, 256);
  int64_t piece = per_row ? (256ll << 20) / per_row / 256 * 256 : Vp;
  if (piece < 2048) piece = 2048;
  // and at most 2^20 tiles of logits (2^29 threads): a launch has to have fewer than 2^32
  piece = std::min(piece, std::max<int64_t>((1 << 20) / tiles(M, 256), 1) * 256);
  p.pieces = tiles(Vp, piece);
  p.piece = up(tiles(Vp, p.pieces), 256);
  p.pieces = tiles(Vp, p.piece);
  p.logits = pick_product(V < p.piece ? V : p.piece, M, p.Dp / VG_BK * segments, true, false);
  if (V <= SHAPE[S128].bm && p.logits.shape == S256) p.logits.shape = S128;          // (a vocabulary of one tile: EPI_DZ_ONE)
  if (p.pieces == 1) p.logits.splits = logits_splits(p.logits.shape, V, M, p.Dp / VG_BK * segments, (int64_t)p.Mp * p.piece * 4);
  p.w_tiles = tiles(V, SHAPE[p.logits.shape].bm);
  p.launchable = launchable(p.logits, p.piece, M);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o = up(o + bytes, 256); return at; };
  p.meta = take(sizeof(VocabMeta));
  p.pos = take(M * 4);
  p.xp = take(p.planes * p.Mp * p.Dp * 2);
  if (!p.direct) p.flag = take(p.flags_n);
  if (distill) p.q = take(M * K * 4 * (backward ? 2 : 1)); else p.label = take(p.Mp * 4);
  if (p.planes == 2) { p.row_x = take(M * 4); p.w_part = take(W_PARTS * 4); }
  if (pack_w) p.wp = take(p.planes * p.piece * p.Dp * 2);
  if (p.logits.splits > 1) p.z_slab = take((int64_t)p.logits.splits * p.Mp * p.piece * 4);
  if (!backward) {
    p.entropy = take(M * 4);
    p.hit_c = take(p.Mp * 4);
    if (p.logits.splits == 1) p.part = take(p.Mp * p.w_tiles * 8);
  } else {
    p.row_g = take(M * 4); p.lse_c = take(p.Mp * 4); p.gscale = take(p.Mp * 4);
    if (!distill) p.label_p = take(p.Mp * 4);
    if (p.planes == 2) { p.exp_c = take(p.Mp * 4); p.xg = take(p.planes * p.Mp * p.Dp * 2); }
    p.dz = take(p.planes * p.Mp * p.piece * 2);
    p.dx = pick_product(p.Dp, M, p.piece / VG_BK * segments, true, true);
    p.dx_direct = p.pieces == 1 && p.dx.splits == 1;          // one sum: straight to its rows
    p.row_of = take(p.Mp * 4);
    if (!p.dx_direct) {
      int64_t rows = (int64_t)p.dx.splits * p.Mp;
      if (p.dx.shape <= S128) {
        const ShapeInfo t = SHAPE[p.dx.shape];
        const int64_t steps = p.piece / VG_BK * segments;
        p.dx_fit = SplitFit{p.dx.shape == S256 ? 256 : 512, (int)std::min<int64_t>(steps / 4, 4 * p.dx.splits), (int)tiles(p.Dp, t.bm), (int)tiles(M, t.bn), t.bn};
        rows = std::max(rows, (int64_t)(p.dx_fit.slots / p.dx_fit.row_tiles) * t.bn);
      }
      p.dx_slab = take(rows * p.Dp * 4);
    }
    p.dw = pick_product(p.Dp, p.piece, p.Mp / VG_BK * segments, false, true);
    p.launchable &= launchable(p.dx, p.Dp, M) & launchable(p.dw, p.Dp, p.piece);
    if (p.dw.splits > 1) p.dw_slab = take((int64_t)p.dw.splits * p.piece * p.Dp * 4);
  }
  p.bytes = o;
  return p;
}

// Few tokens and a W that would have to be laid out, or so little work that the general path is its launches (vocab_few.hpp).  bf16 weights
// that need no layout, both directions, here and there: 16 x 1000 x 128 22 and 33 us, 16 x 16000 x 128 34 and 37, 16 x 4000 x 512 34 and 38;
// 32 x 4000 x 512 (not taken) 43 and 39, 16 x 1000 x 4096 (not taken) 93 and 54.
// (The vocabulary has to be larger than one tile: in a small one the sums are formed again in the backward pass, where 1 - p needs them.)
struct FewPlan { int tokens; int64_t ld_z, dx_rows, splits, ld_slab, z, part, flag, q, entropy, slab, bytes; };
bool few_tokens(int64_t M, int64_t V, int64_t D, int64_t K, int dtype, int pack_w) {
  const bool little = D <= 1024 && up(M, 16) * V * D <= 1 << 25;
  return (pack_w || little) && M <= FEW_TOKENS && V > SHAPE[S128].bm && up(M, 16) * up(V, 64) * 4 <= FEW_LOGITS && !small(M, V, D, K, dtype);
}
FewPlan few_plan(int64_t M, int64_t V, int64_t D, int64_t K, bool distill, int backward) {
  FewPlan p = {};
  p.tokens = M <= 16 ? 16 : 32;
  p.ld_z = up(V, 64); p.ld_slab = up(D, 64);
  const int64_t blocks = p.ld_slab / 64;
  // workgroups for the whole chip, four a CU; their partial sums stay below 16 MB
  p.dx_rows = up(tiles(V, blocks < 1024 ? 1024 / blocks : 1), 64); p.splits = tiles(V, p.dx_rows);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o = up(o + bytes, 256); return at; };
  p.z = take(p.tokens * p.ld_z * 4);
  if (distill) { p.flag = take(up(M, 16)); p.q = take(M * K * 4 * (backward ? 2 : 1)); }
  if (backward) p.slab = take(p.splits * p.tokens * p.ld_slab * 4);
  else { p.part = take(M * (p.ld_z / FEW_ROWS) * 8); p.entropy = take(M * 4); }
  p.bytes = o;
  return p;
}

int needs_pack(const void* w, int64_t ldw, int64_t D, int dtype) {
  return dtype == GNET_F32 || (D & 7) || (ldw & 7) || ldw > (1 << 22) || ((uintptr_t)w & 15);      // (2^22: 32-bit offsets in a tile)
}
struct Problem {
  const void* x; int64_t ldx; const void* w; int64_t ldw; Targets t; int64_t D; int dtype;
  const float* loss;                                 // cross entropy's backward pass: the forward's, or NULL
};

int check(const Problem& q) {
  if (q.dtype != GNET_F32 && q.dtype != GNET_BF16 && q.dtype != GNET_F16) return GNET_ERR_INVALID;
  if (q.t.M < 0 || q.t.V < 1 || q.D < 1 || q.t.K < 1 || q.ldx < q.D || q.ldw < q.D) return GNET_ERR_INVALID;
  if (q.t.M > (1 << 24) || q.t.V > (1ll << 30) || q.t.M * q.t.V > (1ll << 44) || q.D > (1 << 16) || q.t.K > 1024) return GNET_ERR_UNSUPPORTED;
  if (q.t.M * q.D > (1ll << 38) || q.t.V * q.D > (1ll << 38)) return GNET_ERR_UNSUPPORTED;
  if (!(q.t.inv_temp > 0.f) || !(q.t.inv_temp < INFINITY)) return GNET_ERR_INVALID;
  if (!q.w || (q.t.M && (!q.x || !q.t.ids))) return GNET_ERR_INVALID;
  return GNET_OK;
}

// ---- a small vocabulary ------------------------------------------------------------------------------------------------
template <int DT> struct Small {
  static SmallArgs args(const Problem& q) {
    SmallArgs a = {};
    a.t = q.t; a.x = q.x; a.ldx = q.ldx; a.w = q.w; a.ldw = q.ldw; a.D = q.D;
    a.ld_z = (int)up(q.t.V, 64) + 4;
    return a;
  }
  static int forward(const Problem& q, float* loss, float* lse, float* hit, hipStream_t s) {
    SmallArgs a = args(q);
    a.loss = loss; a.lse = lse; a.hit = hit;
    vocab_small<DT, false><<<(unsigned)tiles(q.t.M, SMALL_TOKENS), 64 * SMALL_WAVES, SMALL_TOKENS * a.ld_z * 4, s>>>(a);
    return launch_status();
  }
  static int backward(const Problem& q, char* ws, const float* dloss, void* dx, void* dw, hipStream_t s) {
    SmallArgs a = args(q);
    a.dloss = dloss; a.known_loss = q.loss; a.dx = dx;
    a.dz = (float*)ws; a.ld_dz = up(q.t.V, 16); a.alive = (int*)(a.dz + up(q.t.M, 16) * a.ld_dz);
    vocab_small<DT, true><<<(unsigned)tiles(q.t.M, SMALL_TOKENS), 64 * SMALL_WAVES, SMALL_TOKENS * a.ld_z * 4, s>>>(a);
    if (const int e = launch_status()) return e;
    if (dw) {
      const SmallDwArgs d{q.x, q.ldx, q.t.M, q.t.V, q.D, a.dz, a.ld_dz, a.alive, dw};
      vocab_small_dw<DT><<<dim3((unsigned)tiles(q.t.V, 16), (unsigned)tiles(q.D, 16)), 64 * SMALL_DW_WAVES, 0, s>>>(d);
    }
    return launch_status();
  }
};

// ---- few tokens ------------------------------------------------------------------------------------------------------
template <int DT> struct Few {
  static int targets(const Problem& q, const FewPlan& p, char* ws, const float* dloss, hipStream_t s) {
    TargetsArgs a = {};
    a.t = q.t; a.flags_n = up(q.t.M, 16); a.token_groups = (unsigned)tiles(a.flags_n, 4);
    a.dloss = dloss; a.flag = (uint8_t*)(ws + p.flag); a.q = (float*)(ws + p.q); a.q_sum = a.q + q.t.M * q.t.K;
    if (!dloss) a.entropy = (float*)(ws + p.entropy);
    vocab_targets<<<a.token_groups, 256, 0, s>>>(a);
    return launch_status();
  }
  static FewArgs args(const Problem& q, const FewPlan& p, char* ws) {
    FewArgs a = {};
    a.t = q.t; a.flag = q.t.logits ? (const uint8_t*)(ws + p.flag) : nullptr;
    a.x = q.x; a.ldx = q.ldx; a.w = q.w; a.ldw = q.ldw; a.D = q.D;
    a.z = (float*)(ws + p.z); a.ld_z = p.ld_z;
    return a;
  }
  template <int NT> static int forward(const Problem& q, const FewPlan& p, char* ws, float* loss, float* lse, float* hit, hipStream_t s) {
    if (q.t.logits)
      if (const int e = targets(q, p, ws, nullptr, s)) return e;
    FewArgs a = args(q, p, ws);
    a.part = (float2*)(ws + p.part);
    vocab_few_logits<DT, NT, false><<<(unsigned)(p.ld_z / FEW_ROWS), 256, 0, s>>>(a);
    if (const int e = launch_status()) return e;
    vocab_few_join<<<(unsigned)q.t.M, 256, 0, s>>>(FewJoinArgs{q.t, a.flag, a.z, p.ld_z, a.part, (const float*)(ws + p.q), (const float*)(ws + p.entropy), loss, lse, hit});
    return launch_status();
  }
  template <int NT> static int backward(const Problem& q, const FewPlan& p, char* ws, const float* lse, const float* hit, const float* dloss, void* dx, void* dw, hipStream_t s) {
    if (q.t.logits)
      if (const int e = targets(q, p, ws, dloss, s)) return e;
    FewArgs a = args(q, p, ws);
    a.lse = lse; a.dloss = dloss; a.loss = q.loss;
    vocab_few_logits<DT, NT, true><<<(unsigned)(p.ld_z / FEW_ROWS), 256, 0, s>>>(a);
    if (const int e = launch_status()) return e;
    if (q.t.logits) {
      vocab_few_hits<<<(unsigned)tiles(q.t.M * q.t.K, 256), 256, 0, s>>>(q.t, lse, hit, (const float*)(ws + p.q) + q.t.M * q.t.K, dloss, a.z, p.ld_z);
      if (const int e = launch_status()) return e;
    }
    if (dx) {
      float* slab = (float*)(ws + p.slab);
      vocab_few_dx<DT, NT><<<(unsigned)(p.ld_slab / 64 * up(p.splits, 8)), 256, 0, s>>>(FewDxArgs{q.w, q.ldw, q.t.V, q.D, a.z, p.ld_z, p.dx_rows, p.splits, slab, p.ld_slab});
      if (const int e = launch_status()) return e;
      vocab_few_finish<DT><<<dim3((unsigned)tiles(q.D, 256), (unsigned)q.t.M), 256, 0, s>>>(q.t, a.flag, slab, p.ld_slab, p.tokens * p.ld_slab, (int)p.splits, q.D, dx);
      if (const int e = launch_status()) return e;
    }
    if (dw) {
      const int64_t rows = p.ld_z / FEW_ROWS, most = tiles(q.D, 256), parts = most * rows < 1024 ? most : tiles(1024, rows);
      const int64_t features = up(tiles(q.D, parts), 256);
      vocab_few_dw<DT, NT><<<dim3((unsigned)rows, (unsigned)tiles(q.D, features)), 256, 0, s>>>(FewDwArgs{q.t, a.flag, q.x, q.ldx, q.D, a.z, p.ld_z, features, dw});
    }
    return launch_status();
  }
  static int forward(const Problem& q, void* ws, size_t ws_bytes, float* loss, float* lse, float* hit, hipStream_t s) {
    const FewPlan p = few_plan(q.t.M, q.t.V, q.D, q.t.K, q.t.logits != nullptr, 0);
    if (!ws || ws_bytes < (size_t)p.bytes || ((uintptr_t)ws & 255)) return GNET_ERR_WORKSPACE;
    return p.tokens == 16 ? forward<1>(q, p, (char*)ws, loss, lse, hit, s) : forward<2>(q, p, (char*)ws, loss, lse, hit, s);
  }
  static int backward(const Problem& q, void* ws, size_t ws_bytes, const float* lse, const float* hit, const float* dloss, void* dx, void* dw, hipStream_t s) {
    const FewPlan p = few_plan(q.t.M, q.t.V, q.D, q.t.K, q.t.logits != nullptr, 1);
    if (!ws || ws_bytes < (size_t)p.bytes || ((uintptr_t)ws & 255)) return GNET_ERR_WORKSPACE;
    return p.tokens == 16 ? backward<1>(q, p, (char*)ws, lse, hit, dloss, dx, dw, s) : backward<2>(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
  }
};

template <int DT, class T, int PLANES> struct Run {
  template <int BM, int BN, int WM, int WN, int STAGES, bool AS, bool BS, int EPI> static int launch(VocabGemm& g, int64_t rows, int64_t cols, int splits, hipStream_t s) {
    g.row_tiles = (int)tiles(rows, BM); g.col_tiles = (int)tiles(cols, BN); g.splits = splits;
    // half tiles are workgroups of their own; how many columns of tiles there are is known on the device, so the most of all counts
    const int64_t at_once = vocab_halves<BN, BS>() ? vocab_at_once<BM>() : 1;
    int64_t groups = 0;
    for (int64_t c = g.col_tiles; c > 0; --c) {
      const int64_t share = tiles(std::max((int64_t)g.row_tiles * c * splits, (int64_t)g.fit.slots), 8);
      for (int64_t k = share; k >= 0 && k >= share - 1; --k) groups = std::max(groups, k + (2 * (k % at_once) <= at_once ? k % at_once : 0));
      if (g.fit.slots) groups = share + at_once / 2;                  // (any share up to this one)
      if (!g.cols_from_meta || share + at_once / 2 <= groups) break;
    }
    vocab_gemm<T, BM, BN, WM, WN, STAGES, AS, BS, EPI, PLANES><<<(unsigned)(8 * groups), 64 * WM * WN, 0, s>>>(g);
    return launch_status();
  }
  // columns are tokens (all shapes) or vocabulary (the square ones)
  template <bool AS, bool BS, int EPI> static int gemm(VocabGemm& g, const Product& p, int64_t rows, int64_t cols, hipStream_t s) {
    if constexpr (EPI != EPI_DZ_ONE) { if (p.shape == S256) return launch<256, 256, 2, 4, 2, AS, BS, EPI>(g, rows, cols, p.splits, s); }
    if constexpr (!BS) {
      if (p.shape == S64) return launch<128, 64, 4, 1, 2, AS, BS, EPI>(g, rows, cols, p.splits, s);
      if (p.shape == S32) return launch<128, 32, 4, 1, 2, AS, BS, EPI>(g, rows, cols, p.splits, s);
    }
    return launch<128, 128, 2, 2, 2, AS, BS, EPI>(g, rows, cols, p.splits, s);
  }

  static PackW pack_of_w(const Problem& q, const Plan& p, char* ws, int64_t v0) {
    PackW k = {};
    k.w = (const char*)q.w + v0 * q.ldw * (DT == GNET_F32 ? 4 : 2);
    k.ldw = q.ldw; k.rows = q.t.V - v0; k.rows_out = p.piece; k.dst = (u16*)(ws + p.wp);
    k.each = p.piece <= 8192 ? 4 : 16;                    // (194 x 3858: 11.5 us, 16 a workgroup 19.8; every one looks at the magnitudes first)
    k.c = RowCopy{q.D, p.Dp, p.piece * p.Dp, 1.f};
    return k;
  }
  // everything in front of the first product, the first piece of W included
  static int prepare(const Problem& q, const Plan& p, char* ws, const float* dloss, const float* lse, void* dx, float* hit, hipStream_t s) {
    TargetsArgs a = {};
    a.t = q.t; a.flags_n = p.flags_n; a.token_groups = (unsigned)tiles(p.flags_n, 4);
    a.dloss = dloss;
    if (!p.direct) {
      a.flag = (uint8_t*)(ws + p.flag);
      if (q.t.logits) { a.q = (float*)(ws + p.q); a.q_sum = a.q + q.t.M * q.t.K; if (!dloss) a.entropy = (float*)(ws + p.entropy); }
      if (dloss) a.row_g = (float*)(ws + p.row_g);
      a.ldx = q.ldx; a.D = q.D;
      if (PLANES == 2) {
        a.x = (const float*)q.x; a.row_x = (float*)(ws + p.row_x);
        a.w = (const float*)q.w; a.ldw = q.ldw; a.w_part = (float*)(ws + p.w_part);
      }
      vocab_targets<<<a.token_groups + (PLANES == 2 ? W_PARTS : 0), 256, 0, s>>>(a);
      if (const int e = launch_status()) return e;
    }
    PackArgs k = {};
    k.t = q.t; k.flag = a.flag; k.flags_n = p.flags_n; k.Mp = p.Mp;
    k.rows = 4;
    while (tiles(p.Mp, k.rows) > 1024) k.rows *= 2;             // every workgroup looks at all M flags
    k.token_groups = (unsigned)tiles(p.Mp, k.rows);
    k.x = q.x; k.ldx = q.ldx; k.xp = (u16*)(ws + p.xp);
    k.c = RowCopy{q.D, p.Dp, p.Mp * p.Dp, 1.f};
    k.row_x = a.row_x; k.w_part = a.w_part;
    k.row_g = a.row_g; k.dloss = dloss; k.loss = q.loss; k.lse = lse; k.top_exp = DT == GNET_BF16 ? 0 : 15;
    k.pos = (int32_t*)(ws + p.pos); k.label = q.t.logits ? nullptr : (int32_t*)(ws + p.label);
    k.lse_c = (float*)(ws + p.lse_c); k.gscale = (float*)(ws + p.gscale); k.label_p = (float*)(ws + p.label_p);
    k.xg = (u16*)(ws + p.xg); k.exp_c = (int32_t*)(ws + p.exp_c);
    k.meta = (VocabMeta*)(ws + p.meta);
    if (dx && p.dx_direct) { k.dx = dx; k.row_of = (int32_t*)(ws + p.row_of); }
    if (p.pack_w) { k.w = pack_of_w(q, p, ws, 0); k.w_groups = (unsigned)tiles(p.piece, k.w.each); }
    int64_t groups = k.token_groups + k.w_groups;
    if (hit && q.t.logits) {
      k.dots = DotArgs{q.x, q.ldx, q.w, q.ldw, q.D, hit, (q.t.K + 3) / 4};
      groups += tiles(q.t.M * k.dots.per_token, 4);
    }
    if (dloss) vocab_pack<DT, true><<<grid_of(groups), 256, 0, s>>>(k);
    else vocab_pack<DT, false><<<grid_of(groups), 256, 0, s>>>(k);
    return launch_status();
  }

  // W rows v0 .. of one piece as an operand (packed first where needed)
  static int piece_of_w(const Problem& q, const Plan& p, char* ws, int64_t v0, VocabOperand& o, hipStream_t s) {
    o = VocabOperand{};
    if (p.pack_w) {
      const PackW k = pack_of_w(q, p, ws, v0);
      if (v0) vocab_pack_w<DT><<<(unsigned)tiles(p.piece, k.each), 256, 0, s>>>(k, (const VocabMeta*)(ws + p.meta));
      if (const int e = launch_status()) return e;
      o.p = (const u16*)(ws + p.wp); o.ld = p.Dp; o.plane = p.piece * p.Dp; o.rows = p.piece;
    } else {
      o.p = (const u16*)q.w + v0 * q.ldw; o.ld = q.ldw; o.plane = 0; o.rows = q.t.V - v0;
    }
    o.cols = (int)(p.pack_w ? p.Dp : q.D);
    return GNET_OK;
  }
  static VocabOperand packed_x(const Plan& p, char* ws, bool for_dw = false) {
    VocabOperand o = {};
    o.p = (const u16*)(ws + (for_dw && PLANES == 2 ? p.xg : p.xp)); o.ld = p.Dp; o.plane = p.Mp * p.Dp; o.rows = p.Mp; o.cols = (int)p.Dp;
    return o;
  }
  static VocabGemm logits(const Problem& q, const Plan& p, char* ws, const VocabOperand& w, int64_t v0) {
    VocabGemm g = {};
    g.a = w; g.b = packed_x(p, ws);
    g.k = p.Dp; g.cols_from_meta = 1;
    g.meta = (const VocabMeta*)(ws + p.meta);
    g.inv_temp = q.t.inv_temp; g.valid_rows = q.t.V - v0; g.first_row = (int32_t)v0;
    g.label = q.t.logits ? nullptr : (const int32_t*)(ws + p.label);
    return g;
  }

  // the logits' partial sums, all of them
  static int split_logits(VocabGemm g, const Problem& q, const Plan& p, char* ws, RowsArgs& r, hipStream_t s) {
    g.slab = (float*)(ws + p.z_slab); g.ld_slab = p.piece; g.slab_stride = p.Mp * p.piece; g.out_cols = p.Mp;
    r = RowsArgs{};
    r.t = q.t; r.slab = g.slab; r.ld = p.piece; r.stride = g.slab_stride; r.splits = p.logits.splits; r.meta = g.meta;
    return gemm<false, false, EPI_SLAB>(g, p.logits, q.t.V, q.t.M, s);
  }

  static int forward(const Problem& q, const Plan& p, char* ws, float* loss, float* lse, float* hit, hipStream_t s) {
    if (const int e = prepare(q, p, ws, nullptr, nullptr, nullptr, hit, s)) return e;
    VocabOperand w;
    const int32_t* pos = (const int32_t*)(ws + p.pos);
    const float* weights = (const float*)(ws + p.q);
    const float* entropy = (const float*)(ws + p.entropy);
    if (p.logits.splits > 1) {
      RowsArgs r;
      if (const int e = piece_of_w(q, p, ws, 0, w, s)) return e;
      if (const int e = split_logits(logits(q, p, ws, w, 0), q, p, ws, r, s)) return e;
      r.pos = pos; r.q = weights; r.entropy = entropy; r.loss = loss; r.lse = lse; r.hit = hit;
      vocab_rows<T, PLANES, false><<<(unsigned)q.t.M, 256, 0, s>>>(r);
      return launch_status();
    }
    for (int64_t v0 = 0; v0 < q.t.V; v0 += p.piece) {
      if (const int e = piece_of_w(q, p, ws, v0, w, s)) return e;
      VocabGemm g = logits(q, p, ws, w, v0);
      g.part = (float2*)(ws + p.part); g.hit = (float*)(ws + p.hit_c);
      g.first_row_tile = (int)(v0 / SHAPE[p.logits.shape].bm); g.all_row_tiles = (int)p.w_tiles;
      if (const int e = gemm<false, false, EPI_PART>(g, p.logits, q.t.V - v0 < p.piece ? q.t.V - v0 : p.piece, q.t.M, s)) return e;
    }
    JoinArgs j = {};
    j.t = q.t; j.pos = pos; j.part = (const float2*)(ws + p.part); j.tiles = (int)p.w_tiles; j.hit_c = (const float*)(ws + p.hit_c);
    j.q = weights; j.entropy = entropy;
    j.loss = loss; j.lse = lse; j.hit = hit;
    vocab_join<<<(unsigned)tiles(q.t.M, 4), 256, 0, s>>>(j);
    return launch_status();
  }

  static int finish(FinishArgs f, const Problem& q, hipStream_t s) {
    f.D = q.D; f.quads = (unsigned)tiles(q.D, 4);
    vocab_finish<DT><<<grid_of(tiles(f.rows * f.quads, 64)), 64, 0, s>>>(f);
    return launch_status();
  }

  static int backward(const Problem& q, const Plan& p, char* ws, const float* lse, const float* hit, const float* dloss, void* dx, void* dw, hipStream_t s) {
    if (const int e = prepare(q, p, ws, dloss, lse, dx, nullptr, s)) return e;
    VocabOperand w;
    const VocabMeta* meta = (const VocabMeta*)(ws + p.meta);
    const int elem = DT == GNET_F32 ? 4 : 2;
    for (int64_t v0 = 0; v0 < q.t.V; v0 += p.piece) {
      const int64_t rows = q.t.V - v0 < p.piece ? q.t.V - v0 : p.piece, rows64 = up(rows, VG_BK);
      if (const int e = piece_of_w(q, p, ws, v0, w, s)) return e;
      VocabGemm g = logits(q, p, ws, w, v0);
      g.lse = (const float*)(ws + p.lse_c); g.gscale = (const float*)(ws + p.gscale);
      if (q.loss) g.label_p = (const float*)(ws + p.label_p);
      g.dz = (u16*)(ws + p.dz); g.ld_dz = p.piece; g.plane_dz = p.Mp * p.piece; g.dz_cols = p.Mp;
      if (p.logits.splits > 1) {
        RowsArgs r;
        if (const int e = split_logits(g, q, p, ws, r, s)) return e;
        r.label = g.label; r.gscale = g.gscale; r.label_p = g.label_p; r.dz = g.dz; r.ld_dz = g.ld_dz; r.plane = g.plane_dz;
        vocab_rows<T, PLANES, true><<<(unsigned)p.Mp, 256, 0, s>>>(r);
        if (const int e = launch_status()) return e;
      } else if (const int e = p.logits.shape != S256 && q.t.V <= SHAPE[p.logits.shape].bm ? gemm<false, false, EPI_DZ_ONE>(g, p.logits, rows, q.t.M, s)
                                                                                           : gemm<false, false, EPI_DZ>(g, p.logits, rows, q.t.M, s)) return e;
      if (q.t.logits) {
        HitsArgs h = {};
        h.t = q.t; h.pos = (const int32_t*)(ws + p.pos); h.lse = lse; h.hit = hit;
        h.q = (const float*)(ws + p.q) + q.t.M * q.t.K;
        h.gscale = g.gscale; h.dz = g.dz; h.ld_dz = g.ld_dz; h.plane = g.plane_dz; h.v0 = v0; h.v1 = v0 + rows;
        vocab_hits<T, PLANES><<<grid_of(tiles(q.t.M * q.t.K, 256)), 256, 0, s>>>(h);
        if (const int e = launch_status()) return e;
      }
      VocabOperand dz = {};
      dz.p = g.dz; dz.ld = p.piece; dz.plane = g.plane_dz; dz.rows = p.Mp; dz.cols = (int)p.piece;
      if (dx) {
        VocabGemm d = {};
        d.a = w; d.b = dz; d.k = rows64; d.cols_from_meta = 1; d.meta = meta; d.out_cols = p.Mp;
        if (p.dx_direct) {
          d.out = dx; d.ld_out = q.D; d.out_rows = q.D;
          d.row_of = (const int32_t*)(ws + p.row_of); d.col_exp = (const int32_t*)(ws + p.exp_c);
          if (const int e = gemm<true, false, EPI_OUT>(d, p.dx, p.Dp, q.t.M, s)) return e;
        } else {
          d.slab = (float*)(ws + p.dx_slab); d.ld_slab = p.Dp; d.slab_stride = p.Mp * p.Dp; d.accumulate = v0 > 0; d.fit = p.dx_fit;
          if (const int e = gemm<true, false, EPI_SLAB>(d, p.dx, p.Dp, q.t.M, s)) return e;
        }
      }
      if (dw) {
        VocabGemm d = {};
        d.a = packed_x(p, ws, true); d.b = dz; d.k_from_meta = 1; d.meta = meta;
        d.out_cols = rows;
        void* out = (char*)dw + v0 * q.D * elem;
        if (p.dw.splits == 1) {
          d.out = out; d.ld_out = q.D; d.out_rows = q.D; d.unscale_by_x = 1;
          if (const int e = gemm<true, true, EPI_OUT>(d, p.dw, p.Dp, rows, s)) return e;
        } else {
          d.slab = (float*)(ws + p.dw_slab); d.ld_slab = p.Dp; d.slab_stride = p.piece * p.Dp;
          if (const int e = gemm<true, true, EPI_SLAB>(d, p.dw, p.Dp, rows, s)) return e;
          FinishArgs f = {};
          f.slab = d.slab; f.ld = p.Dp; f.stride = d.slab_stride; f.splits = p.dw.splits;
          f.rows = rows; f.out = out; f.meta = meta; f.by_x = 1;
          if (const int e = finish(f, q, s)) return e;
        }
      }
    }
    if (dx && !p.dx_direct) {
      FinishArgs f = {};
      f.slab = (const float*)(ws + p.dx_slab); f.ld = p.Dp; f.stride = p.Mp * p.Dp; f.splits = p.dx.splits; f.fit = p.dx_fit; f.out_cols = p.Mp;
      f.pos = (const int32_t*)(ws + p.pos); if (PLANES == 2) f.exp_c = (const int32_t*)(ws + p.exp_c);
      f.rows = q.t.M; f.out = dx; f.meta = meta;
      if (const int e = finish(f, q, s)) return e;
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
  const int pack_w = needs_pack(q.w, q.ldw, q.D, q.dtype);
  if (few_tokens(q.t.M, q.t.V, q.D, q.t.K, q.dtype, pack_w)) switch (q.dtype) {
    case GNET_F32: return Few<GNET_F32>::forward(q, ws, ws_bytes, loss, lse, hit, s);
    case GNET_BF16: return Few<GNET_BF16>::forward(q, ws, ws_bytes, loss, lse, hit, s);
    default: return Few<GNET_F16>::forward(q, ws, ws_bytes, loss, lse, hit, s);
  }
  if (small(q.t.M, q.t.V, q.D, q.t.K, q.dtype)) switch (q.dtype) {
    case GNET_F32: return Small<GNET_F32>::forward(q, loss, lse, hit, s);
    case GNET_BF16: return Small<GNET_BF16>::forward(q, loss, lse, hit, s);
    default: return Small<GNET_F16>::forward(q, loss, lse, hit, s);
  }
  const Plan p = make_plan(q.t.M, q.t.V, q.D, q.t.K, q.dtype, q.t.logits != nullptr, pack_w, 0);
  if (!p.launchable) return GNET_ERR_UNSUPPORTED;
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
  const int pack_w = needs_pack(q.w, q.ldw, q.D, q.dtype);
  if (few_tokens(q.t.M, q.t.V, q.D, q.t.K, q.dtype, pack_w)) switch (q.dtype) {
    case GNET_F32: return Few<GNET_F32>::backward(q, ws, ws_bytes, lse, hit, dloss, dx, dw, s);
    case GNET_BF16: return Few<GNET_BF16>::backward(q, ws, ws_bytes, lse, hit, dloss, dx, dw, s);
    default: return Few<GNET_F16>::backward(q, ws, ws_bytes, lse, hit, dloss, dx, dw, s);
  }
  if (small(q.t.M, q.t.V, q.D, q.t.K, q.dtype)) {
    if (!ws || ws_bytes < small_bytes(q.t.M, q.t.V) || ((uintptr_t)ws & 255)) return GNET_ERR_WORKSPACE;
    switch (q.dtype) {
      case GNET_F32: return Small<GNET_F32>::backward(q, (char*)ws, dloss, dx, dw, s);
      case GNET_BF16: return Small<GNET_BF16>::backward(q, (char*)ws, dloss, dx, dw, s);
      default: return Small<GNET_F16>::backward(q, (char*)ws, dloss, dx, dw, s);
    }
  }
  const Plan p = make_plan(q.t.M, q.t.V, q.D, q.t.K, q.dtype, q.t.logits != nullptr, pack_w, 1);
  if (!p.launchable) return GNET_ERR_UNSUPPORTED;
  if (!ws || ws_bytes < (size_t)p.bytes || ((uintptr_t)ws & 255)) return GNET_ERR_WORKSPACE;
  switch (q.dtype) {
    case GNET_F32: return Run<GNET_F32, F16T, 2>::backward(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
    case GNET_BF16: return Run<GNET_BF16, Bf16T, 1>::backward(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
    default: return Run<GNET_F16, F16T, 1>::backward(q, p, (char*)ws, lse, hit, dloss, dx, dw, s);
  }
}

Problem problem(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* ids, int ids64, const float* logits, float temperature,
                int64_t M, int64_t V, int64_t D, int64_t K, int dtype) {
  Problem q = {};
  q.x = x; q.ldx = ldx; q.w = w; q.ldw = ldw; q.D = D; q.dtype = dtype;
  q.t.ids = ids; q.t.ids64 = ids64; q.t.logits = logits; q.t.M = M; q.t.K = (int)(K > 1 << 20 ? 1 << 20 : K); q.t.V = V;
  q.t.inv_temp = 1.f / temperature; q.t.to_log2 = LOG2E / temperature;
  return q;
}

}  // namespace

// ------------------------------------------------------------------------------------------
extern "C" size_t gnet_vocab_workspace_bytes(const void* w, int64_t ldw, int64_t M, int64_t V, int64_t D, int64_t K, int32_t dtype, int32_t backward) {
  if (M <= 0 || V < 1 || D < 1 || K < 0 || M > (1 << 24) || V > (1ll << 30) || D > (1 << 16) || K > 1024) return 0;
  const int pack_w = needs_pack(w, ldw, D, dtype);
  // K = 0: cross entropy
  if (small(M, V, D, K, dtype)) return backward ? small_bytes(M, V) : 0;
  if (few_tokens(M, V, D, K, dtype, pack_w)) return (size_t)few_plan(M, V, D, K, K > 0, backward).bytes;
  return (size_t)make_plan(M, V, D, K, dtype, K > 0, pack_w, backward).bytes;
}

extern "C" int gnet_xent_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* labels, int32_t labels64, int64_t M,
                                 int64_t V, int64_t D, int32_t dtype, float* loss, float* lse, float* hit, void* workspace,
                                 size_t workspace_bytes, gnet_stream_t stream) {
  return run_forward(problem(x, ldx, w, ldw, labels, labels64, nullptr, 1.f, M, V, D, 1, dtype), loss, lse, hit, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int gnet_xent_backward_loss(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* labels, int32_t labels64,
                                       const float* loss, const float* lse, const float* hit, const float* dloss, int64_t M, int64_t V,
                                       int64_t D, int32_t dtype, void* dx, void* dw, void* workspace, size_t workspace_bytes,
                                       gnet_stream_t stream) {
  Problem q = problem(x, ldx, w, ldw, labels, labels64, nullptr, 1.f, M, V, D, 1, dtype);
  q.loss = loss;
  return run_backward(q, lse, hit, dloss, dx, dw, workspace, workspace_bytes, (hipStream_t)stream);
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
