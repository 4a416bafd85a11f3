// The vocabulary losses where the vocabulary is small (a detector's classes): the whole row of logits of a token fits into LDS, and
// what limits the general path is its launches (four forward, eight backward).  One launch forward; two backward.
//   vocab_small<false>   z = x . W^T of 16 tokens, their softmax, losses
//   vocab_small<true>    the same z again, dz = g (softmax(z) - weights), dx = dz . W
//   vocab_small_dw       dW = dz^T . x, a workgroup per 16 x 16 of it
// Products run on the fp32 matrix pipe (v_mfma_f32_16x16x4_f32) with all operands turned into fp32 on the way from memory, exact for every
// type; 16-bit logits on their own pipe.  A contraction's order is free as long as both operands agree: lane group q (16 lanes each) takes elements 4 q .. 4 q + 3 of 16,
// one vector load, where the instruction would have it take element q of four.
// (Included by vocab.hip behind its helpers.)
//
// Bound by latency: 2000 x 81 x 128 fp32 takes 7 us forward, 11 and 9 us backward, of which an empty launch is 2 to 3.
#pragma once

// N consecutive elements as they lie in memory, at an element's alignment
template <int DT, int N> struct SmallRaw {
  typedef std::conditional_t<DT == GNET_F32, float, short> E;
  typedef E V __attribute__((ext_vector_type(N)));
  typedef E U __attribute__((ext_vector_type(N), aligned(sizeof(E))));
  V v;
  // (16 bits at an odd address: the dwords that hold them, shifted.  A vector load that starts inside a dword takes 190 cycles a wave, one
  // at a dword's start 16; what the first and last dword hold besides, up to two bytes outside the row, is not used.)
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (DT == GNET_F32 || N < 4) v = *reinterpret_cast<const U*>((const E*)p + i);
    else {
      typedef unsigned W __attribute__((ext_vector_type(N / 2)));
      typedef unsigned WU __attribute__((ext_vector_type(N / 2), aligned(4)));
      const uintptr_t at = (uintptr_t)((const E*)p + i);
      const W lo = *reinterpret_cast<const WU*>(at & ~(uintptr_t)3);
      const unsigned hi = *reinterpret_cast<const unsigned*>((at + 2 * N - 2) & ~(uintptr_t)3), shift = (unsigned)(at & 2) * 8;
      W o;
#pragma unroll
      for (int k = 0; k < N / 2; ++k) o[k] = __builtin_amdgcn_alignbit(k + 1 < N / 2 ? lo[k + 1 < N / 2 ? k + 1 : k] : hi, lo[k], shift);
      v = __builtin_bit_cast(V, o);
    }
  }
  // `left` of them exist, maybe none, but the row has at least one: the last one in place of the others
  __device__ __forceinline__ void load(const void* p, int64_t i, int64_t left) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = ((const E*)p)[i + min((int64_t)j, left - 1)];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < left ? v[j] : (E)0;
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (DT == GNET_F32) return v[j];
    else return DT == GNET_BF16 ? Bf16T::dec((u16)v[j]) : F16T::dec((u16)v[j]);
  }
  __device__ __forceinline__ void set(int j, float f) {
    if constexpr (DT == GNET_F32) v[j] = f;
    else v[j] = (short)(DT == GNET_BF16 ? Bf16T::enc(f) : F16T::enc(f));
  }
  __device__ __forceinline__ void store(void* p, int64_t i, int64_t left) const {
    if (left >= N) { *reinterpret_cast<U*>((E*)p + i) = v; return; }
#pragma unroll
    for (int j = 0; j < N; ++j) if (j < left) ((E*)p)[i + j] = v[j];
  }
};
template <int DT> __device__ __forceinline__ void small_store(void* p, int64_t i, float v) {
  if constexpr (DT == GNET_F32) ((float*)p)[i] = v;
  else ((u16*)p)[i] = DT == GNET_BF16 ? Bf16T::enc(v) : F16T::enc(v);
}
// 16 rows of W times 16 tokens over one vector of each lane
template <int DT, int N> __device__ __forceinline__ void small_logits(f32x4& acc, const SmallRaw<DT, N>& w, const SmallRaw<DT, N>& x) {
  if constexpr (DT == GNET_F32) {
#pragma unroll
    for (int c = 0; c < N; ++c) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.get(c), x.get(c), acc, 0, 0, 0);
  } else acc = std::conditional_t<DT == GNET_BF16, Bf16T, F16T>::mma(w.v, x.v, acc);
}
__device__ __forceinline__ float half_wave_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float half_wave_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

constexpr int SMALL_TOKENS = 16, SMALL_WAVES = 8;      // a workgroup's tokens: 32 lanes each for the softmax
constexpr int SMALL_AHEAD = 8;                         // vector loads of one operand on the way at a time
constexpr int SMALL_K = 64;                            // targets at most: two a lane
struct SmallArgs {
  Targets t;
  const void* x; int64_t ldx; const void* w; int64_t ldw; int64_t D;
  int ld_z;                                            // LDS elements a token's row of z: 4 more than a multiple of 64 (banks)
  float* loss; float* lse; float* hit;                 // forward
  const float* dloss; const float* known_loss; float* dz; int64_t ld_dz; int* alive; void* dx;      // backward: dz [M up to 16][V up to 16]; known_loss may be NULL
};

template <int DT, bool BACKWARD> __global__ void __launch_bounds__(64 * SMALL_WAVES) vocab_small(const SmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) float z[];
  __shared__ int alive[SMALL_TOKENS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i16 = lane & 15, q4 = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * SMALL_TOKENS;
  const int V = (int)a.t.V, v_tiles = (V + 15) / 16;

  // the logits: rows of the product are the vocabulary, columns the tokens.  Rows and tokens that do not exist repeat the last one, and
  // tokens that are left out are computed like the others: no column looks at another, and theirs are not used.
  {
    constexpr int N = DT == GNET_F32 ? 4 : 8, CHUNK = 4 * N;
    const int64_t m = min(m0 + i16, a.t.M - 1), full = a.D / CHUNK * CHUNK;
    for (int tile = wave; tile < v_tiles; tile += SMALL_WAVES) {
      const int64_t row = (int64_t)min(tile * 16 + i16, V - 1) * a.ldw, x = m * a.ldx;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      for (int64_t d0 = 0; d0 < full; d0 += CHUNK * SMALL_AHEAD) {
        SmallRaw<DT, N> wv[SMALL_AHEAD], xv[SMALL_AHEAD];
#pragma unroll
        for (int u = 0; u < SMALL_AHEAD; ++u) {
          if (d0 + u * CHUNK >= full) continue;
          wv[u].load(a.w, row + d0 + u * CHUNK + q4 * N);
          xv[u].load(a.x, x + d0 + u * CHUNK + q4 * N);
        }
#pragma unroll
        for (int u = 0; u < SMALL_AHEAD; ++u)
          if (d0 + u * CHUNK < full) small_logits<DT>(acc, wv[u], xv[u]);
      }
      if (full < a.D) {
        const int64_t d = full + q4 * N, left = a.D - d;
        SmallRaw<DT, N> wv, xv;
        wv.load(a.w, row + d, left);
        xv.load(a.x, x + d, left);
        small_logits<DT>(acc, wv, xv);
      }
      *reinterpret_cast<f32x4*>(z + i16 * a.ld_z + tile * 16 + q4 * 4) = acc * a.t.inv_temp;
    }
  }
  __syncthreads();

  // softmax: 32 lanes a token, targets sub and sub + 32
  const int token = tid / 32, sub = tid & 31, K = a.t.K;
  const int64_t m = m0 + token;
  float* zt = z + token * a.ld_z;
  int64_t id[2] = {-1, -1};
  float tl[2] = {-INFINITY, -INFINITY}, weight[2] = {0.f, 0.f};
  bool counts[2] = {false, false};
  if (m < a.t.M)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (sub + j * 32 < K) {
        counts[j] = target_counts(a.t, m * K + sub + j * 32, id[j]);
        if (counts[j] && a.t.logits) tl[j] = a.t.logits[m * K + sub + j * 32];
      }
  const bool some = half_wave_max(counts[0] || counts[1] ? 1.f : 0.f) > 0.f;
  float top = -INFINITY, sum = 0.f;
  for (int v = sub; v < V; v += 32) top = fmaxf(top, zt[v]);
  top = half_wave_max(top);
  if (top == -INFINITY) top = 0.f;
  for (int v = sub; v < V; v += 32) sum += exp2f((zt[v] - top) * LOG2E);
  sum = half_wave_sum(sum);
  float entropy = 0.f;
  if (a.t.logits) {
    const float t_top = half_wave_max(fmaxf(tl[0], tl[1]));
#pragma unroll
    for (int j = 0; j < 2; ++j) weight[j] = counts[j] ? exp2f((tl[j] - t_top) * a.t.to_log2) : 0.f;
    const float t_sum = half_wave_sum(weight[0] + weight[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      weight[j] = some ? weight[j] / t_sum : 0.f;
      if (weight[j] != 0.f) entropy += weight[j] * ((tl[j] - t_top) * a.t.inv_temp - logf(t_sum));
    }
  } else weight[0] = counts[0] ? 1.f : 0.f;

  if constexpr (!BACKWARD) {
    if (m >= a.t.M) return;
    const float log_sum = logf(sum), lse = top + log_sum;
    float loss = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float hit = counts[j] ? zt[id[j]] : 0.f;
      if (sub + j * 32 < K) a.hit[m * K + sub + j * 32] = hit;
      if (weight[j] != 0.f) loss += weight[j] * (a.t.logits ? lse - hit : (top - hit) + log_sum);
    }
    loss = half_wave_sum(loss + entropy);
    if (!a.t.logits && loss < 0.f) loss = 0.f;
    if (sub == 0) { a.loss[m] = some ? loss : 0.f; a.lse[m] = some ? lse : 0.f; }
  } else {
    // p, less the weights one after the other (an id may occur more than once), times g
    const float over = 1.f / sum, g = some ? a.dloss[m] * a.t.inv_temp : 0.f;
    for (int v = sub; v < V; v += 32) zt[v] = exp2f((zt[v] - top) * LOG2E) * over;
    for (int k = 0; k < K; ++k) {
      __threadfence_block();                             // lanes of one wave
      const int j = k >> 5;
      if (sub == (k & 31) && (j ? counts[1] : counts[0])) zt[j ? id[1] : id[0]] -= j ? weight[1] : weight[0];
    }
    if (a.known_loss && sub == 0 && counts[0]) zt[id[0]] = expm1f(-a.known_loss[m]);      // (cross entropy)
    __threadfence_block();
    for (int v = sub; v < v_tiles * 16; v += 32) {
      const float d = some && v < V ? zt[v] * g : 0.f;
      zt[v] = d;
      a.dz[m * a.ld_dz + v] = d;
    }
    if (sub == 0) { alive[token] = some; a.alive[m] = some; }
    if (!a.dx) return;
    __syncthreads();
    // dx: rows of the product are tokens, columns features, two neighbours a lane
    for (int64_t d0 = wave * 32; d0 < a.D; d0 += SMALL_WAVES * 32) {
      const int64_t d = d0 + i16 * 2, left = a.D - d;
      f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      auto product = [&](auto whole) {
        for (int t0 = 0; t0 < v_tiles; t0 += SMALL_AHEAD / 2) {
          SmallRaw<DT, 2> wv[SMALL_AHEAD / 2][4];
#pragma unroll
          for (int u = 0; u < SMALL_AHEAD / 2; ++u) {
            if (t0 + u >= v_tiles) continue;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int64_t at = (int64_t)min((t0 + u) * 16 + q4 * 4 + c, V - 1) * a.ldw + d;
              if constexpr (whole) wv[u][c].load(a.w, at);
              else wv[u][c].load(a.w, at, left);
            }
          }
#pragma unroll
          for (int u = 0; u < SMALL_AHEAD / 2; ++u) {
            if (t0 + u >= v_tiles) continue;
            const f32x4 g4 = *reinterpret_cast<const f32x4*>(z + i16 * a.ld_z + (t0 + u) * 16 + q4 * 4);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int h = 0; h < 2; ++h) acc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(g4[c], wv[u][c].get(h), acc[h], 0, 0, 0);
          }
        }
      };
      if (d0 + 32 <= a.D) product(std::true_type{});
      else product(std::false_type{});
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = q4 * 4 + r;
        if (m0 + row >= a.t.M) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (h < left) small_store<DT>(a.dx, (m0 + row) * a.D + d + h, alive[row] ? acc[h][r] : 0.f);
      }
    }
  }
}

// 16 waves share the tokens, and add their results up in order.  (Tiles of 16 x 16: 16 x 32 leaves half as many CUs busy, 4 us more at
// 4096 x 81 x 128.)
constexpr int SMALL_DW_WAVES = 16;
struct SmallDwArgs {
  const void* x; int64_t ldx, M, V, D;
  const float* dz; int64_t ld_dz; const int* alive; void* dw;
};
template <int DT> __global__ void __launch_bounds__(64 * SMALL_DW_WAVES) vocab_small_dw(const SmallDwArgs a) {
  __shared__ float part[SMALL_DW_WAVES][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q4 = lane >> 4;
  const int64_t v0 = (int64_t)blockIdx.x * 16, d0 = (int64_t)blockIdx.y * 16, d = min(d0 + i16, a.D - 1);      // (columns behind D are not stored)
  const int64_t groups = (a.M + 15) / 16, first = groups * wave / SMALL_DW_WAVES, last = groups * (wave + 1) / SMALL_DW_WAVES;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int AHEAD = SMALL_AHEAD / 2;
  for (int64_t g = first; g < last; g += AHEAD) {
    float dz[AHEAD][4];
    int use[AHEAD][4];
    SmallRaw<DT, 1> xv[AHEAD][4];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (g + u >= last) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t m = (g + u) * 16 + c * 4 + q4;
        dz[u][c] = a.dz[m * a.ld_dz + v0 + i16];
        use[u][c] = a.alive[m];
        xv[u][c].load(a.x, min(m, a.M - 1) * a.ldx + d);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (g + u >= last) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(dz[u][c], use[u][c] ? xv[u][c].get(0) : 0.f, acc, 0, 0, 0);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) part[wave][r][lane] = acc[r];
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int row = threadIdx.x / 16, col = threadIdx.x & 15;
  if (v0 + row >= a.V || d0 + col >= a.D) return;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < SMALL_DW_WAVES; ++w) s += part[w][row & 3][(row >> 2) * 16 + col];
  small_store<DT>(a.dw, (v0 + row) * a.D + d0 + col, s);
}
