// The vocabulary losses for few tokens and a W that the 16-bit products cannot read where it lies (32 bits, odd widths): laying W out for
// them reads it once or twice and writes it before the first product.  These kernels read it once a product, at any alignment, and take
// every operand to fp32 in registers (v_mfma_f32_16x16x4_f32, exact for every type; the logits of 16-bit operands on their own pipe); with
// at most FEW_TOKENS tokens that pipe keeps up with memory.  The logits of all tokens are laid out (fp32, FEW_LOGITS bytes at most).
//   vocab_few_logits<false>  z, per 64 rows the maximum and sum of exp      vocab_few_join  lse, loss, hit
//   vocab_few_logits<true>   dz = g (softmax(z) - label)                    vocab_few_hits  dz at the teacher's ids
//   vocab_few_dx             dz . W, split over the vocabulary              vocab_few_finish  dx
//   vocab_few_dw             dz^T . x
// What they reach, 8 x 103105 x 2047 fp32 (0.84 GB a pass over W): logits 220 us, dx 268, dW 250, 3.1 to 3.8 TB/s; both directions 1093 us, and
// 2300 with W laid out first.  8 x 3000 x 593: 34 and 80; 24 x 300 x 2047 70 and 75; 8 x 30000 x 2047 bf16 151 and 262, 24 tokens 203 and 263, 48
// (not taken) 369 and 277.
// As in vocab_small.hpp the elements of a contraction are permuted so that a lane's share is one vector load.
// (Included by vocab.hip behind its helpers.)
#pragma once

constexpr int FEW_TOKENS = 32;
constexpr int64_t FEW_LOGITS = 64ll << 20;
constexpr int FEW_ROWS = 64;                       // vocabulary rows of a workgroup's logits: 16 of each of its 4 waves in the end

// does token m count (flag: vocab_targets', distillation)
__device__ __forceinline__ bool few_counts(const Targets& t, const uint8_t* flag, int64_t m) {
  if (m >= t.M) return false;
  if (flag) return flag[m];
  int64_t id;
  return target_counts(t, m, id);
}

struct FewArgs {
  Targets t; const uint8_t* flag;
  const void* x; int64_t ldx; const void* w; int64_t ldw; int64_t D;
  float* z; int64_t ld_z;                          // [16 NT][V rounded up to 64]: logits, or dz
  float2* part;                                    // forward: [token][ld_z / 64]
  const float* lse; const float* dloss; const float* loss;      // backward; loss may be NULL
};
// The four waves share the contraction, 64 bytes of a row at a time, and exchange their sums: wave w ends with rows 16 w .. of 64.
template <int DT, int NT, bool BACKWARD> __global__ void __launch_bounds__(256) vocab_few_logits(const FewArgs a) {
  constexpr int N = DT == GNET_F32 ? 4 : 8, CHUNK = 4 * N;
  __shared__ f32x4 other[4][3][NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q4 = lane >> 4;
  const int64_t r0 = (int64_t)blockIdx.x * FEW_ROWS;
  const void* w[4];
  const void* x[NT];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (const typename SmallRaw<DT, N>::E*)a.w + min(r0 + i * 16 + i16, a.t.V - 1) * a.ldw;
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = (const typename SmallRaw<DT, N>::E*)a.x + min((int64_t)n * 16 + i16, a.t.M - 1) * a.ldx;
  f32x4 acc[4][NT];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto products = [&](const SmallRaw<DT, N> (&wv)[4], const SmallRaw<DT, N> (&xv)[NT]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) small_logits<DT>(acc[i][n], wv[i], xv[n]);
  };
  const int64_t full = a.D / CHUNK;
  int64_t c = wave;
  constexpr int AHEAD = 2;
  for (; c + 4 * (AHEAD - 1) < full; c += 4 * AHEAD) {
    SmallRaw<DT, N> wv[AHEAD][4], xv[AHEAD][NT];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[u][i].load(w[i], (c + 4 * u) * CHUNK + q4 * N);
#pragma unroll
      for (int n = 0; n < NT; ++n) xv[u][n].load(x[n], (c + 4 * u) * CHUNK + q4 * N);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) products(wv[u], xv[u]);
  }
  for (; c * CHUNK < a.D; c += 4) {
    const int64_t d = c * CHUNK + q4 * N, left = a.D - d;
    SmallRaw<DT, N> wv[4], xv[NT];
    if (c < full) {
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[i].load(w[i], d);
#pragma unroll
      for (int n = 0; n < NT; ++n) xv[n].load(x[n], d);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[i].load(w[i], d, left);
#pragma unroll
      for (int n = 0; n < NT; ++n) xv[n].load(x[n], d, left);
    }
    products(wv, xv);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i != wave)
#pragma unroll
      for (int n = 0; n < NT; ++n) other[i][(wave + 3 - i) & 3][n][lane] = acc[i][n];
  __syncthreads();
  __shared__ float2 stats[4][NT][16];
  const int64_t row = r0 + wave * 16 + q4 * 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i == wave) z = acc[i][n];
#pragma unroll
    for (int k = 0; k < 3; ++k) z += other[wave][k][n][lane];
    z *= a.t.inv_temp;
    const int64_t m = n * 16 + i16;
    if constexpr (BACKWARD) {
      const bool some = few_counts(a.t, a.flag, m);
      const float g = some ? a.dloss[m] * a.t.inv_temp : 0.f, lse = some ? a.lse[m] : 0.f;
      const int64_t label = some && !a.t.logits ? load_id(a.t.ids, m, a.t.ids64) - row : -1;
      const float at_label = some && a.loss ? expm1f(-a.loss[m]) : 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = exp2f((z[r] - lse) * LOG2E), q = a.loss ? at_label : p - 1.f;
        z[r] = some && row + r < a.t.V ? (label == r ? q : p) * g : 0.f;
      }
    } else {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) if (row + r < a.t.V) top = fmaxf(top, z[r]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int r = 0; r < 4; ++r) if (row + r < a.t.V) sum += exp2f((z[r] - from) * LOG2E);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (q4 == 0) stats[wave][n][i16] = float2{top, sum};
    }
    *reinterpret_cast<f32x4*>(a.z + m * a.ld_z + row) = z;
  }
  if constexpr (!BACKWARD) {
    __syncthreads();
    const int m = threadIdx.x;
    if (m < NT * 16 && m < a.t.M) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, stats[k][m / 16][m & 15].x);
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += stats[k][m / 16][m & 15].y * exp2f((stats[k][m / 16][m & 15].x - from) * LOG2E);
      a.part[(int64_t)m * (a.ld_z / FEW_ROWS) + blockIdx.x] = float2{top, sum};
    }
  }
}

struct FewJoinArgs {
  Targets t; const uint8_t* flag;
  const float* z; int64_t ld_z; const float2* part; const float* q; const float* entropy;
  float* loss; float* lse; float* hit;
};
// a workgroup a token; each of its waves joins a quarter of the tiles
__global__ void __launch_bounds__(256) vocab_few_join(const FewJoinArgs a) {
  __shared__ float red[4];
  const int64_t m = blockIdx.x, K = a.t.K;
  const bool some = few_counts(a.t, a.flag, m);
  float top = -INFINITY, sum = 0.f, loss = 0.f;
  const int n = (int)(a.ld_z / FEW_ROWS);
  const float2* part = a.part + m * n;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) top = fmaxf(top, part[i].x);
  top = block_max(top, red);
  if (top == -INFINITY) top = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) sum += part[i].y * exp2f((part[i].x - top) * LOG2E);
  const float log_sum = logf(block_sum(sum, red)), lse = top + log_sum;
  for (int64_t k = threadIdx.x; k < K; k += 256) {
    int64_t id;
    const float hit = target_counts(a.t, m * K + k, id) ? a.z[m * a.ld_z + id] : 0.f;
    a.hit[m * K + k] = hit;
    if (!a.t.logits) {
      loss = (top - hit) + log_sum;
      if (loss < 0.f) loss = 0.f;
    } else {
      const float q = a.q[m * K + k];
      if (q != 0.f) loss += q * (lse - hit);
    }
  }
  if (a.t.logits) loss = block_sum(loss, red) + a.entropy[m];
  if (threadIdx.x == 0) { a.loss[m] = some ? loss : 0.f; a.lse[m] = some ? lse : 0.f; }
}

// (slots with the same id store the same value)
__global__ void __launch_bounds__(256) vocab_few_hits(const Targets t, const float* lse, const float* hit, const float* q, const float* dloss, float* dz, int64_t ld_z) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= t.M * t.K) return;
  const int64_t m = i / t.K;
  int64_t id;
  if (target_counts(t, i, id)) dz[m * ld_z + id] = (exp2f((hit[i] - lse[m]) * LOG2E) - q[i]) * (dloss[m] * t.inv_temp);
}

// dx: rows of the product are tokens, columns 64 features, four a lane; a workgroup takes `rows` rows of the vocabulary (a multiple
// of 64), its waves 16 in turn.  The workgroups of the same rows are eight apart: one L2 gets the lines that blocks of features share.
struct FewDxArgs {
  const void* w; int64_t ldw, V, D; const float* dz; int64_t ld_z, rows, splits; float* slab; int64_t ld_slab;      // [split][16 NT][ld_slab]
};
template <int DT, int NT> __global__ void __launch_bounds__(256) vocab_few_dx(const FewDxArgs a) {
  __shared__ f32x4 other[4][3][NT][64];            // by accumulator: wave w ends with features 4 i16 + w
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q4 = lane >> 4;
  const int64_t blocks = a.ld_slab / 64, split = blockIdx.x / 8 / blocks * 8 + blockIdx.x % 8;
  if (split >= a.splits) return;
  const int64_t d0 = blockIdx.x / 8 % blocks * 64, d = d0 + i16 * 4, left = a.D - d;
  const int64_t first = split * a.rows, last = min(first + a.rows, a.V);
  f32x4 acc[4][NT];
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[h][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int AHEAD = NT == 1 ? 4 : 2;
  auto product = [&](auto whole) {
    for (int64_t v0 = first + wave * 16; v0 < last; v0 += 64 * AHEAD) {
      SmallRaw<DT, 4> wv[AHEAD][4];
      f32x4 g[AHEAD][NT];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t v = v0 + u * 64;
        if (v >= last) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int64_t at = min(v + q4 * 4 + c, a.V - 1) * a.ldw + d;
          if constexpr (whole) wv[u][c].load(a.w, at);
          else wv[u][c].load(a.w, at, left);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) g[u][n] = *reinterpret_cast<const f32x4*>(a.dz + (n * 16 + i16) * a.ld_z + v + q4 * 4);      // (zeros behind V)
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (v0 + u * 64 >= last) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[h][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[u][n][c], wv[u][c].get(h), acc[h][n], 0, 0, 0);
      }
    }
  };
  if (d0 + 64 <= a.D) product(std::true_type{});
  else product(std::false_type{});
#pragma unroll
  for (int h = 0; h < 4; ++h)
    if (h != wave)
#pragma unroll
      for (int n = 0; n < NT; ++n) other[h][(wave + 3 - h) & 3][n][lane] = acc[h][n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 4; ++h) if (h == wave) s = acc[h][n];
#pragma unroll
    for (int k = 0; k < 3; ++k) s += other[wave][k][n][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) a.slab[(split * NT * 16 + n * 16 + q4 * 4 + r) * a.ld_slab + d + wave] = s[r];
  }
}
template <int DT> __global__ void __launch_bounds__(256) vocab_few_finish(const Targets t, const uint8_t* flag, const float* slab, int64_t ld_slab, int64_t stride, int splits, int64_t D, void* dx) {
  const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
  if (d >= D) return;
  float s = 0.f;
  if (few_counts(t, flag, m)) {
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += slab[k * stride + m * ld_slab + d];
  }
  small_store<DT>(dx, m * D + d, s);
}

// dW: rows of the product are the vocabulary, columns 64 features, four a lane.  A workgroup writes 64 rows (all of their features, if there
// are rows enough), its waves 64 features in turn: lines that rows or blocks share are put together in one L2.  (A block of features a
// workgroup: 103105 x 2047 fp32 332 us in place of 250.)
struct FewDwArgs {
  Targets t; const uint8_t* flag; const void* x; int64_t ldx, D; const float* dz; int64_t ld_z, features; void* dw;
};
template <int DT, int NT> __global__ void __launch_bounds__(256) vocab_few_dw(const FewDwArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q4 = lane >> 4;
  const int64_t v0 = (int64_t)blockIdx.x * FEW_ROWS;
  float g[4][NT * 4];                              // token 4 k + q4
  bool some[NT * 4];
#pragma unroll
  for (int k = 0; k < NT * 4; ++k) {
    some[k] = few_counts(a.t, a.flag, k * 4 + q4);
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i][k] = a.dz[(k * 4 + q4) * a.ld_z + v0 + i * 16 + i16];
  }
  const int64_t end = min(a.D, (blockIdx.y + 1) * a.features);
  for (int64_t d0 = blockIdx.y * a.features + wave * 64; d0 < end; d0 += 256) {
    const int64_t d = d0 + i16 * 4, left = a.D - d;
    SmallRaw<DT, 4> xv[NT * 4];
    if (d0 + 64 <= a.D) {
#pragma unroll
      for (int k = 0; k < NT * 4; ++k) xv[k].load(a.x, min((int64_t)k * 4 + q4, a.t.M - 1) * a.ldx + d);
    } else {
#pragma unroll
      for (int k = 0; k < NT * 4; ++k) xv[k].load(a.x, min((int64_t)k * 4 + q4, a.t.M - 1) * a.ldx + d, left);
    }
    float x[NT * 4][4];
#pragma unroll
    for (int k = 0; k < NT * 4; ++k)
#pragma unroll
      for (int h = 0; h < 4; ++h) x[k][h] = some[k] ? xv[k].get(h) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 acc[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NT * 4; ++k)
#pragma unroll
        for (int h = 0; h < 4; ++h) acc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[i][k], x[k][h], acc[h], 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t row = v0 + i * 16 + q4 * 4 + r;
        if (row >= a.t.V) continue;
        SmallRaw<DT, 4> o;
#pragma unroll
        for (int h = 0; h < 4; ++h) o.set(h, acc[h][r]);
        o.store(a.dw, row * a.D + d, left);
      }
    }
  }
}
