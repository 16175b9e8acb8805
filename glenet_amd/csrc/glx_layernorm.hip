// Layer norm over the last dimension, forward and backward (glenet_amd/norm.py).
//
//   y = (x - mean) rstd w + b,   mean = sum x / C,   rstd = 1 / sqrt(sum (x - mean)^2 / C + eps)
//   g = gy w,   xhat = (x - mean) rstd
//   dx = rstd (g - sum g / C - xhat sum(g xhat) / C),   dw = sum_rows gy xhat,   db = sum_rows gy
//
// Both directions are bound by memory: 2 elements per value forward, 3 backward.  A group of L threads owns a row and keeps it
// in registers between the two sums and the write (one pass over memory, the variance from centred values); L is a part of a
// wave for narrow rows (sums by shuffles, several rows per wave), a block for wide ones.  In the backward pass a thread owns
// the SAME columns of every row its group visits, so dw and db grow in registers and leave the block once; a second launch adds
// the blocks' parts in a fixed order (no atomics: the same result every time).
//
// 131072 x 1024 bf16: forward 107 us (5.0 TB/s), backward 178 + 5 (4.4; a large copy: 5.1); 58733 x 64 fp32: 9 and 12 + 3 us
// (3.4 TB/s and 3.0: 30 and 45 MB are over before all of the card's memory is busy); 128 x 256: 3.5 and 6.5, all latency.
#include "glx_elem.h"

#define LN_BLOCKS 1024        // forward / backward groups stride over the rows from this many blocks
#define LN_COL_ROWS 64        // rows of one split of the column sums of wide rows, at least

template <typename T> struct LnVec { static constexpr int N = sizeof(T) == 4 ? 4 : 8; };

struct LnArgs {
  const void* x; const void* gy; const void* w; const void* b;
  void* y;                    // forward: y; backward: dx
  float* mean; float* rstd;
  float* part;                // [blocks][2][C]
  void* dw; void* db;         // written by a backward pass of one block
  long long ldx, ldg, rows, C;
  float eps;
  int wf32;                   // the weights are fp32 (else of x's type)
};

// VEC consecutive values as floats; beyond the row's end: `fill`
template <typename T>
__device__ __forceinline__ void ln_load(const T* __restrict__ p, long long col, long long C, float fill, float* v) {
  constexpr int V = LnVec<T>::N;
  if (col + V <= C) {
    const auto r = GlxVec<T, V>::load(p + col);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)r[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = col + i < C ? (float)p[col + i] : fill;
  }
}
template <typename T>
__device__ __forceinline__ void ln_store(T* __restrict__ p, long long col, long long C, const float* v) {
  constexpr int V = LnVec<T>::N;
  if (col + V <= C) {
    typename GlxVec<T, V>::vec r;
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = (T)v[i];
    GlxVec<T, V>::store(p + col, r);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (col + i < C) p[col + i] = (T)v[i];
  }
}
template <typename T>
__device__ __forceinline__ void ln_load_w(const void* w, int wf32, long long col, long long C, float fill, float* v) {
  constexpr int V = LnVec<T>::N;
  if (!w) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = fill;
  } else if (wf32 && sizeof(T) == 2) {
    const float* p = (const float*)w;
#pragma unroll
    for (int h = 0; h < V; h += 4) ln_load<float>(p, col + h, C, 0.f, v + h);
  } else {
    ln_load<T>((const T*)w, col, C, 0.f, v);
  }
}

// the sum over a row's group of L threads, in every thread of it; L > 64: `red` holds one value per wave.  A row's two sums use
// two such arrays: the barrier of the second one stands between the first one's reads and its next writes
template <int L>
__device__ __forceinline__ float ln_sum(float s, float* red) {
  constexpr int W = L < 64 ? L : 64;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) s += red[i];
  }
  return s;
}

// one row vector as it lies in memory; beyond the row's end zeros
template <typename T>
__device__ __forceinline__ typename GlxVec<T, LnVec<T>::N>::vec ln_raw(const T* __restrict__ p, long long col, long long C) {
  constexpr int V = LnVec<T>::N;
  if (col + V <= C) return GlxVec<T, V>::load(p + col);
  typename GlxVec<T, V>::vec r = {};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (col + i < C) r[i] = p[col + i];
  return r;
}

template <typename T, int L, int NV>
__global__ __launch_bounds__(256) void k_ln_forward(LnArgs a) {
  constexpr int V = LnVec<T>::N, G = 256 / L;
  __shared__ float red[2][16];
  const int t = threadIdx.x % L;
  const float inv = 1.f / (float)a.C;
  for (long long row = (long long)blockIdx.x * G + threadIdx.x / L; row < a.rows; row += (long long)gridDim.x * G) {
    const T* x = (const T*)a.x + row * a.ldx;
    typename GlxVec<T, V>::vec r[NV];                          // (as read: half the registers of floats for 16-bit rows)
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) r[j] = ln_raw<T>(x, (long long)(j * L + t) * V, a.C);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += (float)r[j][i];
    const float mean = ln_sum<L>(s, red[0]) * inv;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const long long left = a.C - (long long)(j * L + t) * V;
      if (left >= V) {
#pragma unroll
        for (int i = 0; i < V; ++i) { const float d = (float)r[j][i] - mean; s += d * d; }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) { const float d = (float)r[j][i] - mean; s += i < left ? d * d : 0.f; }
      }
    }
    const float rstd = 1.f / sqrtf(ln_sum<L>(s, red[1]) * inv + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const long long col = (long long)(j * L + t) * V;
      if (col >= a.C) break;
      float v[V], w[V], b[V];
      ln_load_w<T>(a.w, a.wf32, col, a.C, 1.f, w);
      ln_load_w<T>(a.b, a.wf32, col, a.C, 0.f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = ((float)r[j][i] - mean) * rstd * w[i] + b[i];
      ln_store<T>((T*)a.y + row * a.C, col, a.C, v);
    }
    if (a.mean && t == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  }
}

// Wider rows than 256 threads hold in four vectors each: three passes, the second and third from the caches, two blocks per compute
// unit (512 x 20736 fp32: 23 us, 83 KB a row; held in the registers of 1024 threads, one block per compute unit, 31 us)
template <typename T>
__global__ __launch_bounds__(1024) void k_ln_forward_long(LnArgs a) {
  constexpr int V = LnVec<T>::N;
  __shared__ float red[2][16];
  const double inv = 1.0 / (double)a.C;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    float s = 0.f;
#pragma unroll 4
    for (long long col = (long long)threadIdx.x * V; col < a.C; col += 1024 * V) {
      float v[V];
      ln_load<T>(x, col, a.C, 0.f, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[i];
    }
    const float mean = (float)(ln_sum<1024>(s, red[0]) * inv);
    s = 0.f;
#pragma unroll 4
    for (long long col = (long long)threadIdx.x * V; col < a.C; col += 1024 * V) {
      float v[V];
      ln_load<T>(x, col, a.C, mean, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += (v[i] - mean) * (v[i] - mean);
    }
    const float rstd = 1.f / sqrtf((float)(ln_sum<1024>(s, red[1]) * inv) + a.eps);
#pragma unroll 4
    for (long long col = (long long)threadIdx.x * V; col < a.C; col += 1024 * V) {
      float v[V], w[V], b[V];
      ln_load<T>(x, col, a.C, 0.f, v);
      ln_load_w<T>(a.w, a.wf32, col, a.C, 1.f, w);
      ln_load_w<T>(a.b, a.wf32, col, a.C, 0.f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (v[i] - mean) * rstd * w[i] + b[i];
      ln_store<T>((T*)a.y + row * a.C, col, a.C, v);
    }
    if (a.mean && threadIdx.x == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  }
}

// dx of the rows and, SUMS, the block's part of dw / db (one block: dw / db themselves)
template <typename T, int L, int NV, bool SUMS>
__global__ __launch_bounds__(256) void k_ln_backward(LnArgs a) {
  constexpr int V = LnVec<T>::N, G = 256 / L;
  __shared__ float red[2][16];
  const int t = threadIdx.x % L;
  const float inv = 1.f / (float)a.C;
  float dw[SUMS ? NV : 1][V], db[SUMS ? NV : 1][V];
  if (SUMS) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) dw[j][i] = db[j][i] = 0.f;
  }
  for (long long row = (long long)blockIdx.x * G + threadIdx.x / L; row < a.rows; row += (long long)gridDim.x * G) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* gy = (const T*)a.gy + row * a.ldg;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float h[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const long long col = (long long)(j * L + t) * V;
      float w[V];
      ln_load<T>(x, col, a.C, mean, h[j]);
      ln_load<T>(gy, col, a.C, 0.f, g[j]);
      ln_load_w<T>(a.w, a.wf32, col, a.C, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[j][i] = (h[j][i] - mean) * rstd;
        if (SUMS) { dw[j][i] += g[j][i] * h[j][i]; db[j][i] += g[j][i]; }
        g[j][i] *= w[i];
        const bool in = col + i < a.C;              // (beyond the row: no 0 * inf of a broken row's rstd)
        s1 += in ? g[j][i] : 0.f;
        s2 += in ? g[j][i] * h[j][i] : 0.f;
      }
    }
    s1 = ln_sum<L>(s1, red[0]) * inv;
    s2 = ln_sum<L>(s2, red[1]) * inv;
    if (a.y) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[j][i] = rstd * (g[j][i] - s1 - h[j][i] * s2);
        ln_store<T>((T*)a.y + row * a.C, (long long)(j * L + t) * V, a.C, g[j]);
      }
    }
  }
  if (!SUMS) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.C;
  auto put = [&](int k, long long c, float v) {                // column c of dw (k = 0) or db
    if (gridDim.x > 1) part[k * a.C + c] = v;
    else if (void* out = k ? a.db : a.dw) {
      if (a.wf32) ((float*)out)[c] = v;
      else ((T*)out)[c] = (T)v;
    }
  };
  if (G > 1) {
    // the wave's groups by shuffles, the block's four waves through LDS
    __shared__ float acc[4][(L < 64 ? L : 64) * NV * V];
#pragma unroll
    for (int o = 32; o >= L; o >>= 1)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dw[j][i] += __shfl_xor(dw[j][i], o, 64);
          db[j][i] += __shfl_xor(db[j][i], o, 64);
        }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if ((threadIdx.x & 63) < L) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[threadIdx.x >> 6][(j * L + t) * V + i] = k ? db[j][i] : dw[j][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += 256) put(k, c, acc[0][c] + acc[1][c] + acc[2][c] + acc[3][c]);
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const long long col = (long long)(j * L + t) * V;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (col + i < a.C) { put(0, col + i, dw[j][i]); put(1, col + i, db[j][i]); }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void k_ln_backward_long(LnArgs a) {
  constexpr int V = LnVec<T>::N;
  __shared__ float red[2][16];
  const double inv = 1.0 / (double)a.C;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* gy = (const T*)a.gy + row * a.ldg;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
    for (long long col = (long long)threadIdx.x * V; col < a.C; col += 1024 * V) {
      float h[V], g[V], w[V];
      ln_load<T>(x, col, a.C, mean, h);
      ln_load<T>(gy, col, a.C, 0.f, g);
      ln_load_w<T>(a.w, a.wf32, col, a.C, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool in = col + i < a.C;
        s1 += in ? g[i] * w[i] : 0.f;
        s2 += in ? g[i] * w[i] * ((h[i] - mean) * rstd) : 0.f;
      }
    }
    s1 = (float)(ln_sum<1024>(s1, red[0]) * inv);
    s2 = (float)(ln_sum<1024>(s2, red[1]) * inv);
#pragma unroll 4
    for (long long col = (long long)threadIdx.x * V; col < a.C; col += 1024 * V) {
      float h[V], g[V], w[V];
      ln_load<T>(x, col, a.C, mean, h);
      ln_load<T>(gy, col, a.C, 0.f, g);
      ln_load_w<T>(a.w, a.wf32, col, a.C, 1.f, w);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = rstd * (g[i] * w[i] - s1 - (h[i] - mean) * rstd * s2);
      ln_store<T>((T*)a.y + row * a.C, col, a.C, g);
    }
  }
}

// dw / db of wide rows (no thread holds a row's columns and two sums beside them): a wave's lanes own 64 V columns, the block's
// four waves take the split's rows in turn
template <typename T>
__global__ __launch_bounds__(256) void k_ln_columns(LnArgs a, long long rows_per) {
  constexpr int V = LnVec<T>::N;
  __shared__ float acc[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long c0 = (long long)blockIdx.x * 64 * V, col = c0 + lane * V;
  const long long r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < a.rows ? r0 + rows_per : a.rows;
  float dw[V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;
#pragma unroll 2
  for (long long row = r0 + wave; row < r1; row += 4) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float h[V], g[V];
    ln_load<T>((const T*)a.x + row * a.ldx, col, a.C, mean, h);
    ln_load<T>((const T*)a.gy + row * a.ldg, col, a.C, 0.f, g);
#pragma unroll
    for (int i = 0; i < V; ++i) { dw[i] += g[i] * ((h[i] - mean) * rstd); db[i] += g[i]; }
  }
  float* part = a.part + (long long)blockIdx.y * 2 * a.C;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) acc[wave][lane * V + i] = k ? db[i] : dw[i];
    __syncthreads();
    for (int c = threadIdx.x; c < 64 * V; c += 256)
      if (c0 + c < a.C) part[k * a.C + c0 + c] = acc[0][c] + acc[1][c] + acc[2][c] + acc[3][c];
    __syncthreads();
  }
}

// the parts' sums: 16 columns of dw | db per block, 64 threads down the parts of each
template <typename W>
__global__ __launch_bounds__(1024) void k_ln_join(const float* __restrict__ part, int parts, long long C, W* __restrict__ dw,
                                                 W* __restrict__ db) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const long long col = (long long)blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < 2 * C) {
#pragma unroll 4
    for (int p = r; p < parts; p += 64) s += part[(long long)p * 2 * C + col];
  }
  red[r][c] = s;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (r < o) red[r][c] += red[r + o][c];
    __syncthreads();
  }
  if (r == 0 && col < 2 * C) {
    W* out = col < C ? dw : db;
    if (out) out[col < C ? col : col - C] = (W)red[0][c];
  }
}

// ------------------------------------------------------------------------------------------------ plans
struct LnPlan {
  int L, NV;                  // threads of a row's group, vectors per thread; L = 0: a row in passes
  bool fused;                 // backward: the column sums ride on dx
  int blocks, parts;          // backward: blocks of the row kernel; parts of the column sums
  long long rows_per;         // rows of a split of k_ln_columns
};
static LnPlan ln_plan(long long rows, long long C, int dtype) {
  const int V = dtype == GLX_F32 ? 4 : 8;
  const long long nvec = (C + V - 1) / V;
  LnPlan p = {};
  static const int forms[][2] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}};
  for (auto& f : forms)
    if (nvec <= (long long)f[0] * f[1]) { p.L = f[0]; p.NV = f[1]; break; }
  const int G = p.L ? 256 / p.L : 1;
  p.fused = p.L;
  const long long groups = (rows + G - 1) / G;
  // eight visits a group: the parts stay small beside the rows.  Up to four groups one block does it all, without parts or a join
  long long want = groups / 8;
  want = p.fused && groups <= 4 ? 1 : want < 256 ? 256 : (want > LN_BLOCKS ? LN_BLOCKS : want);
  p.blocks = (int)(groups < want ? groups : want);
  if (p.fused) {
    p.parts = p.blocks;
  } else {
    const long long cb = (C + 64 * V - 1) / (64 * V);
    long long splits = (1024 + cb - 1) / cb, most = (rows + LN_COL_ROWS - 1) / LN_COL_ROWS;
    splits = splits > most ? most : splits;
    if (splits < 1) splits = 1;
    p.rows_per = (rows + splits - 1) / splits;
    p.parts = rows ? (int)((rows + p.rows_per - 1) / p.rows_per) : 0;
    if (p.parts == 1) p.parts = 2;                    // (an empty second part: these are always joined)
  }
  return p;
}

template <typename T>
static void ln_launch_forward(const LnPlan& p, const LnArgs& a, hipStream_t st) {
  const int G = p.L ? 256 / p.L : 1;
  const long long groups = (a.rows + G - 1) / G;
  const dim3 grid((unsigned)(groups < 8 * LN_BLOCKS ? groups : 8 * LN_BLOCKS));
#define LN_F(L_, N_) if (p.L == L_ && p.NV == N_) { hipLaunchKernelGGL((k_ln_forward<T, L_, N_>), grid, dim3(256), 0, st, a); return; }
  LN_F(8, 1) LN_F(16, 1) LN_F(32, 1) LN_F(64, 1) LN_F(64, 2) LN_F(64, 4) LN_F(256, 2) LN_F(256, 4)
#undef LN_F
  hipLaunchKernelGGL((k_ln_forward_long<T>), grid, dim3(1024), 0, st, a);
}
template <typename T>
static void ln_launch_backward(const LnPlan& p, const LnArgs& a, bool sums, hipStream_t st) {
  const dim3 grid(p.blocks);
#define LN_B(L_, N_)                                                                                                              \
  if (p.L == L_ && p.NV == N_) {                                                                                                  \
    if (sums) hipLaunchKernelGGL((k_ln_backward<T, L_, N_, true>), grid, dim3(256), 0, st, a);                                     \
    else hipLaunchKernelGGL((k_ln_backward<T, L_, N_, false>), grid, dim3(256), 0, st, a);                                        \
    return;                                                                                                                       \
  }
  LN_B(8, 1) LN_B(16, 1) LN_B(32, 1) LN_B(64, 1) LN_B(64, 2) LN_B(64, 4) LN_B(256, 2) LN_B(256, 4)
#undef LN_B
  if (p.L == 0 && a.y) hipLaunchKernelGGL((k_ln_backward_long<T>), grid, dim3(1024), 0, st, a);
  if (sums) {
    constexpr int V = LnVec<T>::N;
    hipLaunchKernelGGL((k_ln_columns<T>), dim3((unsigned)((a.C + 64 * V - 1) / (64 * V)), p.parts), dim3(256), 0, st, a, p.rows_per);
  }
}

static int ln_check(const char* who, int dtype, int wdtype, const void* weight, const void* bias, long long rows, long long width) {
  GLX_REQUIRE(glx_elem_ok(dtype), "%s: dtype %d", who, dtype);
  GLX_REQUIRE((!weight && !bias) || wdtype == GLX_F32 || wdtype == dtype, "%s: weights of type %d with inputs of type %d", who, wdtype, dtype);
  GLX_REQUIRE(width >= 1 && width <= (1ll << 31), "%s: width %lld", who, width);
  GLX_REQUIRE(rows >= 0 && rows <= (1ll << 40), "%s: %lld rows", who, rows);
  return GLX_OK;
}

extern "C" int glx_layer_norm_forward(const void* x, int64_t ldx, int dtype, const void* weight, const void* bias, int wdtype,
                                      int64_t rows, int64_t width, float eps, void* y, float* mean, float* rstd, void* stream) {
  if (int rc = ln_check("glx_layer_norm_forward", dtype, wdtype, weight, bias, rows, width)) return rc;
  if (rows == 0) return GLX_OK;
  GLX_REQUIRE(x && y && ldx >= 0 && !mean == !rstd, "glx_layer_norm_forward: bad pointers");
  LnArgs a = {};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.ldx = ldx; a.rows = rows; a.C = width; a.eps = eps; a.wf32 = wdtype == GLX_F32;
  const LnPlan p = ln_plan(rows, width, dtype);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == GLX_F32) ln_launch_forward<float>(p, a, st);
  else if (dtype == GLX_BF16) ln_launch_forward<__bf16>(p, a, st);
  else ln_launch_forward<_Float16>(p, a, st);
  GLX_LAUNCH_CHECK();
  return GLX_OK;
}

extern "C" size_t glx_layer_norm_workspace_bytes(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0) return 0;
  const LnPlan p = ln_plan(rows, width, GLX_F32), q = ln_plan(rows, width, GLX_BF16);
  const int parts = p.parts > q.parts ? p.parts : q.parts;
  return parts > 1 ? glx_align((size_t)parts * 2 * width * sizeof(float)) : 0;
}

extern "C" int glx_layer_norm_backward(const void* gy, int64_t ldg, const void* x, int64_t ldx, int dtype, const void* weight,
                                       int wdtype, const float* mean, const float* rstd, int64_t rows, int64_t width, void* dx,
                                       void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ln_check("glx_layer_norm_backward", dtype, wdtype, weight, nullptr, rows, width)) return rc;
  const bool sums = dweight || dbias;
  GLX_REQUIRE(!sums || wdtype == GLX_F32 || wdtype == dtype, "glx_layer_norm_backward: weight gradients of type %d", wdtype);
  GLX_REQUIRE(rows == 0 || (gy && x && mean && rstd && ldx >= 0 && ldg >= 0), "glx_layer_norm_backward: bad pointers");
  if (sums && workspace_bytes < glx_layer_norm_workspace_bytes(rows, width)) {
    glx_set_error("glx_layer_norm_backward: workspace %zu < %zu bytes", workspace_bytes, glx_layer_norm_workspace_bytes(rows, width));
    return GLX_EWORKSPACE;
  }
  if (!sums && (!dx || rows == 0)) return GLX_OK;
  LnArgs a = {};
  a.x = x; a.gy = gy; a.w = weight; a.y = dx; a.mean = (float*)mean; a.rstd = (float*)rstd; a.part = (float*)workspace; a.dw = dweight; a.db = dbias;
  a.ldx = ldx; a.ldg = ldg; a.rows = rows; a.C = width; a.wf32 = wdtype == GLX_F32;
  const LnPlan p = ln_plan(rows, width, dtype);
  hipStream_t st = (hipStream_t)stream;
  if (rows > 0) {
    if (dtype == GLX_F32) ln_launch_backward<float>(p, a, sums, st);
    else if (dtype == GLX_BF16) ln_launch_backward<__bf16>(p, a, sums, st);
    else ln_launch_backward<_Float16>(p, a, sums, st);
  }
  if (sums && !(p.fused && p.parts == 1 && rows > 0)) {
    const dim3 grid((unsigned)((2 * width + 15) / 16));
    const int parts = rows > 0 ? p.parts : 0;
    if (wdtype == GLX_F32)
      hipLaunchKernelGGL((k_ln_join<float>), grid, dim3(1024), 0, st, a.part, parts, (long long)width, (float*)dweight, (float*)dbias);
    else if (wdtype == GLX_BF16)
      hipLaunchKernelGGL((k_ln_join<__bf16>), grid, dim3(1024), 0, st, a.part, parts, (long long)width, (__bf16*)dweight, (__bf16*)dbias);
    else
      hipLaunchKernelGGL((k_ln_join<_Float16>), grid, dim3(1024), 0, st, a.part, parts, (long long)width, (_Float16*)dweight, (_Float16*)dbias);
  }
  GLX_LAUNCH_CHECK();
  return GLX_OK;
}
