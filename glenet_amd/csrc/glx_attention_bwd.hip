// Cross attention of stacked frames, backward (glenet_amd/attention.py; the layouts: glx_attention.h).
//
//   P = 2^(scale2 Q K^T - lse),  dP = dO V^T,  delta = rowsum(dO O),  dS = P (dP - delta)
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
//
// Nothing of the size of the scores is stored: P is formed again from Q, K and the row's lse in each of two launches, one that
// owns rows (dQ, and delta for the other one) and one that owns keys (dK, dV; the rows of all query heads that share a key head
// are its sum).  Seven tile products instead of the five of a single pass that would need atomics or a second dQ buffer; the
// results are the same bits every time.  Few tiles are split over the other side and added by a last launch.
//
// 2 frames of 4096 queries over 16384 keys, 8 heads of 128 on 2 key heads, bf16: dQ 862 us (957 TFLOP/s; a large library product
// reaches 1156; products 48 % of a SIMD's cycles, vector instructions 52 %), dK / dV 1395 us (788; products 37 %, vector instructions
// 35 %: one wave per SIMD holds K, V, dK and dV, its LDS reads take as long as its products).
//
// P and dS are rounded to the inputs' type in front of their products.  fp16 would lose both to its range -- over a thousand
// keys P sits where fp16 has few bits left, and dS inherits the loss' scale -- so P is multiplied by 2^12 and dS by a power of
// two that keeps a wave's largest value between 2^8 and 2^15 (taken from the first tile, lowered with the accumulators when a
// later tile would pass it).
//
// dS sums to zero over a row, so what the keys of a row have in common leaves dQ, but the roundings of dS times it stay.  With few
// channels the scores pull a row's keys together: at dim 8, 4 x 4012 x 2768, 2 heads, bf16, dQ was 2.7e-3 off (the rounding of
// the result alone: 1.7e-3).  Heads of up to 32 channels, whose time is the exponentials, so add what the rounding left in a
// second product (there 201 -> 208 us a training pass, and dQ below 2.4e-3); wider ones do not.  The same for P and dS in front
// of dV and dK, where a few rows of a few channels left 1.6 times the rounding of the result.
#include "glx_attention.h"

#include <type_traits>

#define XA_PSCALE 4096.f      // fp16: of P

int xa_splits(long long blocks, long long keys_per_frame, int per_cu);
void xa_rows_plan(const glx_attention* t, int* rw, long long* tiles, int* splits);
int xa_check(const char* who, const glx_attention* t);
XaArgs xa_args(const glx_attention* t);

// fp16: 2^e for the values of one 32 x 32 tile; N accumulators of earlier tiles follow a change
template <typename T, int N>
__device__ __forceinline__ void xa_range(xf16& s, xf16 (&acc)[N], int& e) {
  if constexpr (__is_same(T, _Float16)) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[i]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (top > 0.f && top < 3e38f) {
      const int want = 8 - ilogbf(top);
      if (e > 200) {
        e = want > 120 ? 120 : want;
      } else if (ldexpf(top, e) >= 32768.f) {
        const float f = ldexpf(1.f, want - e);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int k = 0; k < 16; ++k) acc[i][k] *= f;
        e = want;
      }
    }
    const float f = ldexpf(1.f, e > 200 ? 0 : e);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= f;
  }
}
template <typename T>
__device__ __forceinline__ float xa_unrange(int e) {
  return __is_same(T, _Float16) && e <= 200 ? ldexpf(1.f, -e) : 1.f;
}

// ------------------------------------------------------------------------------------------------ dQ, delta
template <typename T, int DP, int RW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(xa_waves<T, DP>(RW)))) void k_xa_dq(XaArgs a) {
  constexpr int KW = 4 / RW, BN = KW == 4 ? 128 : 64, SUB = BN / 32 / KW;
  constexpr int KS = DP / 16, DT = DP / 32;
  typedef XaTile<T, DP> Tile;
  constexpr int TB = BN * Tile::LD;
  constexpr int JB = KW > 1 ? 4 * 32 * (DP + 1) * 4 : 0;
  constexpr int BYTES = 4 * TB > JB ? 4 * TB : JB;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l32 = lane & 31;
  const int rw = wave / KW, kw = wave % KW;
  const int hk = blockIdx.y;
  const int split = blockIdx.x % a.splits;
  const XaPlace f = xa_place(a, blockIdx.x / a.splits, RW * 32, false);
  if (f.tile < 0) return;
  const int rows = f.nq * a.group, row = f.tile * RW * 32 + rw * 32 + l32;
  const int tiles = (f.nk + BN - 1) / BN;
  const int t0 = (int)((long long)tiles * split / a.splits), t1 = (int)((long long)tiles * (split + 1) / a.splits);
  const bool live = row < rows;
  const int qi = live ? row / a.group : 0, head = hk * a.group + (live ? row - qi * a.group : 0);
  const long long at = (f.q0 + qi) * a.heads + head;
  const T* kbase = (const T*)a.k + f.k0 * a.sk + hk * a.hk;
  const T* vbase = (const T*)a.v + f.k0 * a.sv + hk * a.hv;
  typename XaFrag<T>::vec Q[KS], G[KS];
  // a frame of few keys: delta is formed below from the row's own P and dP, and is exact where the softmax has one key
  const bool few = f.nk <= 32;
  float delta = 0.f;
  {
    const T* p = (const T*)a.q + (f.q0 + qi) * a.sq + head * a.hq;
    const T* g = (const T*)a.go + (f.q0 + qi) * a.sg + head * a.hg;
    const T* o = (const T*)a.o + at * a.dim;
    const __bf16* rest = a.rest + at * a.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Q[s] = G[s] = typename XaFrag<T>::vec{};
      if (!live) continue;
      Q[s] = xa_row<T>(p, s * 16 + half * 8, a.dim);
      G[s] = xa_row<T>(g, s * 16 + half * 8, a.dim);
      const typename XaFrag<T>::vec x = xa_row<T>(o, s * 16 + half * 8, a.dim);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += (float)G[s][i] * (float)x[i];
      if (sizeof(T) == 2 && a.rest) {
        const XaFrag<__bf16>::vec y = xa_row<__bf16>(rest, s * 16 + half * 8, a.dim);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta += (float)G[s][i] * (float)y[i];
      }
    }
    delta += __shfl_xor(delta, 32, 64);
  }
  const float lse = live ? a.lse[at] : INFINITY;
  if (lse == INFINITY) delta = 0.f;                           // a row without keys: no gradient, whatever dO holds
  if (live && kw == 0 && half == 0 && split == 0 && !(few && lse != INFINITY)) a.delta[at] = delta;
  if (!a.dq && !few) return;
  xf16 D[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) D[i] = (xf16)(0.f);
  int e = 999;
  XaLoad<T, DP, BN> kl, vl;
  const bool kdma = a.dma & 2, vdma = a.dma & 4;
  auto koff = [&](int r) { return (long long)r * a.sk; };
  auto voff = [&](int r) { return (long long)r * a.sv; };
  kl.place(koff, a.dim);
  vl.place(voff, a.dim);
  unsigned long long ok[2] = {0, 0}, nok[2] = {0, 0};
  auto on = [&](int r) { return (bool)((nok[r >> 6] >> (r & 63)) & 1); };
  auto load = [&](int t, char* to) {
    const int k0 = t * BN, n = f.nk - k0;
#pragma unroll
    for (int h = 0; h < BN / 64; ++h) nok[h] = xa_valid(a.mask, f.k0 + k0 + h * 64, n - h * 64);
    kl.issue(to, kbase + (long long)k0 * a.sk, koff, on, n, a.dim, kdma);
    vl.issue(to + TB, vbase + (long long)k0 * a.sv, voff, on, n, a.dim, vdma);
  };
  // (masked products with the values are replaced, so only the keys' rows have to be clean)
  auto settle = [&](char* to) { kl.settle(to, on, nok[0] == ~0ull && nok[BN / 64 - 1] == ~0ull); };
  if (t0 < t1) {
    load(t0, smem);
    settle(smem);
  }
  ok[0] = nok[0]; ok[1] = nok[1];
  __syncthreads();
  int buf = 0;
  if (few && kw == 0 && t0 < t1 && (unsigned)ok[0]) {
    const unsigned valid = (unsigned)ok[0], mine = valid >> (half * 4);
    const bool one = (valid & (valid - 1)) == 0;
    xf16 s = (xf16)(0.f), d = (xf16)(0.f);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      xa_mma(s, xa_along<T, DP>(smem, l32, k, half), Q[k]);
      xa_mma(d, xa_along<T, DP>(smem + TB, l32, k, half), G[k]);
    }
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((mine >> ((i >> 2) * 8 + (i & 3))) & 1) {
        const float p = one ? 1.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse));
        x += p * d[i];
        y += p;
      }
    x += __shfl_xor(x, 32, 64);
    y += __shfl_xor(y, 32, 64);
    delta = y > 0.f ? x / y : 0.f;
    if (live && half == 0 && lse != INFINITY) a.delta[at] = delta;
  }
  for (int t = t0; t < t1; ++t) {
    const bool more = t + 1 < t1;
    char* next = smem + (buf ^ 1) * 2 * TB;
    if (more) load(t + 1, next);
    const char* tk = smem + buf * 2 * TB;
    const char* tv = tk + TB;
    {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int c0 = (u * KW + kw) * 32;
        const unsigned valid = (unsigned)(ok[c0 >> 6] >> (c0 & 63));
        if (!valid) continue;
        xf16 s = (xf16)(0.f), d = (xf16)(0.f);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          xa_mma(s, xa_along<T, DP>(tk, c0 + l32, k, half), Q[k]);
          xa_mma(d, xa_along<T, DP>(tv, c0 + l32, k, half), G[k]);
        }
        const unsigned mine = valid >> (half * 4);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse)) * (d[i] - delta);
          s[i] = (mine >> ((i >> 2) * 8 + (i & 3))) & 1 ? p : 0.f;
        }
        xa_range<T, DT>(s, D, e);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const typename XaFrag<T>::vec p = xa_pack<T>(s, c);
          if constexpr (sizeof(T) == 2 && DP == 32) {         // what the rounding of dS left (above)
            xf16 rest;
#pragma unroll
            for (int i = 0; i < 8; ++i) rest[i] = s[c * 8 + i] - (float)p[i];
            xa_mma(D[0], xa_down<T, DP>(tk, c0 + c * 16, 0, lane), xa_pack<T>(rest, 0));
          }
#pragma unroll
          for (int i = 0; i < DT; ++i) xa_mma(D[i], xa_down<T, DP>(tk, c0 + c * 16, i * 32, lane), p);
        }
      }
    }
    if (more) settle(next);
    ok[0] = nok[0]; ok[1] = nok[1];
    __syncthreads();
    buf ^= 1;
  }
  const float size = a.scale * xa_unrange<T>(e);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int k = 0; k < 16; ++k) D[i][k] *= size;
  if (KW > 1) {
    float* x = (float*)smem + wave * 32 * (DP + 1);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) x[l32 * (DP + 1) + i * 32 + (k >> 2) * 8 + half * 4 + (k & 3)] = D[i][k];
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float v = 0.f;
#pragma unroll
          for (int j = 0; j < KW; ++j) v += x[j * 32 * (DP + 1) + l32 * (DP + 1) + i * 32 + (k >> 2) * 8 + half * 4 + (k & 3)];
          D[i][k] = v;
        }
    }
  }
  if (!live || kw != 0 || !a.dq) return;
  float* part = a.part + ((long long)split * a.nq * a.heads + at) * a.dim;
  T* out = (T*)a.dq + at * a.dim;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = i * 32 + g * 8 + half * 4 + k;
        if (d >= a.dim) continue;
        if (a.splits > 1) part[d] = D[i][g * 4 + k];
        else out[d] = (T)D[i][g * 4 + k];
      }
}

// ------------------------------------------------------------------------------------------------ dK, dV
template <typename T, int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP == 32 ? 2 : 1))) void k_xa_dkv(XaArgs a) {
  constexpr int BM = sizeof(T) == 2 ? 64 : 32, PARTS = BM / 32;
  constexpr int KS = DP / 16, DT = DP / 32;
  typedef XaTile<T, DP> Tile;
  constexpr int TB = BM * Tile::LD;
  __shared__ __attribute__((aligned(16))) char smem[2 * 2 * TB];
  __shared__ __attribute__((aligned(16))) float srow[2][2][BM];         // stage; lse, delta
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l32 = lane & 31;
  const int hk = blockIdx.y;
  const int split = blockIdx.x % a.splits;
  const XaPlace f = xa_place(a, blockIdx.x / a.splits, 128, true);
  if (f.tile < 0) return;
  const int rows = f.nq * a.group, key = f.tile * 128 + wave * 32 + l32;
  const int step = a.group <= BM ? BM / a.group * a.group : BM, tiles = (rows + step - 1) / step;
  const int t0 = (int)((long long)tiles * split / a.splits), t1 = (int)((long long)tiles * (split + 1) / a.splits);
  const bool there = key < f.nk, valid = there && (!a.mask || a.mask[f.k0 + key] != 0);
  typename XaFrag<T>::vec K[KS], V[KS];
  {
    const T* k = (const T*)a.k + (f.k0 + key) * a.sk + hk * a.hk;
    const T* v = (const T*)a.v + (f.k0 + key) * a.sv + hk * a.hv;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      K[s] = V[s] = typename XaFrag<T>::vec{};
      if (!valid) continue;
      K[s] = xa_row<T>(k, s * 16 + half * 8, a.dim);
      V[s] = xa_row<T>(v, s * 16 + half * 8, a.dim);
    }
  }
  xf16 dK[DT], dV[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) dK[i] = dV[i] = (xf16)(0.f);
  int e = 999;
  XaLoad<T, DP, BM> ql, gl;
  const bool qdma = (a.dma & 1) && a.group <= BM, gdma = (a.dma & 8) && a.group <= BM;
  // a tile holds whole queries, so that a thread's rows are the same distance from every tile's first query
  auto qoff = [&](int r) {
    const int qi = r / a.group;
    return qi * a.sq + (r - qi * a.group) * a.hq;
  };
  auto goff = [&](int r) {
    const int qi = r / a.group;
    return qi * a.sg + (r - qi * a.group) * a.hg;
  };
  ql.place(qoff, a.dim);
  gl.place(goff, a.dim);
  float lse = INFINITY, delta = 0.f;
  int there_next = 0;                                          // rows of the tile on its way
  auto load = [&](int t, int buf) {
    const long long r0 = (long long)t * step;
    const int n = rows - r0 < step ? (int)(rows - r0) : step;
    there_next = n;
    auto on = [&](int r) { return r < n; };
    char* to = smem + buf * 2 * TB;
    const long long q0 = f.q0 + r0 / a.group;
    const int g0 = hk * a.group + (int)(r0 % a.group);        // (0 behind hk but for groups wider than a tile)
    // groups wider than a tile start within a query: their offsets are not those of `place`
    auto qwide = [&](int r) {
      const int qi = (int)((r0 + r) / a.group);
      return (qi - r0 / a.group) * a.sq + ((r0 + r - (long long)qi * a.group) - r0 % a.group) * a.hq;
    };
    auto gwide = [&](int r) {
      const int qi = (int)((r0 + r) / a.group);
      return (qi - r0 / a.group) * a.sg + ((r0 + r - (long long)qi * a.group) - r0 % a.group) * a.hg;
    };
    ql.issue(to, (const T*)a.q + q0 * a.sq + g0 * a.hq, qwide, on, n, a.dim, qdma);
    gl.issue(to + TB, (const T*)a.go + q0 * a.sg + g0 * a.hg, gwide, on, n, a.dim, gdma);
    lse = INFINITY; delta = 0.f;
    if ((int)threadIdx.x < n) {
      const long long r = r0 + threadIdx.x, qi = r / a.group;
      const long long at = (f.q0 + qi) * a.heads + hk * a.group + (r - qi * a.group);
      lse = a.lse[at]; delta = a.delta[at];
    }
  };
  auto settle = [&](int buf) {
    auto on = [&](int r) { return r < there_next; };
    char* to = smem + buf * 2 * TB;
    ql.settle(to, on, there_next == BM);
    gl.settle(to + TB, on, there_next == BM);
    if ((int)threadIdx.x < BM) { srow[buf][0][threadIdx.x] = lse; srow[buf][1][threadIdx.x] = delta; }
  };
  if (t0 < t1) { load(t0, 0); settle(0); }
  __syncthreads();
  int buf = 0;
  auto sweep = [&](auto masked) {
  constexpr bool MASKED = decltype(masked)::value;
  for (int t = t0; t < t1; ++t) {
    const bool more = t + 1 < t1;
    if (more) load(t + 1, buf ^ 1);
    const char* tq = smem + buf * 2 * TB;
    const char* tg = tq + TB;
    xf16 s[PARTS], d[PARTS];
    xf4 ls[4], de[4];
    auto stats = [&](int u) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        ls[g] = *reinterpret_cast<const xf4*>(&srow[buf][0][u * 32 + g * 8 + half * 4]);
        de[g] = *reinterpret_cast<const xf4*>(&srow[buf][1][u * 32 + g * 8 + half * 4]);
      }
    };
    auto weigh = [&](int u, int i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], a.scale2, -ls[i >> 2][i & 3]));
      const float q = p * (d[u][i] - de[i >> 2][i & 3]);
      s[u][i] = MASKED && !valid ? 0.f : __is_same(T, _Float16) ? p * XA_PSCALE : p;
      d[u][i] = MASKED && !valid ? 0.f : q;
    };
    // steps: the two score products of part u, k by k; its two gradient products, eight rows and 32 channels at a time.  Part u's
    // scores are weighed beside the products that follow them
    constexpr int GS = 2 * DT, STEPS = PARTS * (KS + GS);
    typename XaFrag<T>::vec ring[XA_AHEAD + 1][2];
    auto read = [&](int n) {
      const int r = n % (XA_AHEAD + 1);
      if (n < PARTS * KS) {
        const int row = n / KS * 32 + l32;
        ring[r][0] = xa_along<T, DP>(tq, row, n % KS, half);
        ring[r][1] = xa_along<T, DP>(tg, row, n % KS, half);
      } else {
        const int g = n - PARTS * KS, row = g / GS * 32 + g % GS / DT * 16;
        ring[r][0] = xa_down<T, DP>(tg, row, g % DT * 32, lane);
        ring[r][1] = xa_down<T, DP>(tq, row, g % DT * 32, lane);
      }
    };
#pragma unroll
    for (int n = 0; n < XA_AHEAD; ++n) read(n);
    typename XaFrag<T>::vec p, q;
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      const int r = n % (XA_AHEAD + 1);
      if (n + XA_AHEAD < STEPS) read(n + XA_AHEAD);
      if (n == (PARTS > 1 ? KS - 1 : 0)) stats(0);
      XA_STEP();
      if (n < PARTS * KS) {
        const int u = n / KS, k = n % KS;
        if (k == 0) s[u] = d[u] = (xf16)(0.f);
        xa_mma(s[u], ring[r][0], K[k]);
        xa_mma(d[u], ring[r][1], V[k]);
        if (u > 0) {
#pragma unroll
          for (int i = k * 16 / KS; i < (k + 1) * 16 / KS; ++i) weigh(u - 1, i);
        }
      } else {
        const int g = n - PARTS * KS, u = g / GS, j = g % GS;
        if (g == 0) {
          if (PARTS == 1) {
#pragma unroll
            for (int i = 0; i < 16; ++i) weigh(0, i);
          } else {
            stats(1);
          }
        }
        if (j == 0) xa_range<T, DT>(d[u], dK, e);
        if (j % DT == 0) { p = xa_pack<T>(s[u], j / DT); q = xa_pack<T>(d[u], j / DT); }
        xa_mma(dV[j % DT], ring[r][0], p);
        xa_mma(dK[j % DT], ring[r][1], q);
        if constexpr (sizeof(T) == 2 && DP == 32) {            // what their rounding left (above)
          xf16 x;
#pragma unroll
          for (int i = 0; i < 8; ++i) { x[i] = s[u][j / DT * 8 + i] - (float)p[i]; x[i + 8] = d[u][j / DT * 8 + i] - (float)q[i]; }
          xa_mma(dV[0], ring[r][0], xa_pack<T>(x, 0));
          xa_mma(dK[0], ring[r][1], xa_pack<T>(x, 1));
        }
        if (PARTS > 1 && u == 0) {
#pragma unroll
          for (int i = j * 16 / GS; i < (j + 1) * 16 / GS; ++i) weigh(PARTS - 1, i);
        }
      }
    }
    if (more) settle(buf ^ 1);
    __syncthreads();
    buf ^= 1;
  }
  };
  // (all waves of the block take the same way: they meet at the barriers inside)
  if (__syncthreads_and(valid)) sweep(std::false_type());
  else sweep(std::true_type());
  if (!there) return;
  const float ksize = a.scale * xa_unrange<T>(e), vsize = __is_same(T, _Float16) ? 1.f / XA_PSCALE : 1.f;
  const long long at = (f.k0 + key) * a.kvheads + hk, n = a.nk * a.kvheads * a.dim;
  float* pk = a.part + (long long)split * 2 * n + at * a.dim;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = i * 32 + g * 8 + half * 4 + k;
        if (d >= a.dim) continue;
        // (a masked state's weights are 0, but 0 times a gradient or a query that is no number is none either)
        const float x = valid ? dK[i][g * 4 + k] * ksize : 0.f, y = valid ? dV[i][g * 4 + k] * vsize : 0.f;
        if (a.splits > 1) {
          pk[d] = x; pk[n + d] = y;
        } else {
          if (a.dk) ((T*)a.dk)[at * a.dim + d] = (T)x;
          if (a.dv) ((T*)a.dv)[at * a.dim + d] = (T)y;
        }
      }
}

// out = the splits' sum, in order
template <typename T>
__global__ __launch_bounds__(256) void k_xa_sum(const float* __restrict__ part, long long n, long long step, int splits, T* __restrict__ out) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float v = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) v += part[s * step + i];
    out[i] = (T)v;
  }
}

// ------------------------------------------------------------------------------------------------ host
struct XaBackward { int rw, qsplits, ksplits; long long qtiles, ktiles; size_t delta, qpart, kpart, bytes; };
static XaBackward xa_backward_plan(const glx_attention* t) {
  XaBackward p;
  const int group = t->heads / t->kv_heads, fr = t->frames > 0 ? t->frames : 1;
  const bool counts = t->q_cnt != nullptr;
  const long long rows = t->q_rows * group / fr;
  xa_rows_plan(t, &p.rw, &p.qtiles, &p.qsplits);
  p.ktiles = xa_tiles(t->k_rows, t->frames, (int)t->k_len, counts, 128);
  p.ksplits = xa_splits((counts ? t->k_rows / 128 + 1 : p.ktiles) * t->kv_heads, rows, 2);
  p.delta = 0;
  p.qpart = glx_align((size_t)t->q_rows * t->heads * sizeof(float));
  p.kpart = p.qpart + (p.qsplits > 1 ? glx_align((size_t)p.qsplits * t->q_rows * t->heads * t->dim * sizeof(float)) : 0);
  p.bytes = p.kpart + (p.ksplits > 1 ? glx_align((size_t)p.ksplits * 2 * t->k_rows * t->kv_heads * t->dim * sizeof(float)) : 0);
  return p;
}
extern "C" size_t glx_attention_backward_workspace_bytes(const glx_attention* t) {
  if (xa_check("glx_attention_backward_workspace_bytes", t) != GLX_OK) return 0;
  return xa_backward_plan(t).bytes + 256;
}

template <typename T, int DP>
static void xa_launch_backward(const XaBackward& p, XaArgs& a, char* ws, hipStream_t st) {
  if (p.qtiles) {
    const dim3 grid((unsigned)(p.qtiles * p.qsplits), a.kvheads);
    a.splits = p.qsplits;
    a.part = (float*)(ws + p.qpart);
    constexpr int SMALL = sizeof(T) == 4 && DP > 64 ? 2 : 1;
    if (p.rw == SMALL) hipLaunchKernelGGL((k_xa_dq<T, DP, SMALL>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_xa_dq<T, DP, 4>), grid, dim3(256), 0, st, a);
    if (a.dq && p.qsplits > 1) {
      const long long n = a.nq * a.heads * a.dim, blocks = (n + 1023) / 1024;
      hipLaunchKernelGGL((k_xa_sum<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, a.part, n, n, p.qsplits, (T*)a.dq);
    }
  }
  if (p.ktiles && (a.dk || a.dv)) {
    a.splits = p.ksplits;
    a.part = (float*)(ws + p.kpart);
    hipLaunchKernelGGL((k_xa_dkv<T, DP>), dim3((unsigned)(p.ktiles * p.ksplits), a.kvheads), dim3(256), 0, st, a);
    if (p.ksplits > 1) {
      const long long n = a.nk * a.kvheads * a.dim, blocks = (n + 1023) / 1024;
      const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
      if (a.dk) hipLaunchKernelGGL((k_xa_sum<T>), grid, dim3(256), 0, st, a.part, n, 2 * n, p.ksplits, (T*)a.dk);
      if (a.dv) hipLaunchKernelGGL((k_xa_sum<T>), grid, dim3(256), 0, st, a.part + n, n, 2 * n, p.ksplits, (T*)a.dv);
    }
  }
}
template <typename T>
static void xa_backward_of(const XaBackward& p, XaArgs& a, char* ws, hipStream_t st) {
  if (a.dim <= 32) xa_launch_backward<T, 32>(p, a, ws, st);
  else if (a.dim <= 64) xa_launch_backward<T, 64>(p, a, ws, st);
  else if (a.dim <= 96) xa_launch_backward<T, 96>(p, a, ws, st);
  else xa_launch_backward<T, 128>(p, a, ws, st);
}

extern "C" int glx_attention_backward(const glx_attention* t, const void* grad_out, int64_t g_stride, int64_t g_head_stride,
                                      void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = xa_check("glx_attention_backward", t)) return rc;
  GLX_REQUIRE(t->q_rows == 0 || (grad_out && t->lse), "glx_attention_backward: null gradient or lse");
  const XaBackward p = xa_backward_plan(t);
  if (!workspace || workspace_bytes < p.bytes) {
    glx_set_error("glx_attention_backward: workspace %zu < %zu bytes", workspace_bytes, p.bytes);
    return GLX_EWORKSPACE;
  }
  GLX_REQUIRE(p.qtiles * p.qsplits < (1ll << 31) && p.ktiles * p.ksplits < (1ll << 31), "glx_attention_backward: too many rows");
  XaArgs a = xa_args(t);
  a.go = grad_out; a.sg = g_stride; a.hg = g_head_stride;
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.dma |= xa_chunked(grad_out, g_stride, g_head_stride, a.dim, t->dtype) << 3;
  a.delta = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  if (t->dtype == GLX_F32) xa_backward_of<float>(p, a, (char*)workspace, st);
  else if (t->dtype == GLX_BF16) xa_backward_of<__bf16>(p, a, (char*)workspace, st);
  else xa_backward_of<_Float16>(p, a, (char*)workspace, st);
  GLX_LAUNCH_CHECK();
  return GLX_OK;
}
