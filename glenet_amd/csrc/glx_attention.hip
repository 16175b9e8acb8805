// Cross attention of stacked frames, forward (glenet_amd/attention.py; the layouts: glx_attention.h).
//
//   O = softmax(scale Q K^T) V over a frame's unmasked keys, one pass over the keys with a running maximum and sum per row:
//   S^T = K Q^T (a lane owns a row's scores), p = 2^(s - m), O^T <- O^T 2^(m_old - m) + V^T p.  A row without keys gives 0.
//
// A block is four waves: four tiles of 32 rows that share the staged keys, or, where a frame has few rows, ONE tile whose
// waves take the staged keys in turn and are joined at the end.  Few tiles are split over the keys as well; the splits' results
// (O unnormalised, m, l) are joined by a second launch.  Scores, m, l and O are fp32; for 16-bit inputs p is rounded to their
// type in front of the second product (each to half a step, unbiased: together with the rounding of O 1.4 times the error that O's
// alone leaves).  O is divided by the sum of the ROUNDED p -- a row that one key dominates is then as exact as that key's value --
// and the log-sum-exp, from which the backward pass forms p again in fp32, is that of the unrounded ones.  Few rows, whose time is
// the keys' way from memory, take what the rounding left in a second product (one query over 4 x 32768, bf16: 2.3e-3 off, then
// 1.7e-3, 114.6 us both); with four row tiles it would cost 5 to 7 % (2 x 4096 x 16384, 128 channels: 2.71 -> 2.84 ms a training
// pass; 6 x 217 x 1531, 40 channels: 27.5 -> 29.4 us).
//
// 2 frames of 4096 queries over 16384 keys, 8 heads of 128 on 2 key heads, bf16: 734 us (749 TFLOP/s; a large library product
// reaches 1156).  Of a SIMD's cycles products take 35 % and vector instructions 54 % (ten per product: an exponential, its argument,
// the maximum, the sum, the rounding), so that they mostly take turns.  One query over each of 4 x 32768 keys, 32 heads on 8: 108 us
// (5.0 TB/s of keys and values) and 5 us for the join.
#include "glx_attention.h"

template <typename T, int DP, int RW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(xa_waves<T, DP>(RW)))) void k_xa_forward(XaArgs a) {
  constexpr int KW = 4 / RW, BN = KW == 4 ? 128 : 64, SUB = BN / 32 / KW;          // keys of a staged tile, of them 32 SUB a wave's
  constexpr int KS = DP / 16, DT = DP / 32;
  typedef XaTile<T, DP> Tile;
  constexpr int TB = BN * Tile::LD;
  constexpr int JB = KW > 1 ? 4 * 32 * (DP + 1) * 4 : 0;
  constexpr int BYTES = 4 * TB > JB ? 4 * TB : JB;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  __shared__ float sm[4][32], sl[4][32], slr[4][32];
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
  const T* kbase = (const T*)a.k + f.k0 * a.sk + hk * a.hk;
  const T* vbase = (const T*)a.v + f.k0 * a.sv + hk * a.hv;
  typename XaFrag<T>::vec Q[KS];
  {
    const T* p = (const T*)a.q + (f.q0 + qi) * a.sq + head * a.hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Q[s] = typename XaFrag<T>::vec{};
      if (live) Q[s] = xa_row<T>(p, s * 16 + half * 8, a.dim);
      if (a.scale2 < 0.f) Q[s] = -Q[s];                      // the maximum is taken of unscaled scores
    }
  }
  xf16 O[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) O[i] = (xf16)(0.f);
  const float scale2 = fabsf(a.scale2);
  // fp16 ends at 2^-25: beside a key of weight 1 the many small ones of a long row would vanish (131 072 of 2^-25.4 are 3e-3 of it).
  // So p is formed 2^11 times as large, and m lags by 2^4 at most: up to 2^15, down to 2^-36 of a row's largest
  constexpr bool FP16 = __is_same(T, _Float16);
  constexpr float UP = FP16 ? 11.f : 0.f, LAG = FP16 ? 4.f : 8.f;
  float m = -INFINITY, l = 0.f, lr = 0.f;                     // m unscaled; sums of p, of the rounded p (16-bit)
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
  // (masked scores are replaced, so only the values' rows have to be clean; a key of -infinity is one of weight 0)
  auto settle = [&](char* to) {
    vl.settle(to + TB, on, nok[0] == ~0ull && nok[BN / 64 - 1] == ~0ull);
    if (kdma && a.dim < DP) kl.trim(to, a.dim);
  };
  if (t0 < t1) {
    load(t0, smem);
    settle(smem);
  }
  ok[0] = nok[0]; ok[1] = nok[1];
  __syncthreads();
  int buf = 0;
  for (int t = t0; t < t1; ++t) {
    const bool more = t + 1 < t1;
    char* next = smem + (buf ^ 1) * 2 * TB;
    if (more) load(t + 1, next);
    const char* tk = smem + buf * 2 * TB;
    const char* tv = tk + TB;
    unsigned valid[SUB];
    bool some = false, every = true;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const int c0 = (u * KW + kw) * 32;                      // first of this wave's 32 keys
      valid[u] = (unsigned)(ok[c0 >> 6] >> (c0 & 63));
      some |= valid[u] != 0;
      every &= valid[u] == 0xffffffffu;
    }
    if (some) {
      xf16 s[SUB];
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        s[u] = (xf16)(0.f);
#pragma unroll
        for (int k = 0; k < KS; ++k) xa_mma(s[u], xa_along<T, DP>(tk, (u * KW + kw) * 32 + l32, k, half), Q[k]);
      }
      if (!every) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((valid[u] >> (half * 4 + (i >> 2) * 8 + (i & 3))) & 1)) s[u][i] = -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // m follows the maximum only where p would pass 2^LAG: then O and l shrink, else the tile is added as it is
      if (__any((top - m) * scale2 > LAG || m == -INFINITY)) {
        const float now = fmaxf(m, top), shrink = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - now) * scale2);
        m = now;
        l *= shrink;
        lr *= shrink;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) O[i][e] *= shrink;
      }
      // (16-bit: one fused operation; its rounding of m scale2 is a factor that p and l share.  fp32 keeps 2^0 = 1 exactly)
      const float ref = m == -INFINITY ? 0.f : m, at = ref * scale2 - UP;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[u][i] = __builtin_amdgcn_exp2f(sizeof(T) == 2 ? __builtin_fmaf(s[u][i], scale2, -at) : (s[u][i] - ref) * scale2);
          if (!every && scale2 == 0.f && !((valid[u] >> (half * 4 + (i >> 2) * 8 + (i & 3))) & 1)) s[u][i] = 0.f;
          sum += s[u][i];
        }
        l += sum;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const typename XaFrag<T>::vec p = xa_pack<T>(s[u], c);
          if constexpr (KW > 1 && sizeof(T) == 2) {            // and what the rounding left
            xf16 rest;
#pragma unroll
            for (int i = 0; i < 8; ++i) rest[i] = s[u][c * 8 + i] - (float)p[i];
            const typename XaFrag<T>::vec r = xa_pack<T>(rest, 0);
#pragma unroll
            for (int i = 0; i < DT; ++i) {
              const typename XaFrag<T>::vec v = xa_down<T, DP>(tv, (u * KW + kw) * 32 + c * 16, i * 32, lane);
              xa_mma(O[i], v, r);
              xa_mma(O[i], v, p);
            }
          } else {
            lr = xa_total(p, lr);
#pragma unroll
            for (int i = 0; i < DT; ++i) xa_mma(O[i], xa_down<T, DP>(tv, (u * KW + kw) * 32 + c * 16, i * 32, lane), p);
          }
        }
      }
    }
    if (more) settle(next);
    ok[0] = nok[0]; ok[1] = nok[1];
    __syncthreads();
    buf ^= 1;
  }
  l += __shfl_xor(l, 32, 64);
  if (sizeof(T) == 2 && KW == 1) lr += __shfl_xor(lr, 32, 64);
  else lr = l;
  m = m == -INFINITY ? m : m * scale2 - UP;                   // l and O are sums of 2^(s scale2 - m)
  if (KW > 1) {                                               // the waves of a row tile, joined in order
    if (half == 0) { sm[wave][l32] = m; sl[wave][l32] = l; slr[wave][l32] = lr; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < KW; ++i) top = fmaxf(top, sm[rw * KW + i][l32]);
    const float at = top == -INFINITY ? 0.f : top;
    float* x = (float*)smem + wave * 32 * (DP + 1);
    const float w = __builtin_amdgcn_exp2f(m - at);
    float all = 0.f, allr = 0.f;
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const float u = exp2f(sm[rw * KW + i][l32] - at);
      all += sl[rw * KW + i][l32] * u;
      allr += slr[rw * KW + i][l32] * u;
    }
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[l32 * (DP + 1) + i * 32 + (e >> 2) * 8 + half * 4 + (e & 3)] = O[i][e] * w;
    __syncthreads();
    m = top; l = all; lr = allr;
    if (kw == 0) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float v = 0.f;
#pragma unroll
          for (int j = 0; j < KW; ++j)
            v += x[j * 32 * (DP + 1) + l32 * (DP + 1) + i * 32 + (e >> 2) * 8 + half * 4 + (e & 3)];
          O[i][e] = v;
        }
    }
  }
  if (!live || kw != 0) return;
  const long long at = (f.q0 + qi) * a.heads + head;
  if (a.splits > 1) {
    float* part = a.part + ((long long)split * a.nq * a.heads + at) * (a.dim + 3);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = i * 32 + (e >> 2) * 8 + half * 4 + (e & 3);
        if (d < a.dim) part[3 + d] = O[i][e];
      }
    if (half == 0) { part[0] = m; part[1] = l; part[2] = lr; }
    return;
  }
  const float inv = lr == 0.f ? 0.f : 1.f / lr;
  T* out = (T*)a.out + at * a.dim;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + half * 4;
      typename GlxVec<T, 4>::vec v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(O[i][g * 4 + e] * inv);
      if (d + 4 <= a.dim) GlxVec<T, 4>::store(out + d, v);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < a.dim) out[d + e] = v[e];
      if (sizeof(T) == 2 && a.rest) {
        __bf16* rest = a.rest + at * a.dim;
        GlxVec<__bf16, 4>::vec w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (__bf16)(O[i][g * 4 + e] * inv - (float)v[e]);
        if (d + 4 <= a.dim) GlxVec<__bf16, 4>::store(rest + d, w);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.dim) rest[d + e] = w[e];
      }
    }
  if (a.lse && half == 0) a.lse[at] = l == 0.f ? INFINITY : m + log2f(l);
}

// the splits of a row: one wave per row
template <typename T>
__global__ __launch_bounds__(256) void k_xa_join(XaArgs a) {
  const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), rows = a.nq * a.heads;
  const int lane = threadIdx.x & 63;
  if (at >= rows) return;
  const long long step = rows * (a.dim + 3);
  const float* part = a.part + at * (a.dim + 3);
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, part[s * step]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float base = top == -INFINITY ? 0.f : top;
  float l = 0.f, lr = 0.f;
  for (int s = lane; s < a.splits; s += 64) {
    const float u = exp2f(part[s * step] - base);
    l += part[s * step + 1] * u;
    lr += part[s * step + 2] * u;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { l += __shfl_xor(l, o, 64); lr += __shfl_xor(lr, o, 64); }
  const float inv = lr == 0.f ? 0.f : 1.f / lr;
  for (int d = lane; d < a.dim; d += 64) {
    float v = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) v += part[s * step + 3 + d] * exp2f(part[s * step] - base);
    const T o = (T)(v * inv);
    ((T*)a.out)[at * a.dim + d] = o;
    if (sizeof(T) == 2 && a.rest) a.rest[at * a.dim + d] = (__bf16)(v * inv - (float)o);
  }
  if (a.lse && lane == 0) a.lse[at] = l == 0.f ? INFINITY : top + log2f(l);
}

// ------------------------------------------------------------------------------------------------ host
// one round of blocks on 256 compute units that hold `per_cu` each (two rounds of half the keys, 4 x 128 queries over 2048 states,
// fp32, 4 heads of 64, training: 134 us instead of 122; one query over 4 x 32768, bf16: 120 instead of 115)
int xa_splits(long long blocks, long long keys_per_frame, int per_cu) {
  if (blocks < 1) blocks = 1;
  long long s = 256 * per_cu / blocks, most = keys_per_frame / 256;        // 256 keys a split, at least
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}
// row tiles of four waves, or of one (two: fp32 heads beyond 64, the keys of four waves do not fit LDS twice) where the large
// ones would leave compute units without work even when the keys are split; `rw`, tiles, splits over `keys` states per frame
void xa_rows_plan(const glx_attention* t, int* rw, long long* tiles, int* splits) {
  const int group = t->heads / t->kv_heads, fr = t->frames > 0 ? t->frames : 1, small = t->dtype == GLX_F32 && t->dim > 64 ? 2 : 1;
  const bool counts = t->q_cnt != nullptr;
  const long long keys = t->k_rows / fr, rows = t->q_rows * group;
  for (*rw = 4;; *rw = small) {
    *tiles = xa_tiles(rows, t->frames, (int)(t->q_len * group), counts, *rw * 32);
    const long long blocks = (counts ? rows / (*rw * 32) + 1 : *tiles) * t->kv_heads;
    const long long lds = 4ll * (*rw == 1 ? 128 : 64) * ((t->dim + 31) / 32 * 32) * (long long)glx_elem_size(t->dtype);
    *splits = xa_splits(blocks, keys, lds <= 80 * 1024 ? 2 : 1);
    if (*rw == small || (rows > 64 * fr && blocks * *splits >= 256)) return;
  }
}
struct XaForward { int rw, splits; long long tiles; };
static XaForward xa_forward_plan(const glx_attention* t) {
  XaForward p;
  xa_rows_plan(t, &p.rw, &p.tiles, &p.splits);
  return p;
}

int xa_check(const char* who, const glx_attention* t) {
  GLX_REQUIRE(t, "%s: null descriptor", who);
  GLX_REQUIRE(glx_elem_ok(t->dtype), "%s: dtype %d", who, t->dtype);
  GLX_REQUIRE(t->frames >= 0 && t->q_rows >= 0 && t->k_rows >= 0 && t->heads >= 1 && t->kv_heads >= 1, "%s: negative sizes", who);
  GLX_REQUIRE(t->heads % t->kv_heads == 0, "%s: %d heads over %d key heads", who, t->heads, t->kv_heads);
  GLX_REQUIRE(t->dim >= 1 && t->dim <= 128, "%s: head dimension %d (1 .. 128)", who, t->dim);
  GLX_REQUIRE(t->kv_heads <= 65535 && t->q_rows * t->heads < (1ll << 31) && t->k_rows * t->kv_heads < (1ll << 31), "%s: too many rows", who);
  GLX_REQUIRE(!t->q_cnt == !t->k_cnt, "%s: counts of one side only", who);
  GLX_REQUIRE(t->q_cnt || (t->q_len >= 0 && t->k_len >= 0 && t->q_len * t->frames == t->q_rows && t->k_len * t->frames == t->k_rows),
              "%s: %d frames of %lld queries and %lld keys do not fill the tensors", who, t->frames, (long long)t->q_len, (long long)t->k_len);
  GLX_REQUIRE(t->q_rows == 0 || (t->q && t->out), "%s: null queries or output", who);
  GLX_REQUIRE(t->k_rows == 0 || (t->k && t->v), "%s: null keys or values", who);
  return GLX_OK;
}
XaArgs xa_args(const glx_attention* t) {
  XaArgs a = {};
  a.q = t->q; a.k = t->k; a.v = t->v; a.out = t->out; a.o = t->out; a.lse = t->lse; a.rest = (__bf16*)t->out_rest; a.mask = t->key_mask;
  a.qcnt = t->q_cnt; a.kcnt = t->k_cnt;
  a.sq = t->q_stride; a.hq = t->q_head_stride; a.sk = t->k_stride; a.hk = t->k_head_stride; a.sv = t->v_stride; a.hv = t->v_head_stride;
  a.nq = t->q_rows; a.nk = t->k_rows;
  a.frames = t->frames; a.lq = (int)t->q_len; a.lk = (int)t->k_len; a.heads = t->heads; a.kvheads = t->kv_heads;
  a.group = t->heads / t->kv_heads; a.dim = t->dim; a.splits = 1;
  a.dma = xa_chunked(t->q, a.sq, a.hq, a.dim, t->dtype) | xa_chunked(t->k, a.sk, 0, a.dim, t->dtype) << 1
          | xa_chunked(t->v, a.sv, 0, a.dim, t->dtype) << 2;
  if (a.hk * glx_elem_size(t->dtype) % 16) a.dma &= ~2;
  if (a.hv * glx_elem_size(t->dtype) % 16) a.dma &= ~4;
  a.scale = t->scale; a.scale2 = t->scale * 1.4426950408889634f;
  return a;
}

extern "C" size_t glx_attention_workspace_bytes(const glx_attention* t) {
  if (xa_check("glx_attention_workspace_bytes", t) != GLX_OK) return 0;
  const XaForward p = xa_forward_plan(t);
  return glx_align(p.splits > 1 ? (size_t)p.splits * t->q_rows * t->heads * (t->dim + 3) * sizeof(float) : 0) + 256;
}

template <typename T, int DP>
static void xa_launch_forward(const XaForward& p, const XaArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(p.tiles * p.splits), a.kvheads);
  constexpr int SMALL = sizeof(T) == 4 && DP > 64 ? 2 : 1;
  if (p.rw == SMALL) hipLaunchKernelGGL((k_xa_forward<T, DP, SMALL>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_xa_forward<T, DP, 4>), grid, dim3(256), 0, st, a);
}
template <typename T>
static void xa_forward_of(const XaForward& p, const XaArgs& a, hipStream_t st) {
  if (a.dim <= 32) xa_launch_forward<T, 32>(p, a, st);
  else if (a.dim <= 64) xa_launch_forward<T, 64>(p, a, st);
  else if (a.dim <= 96) xa_launch_forward<T, 96>(p, a, st);
  else xa_launch_forward<T, 128>(p, a, st);
  if (p.splits > 1) hipLaunchKernelGGL((k_xa_join<T>), dim3((unsigned)((a.nq * a.heads + 3) / 4)), dim3(256), 0, st, a);
}

extern "C" int glx_attention_forward(const glx_attention* t, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = xa_check("glx_attention_forward", t)) return rc;
  if (t->q_rows == 0) return GLX_OK;
  const XaForward p = xa_forward_plan(t);
  XaArgs a = xa_args(t);
  a.splits = p.splits;
  a.part = (float*)workspace;
  if (p.splits > 1 && (!workspace || workspace_bytes < glx_attention_workspace_bytes(t) - 256)) {
    glx_set_error("glx_attention_forward: workspace %zu < %zu bytes", workspace_bytes, glx_attention_workspace_bytes(t));
    return GLX_EWORKSPACE;
  }
  GLX_REQUIRE(p.tiles * p.splits < (1ll << 31), "glx_attention_forward: too many rows");
  hipStream_t st = (hipStream_t)stream;
  if (t->dtype == GLX_F32) xa_forward_of<float>(p, a, st);
  else if (t->dtype == GLX_BF16) xa_forward_of<__bf16>(p, a, st);
  else xa_forward_of<_Float16>(p, a, st);
  GLX_LAUNCH_CHECK();
  return GLX_OK;
}
