// Cross attention of stacked frames: what the forward and backward kernels share (glx_attention.hip, glx_attention_bwd.hip).
//
// Queries (Nq, H, D) and encoder states (Nk, Hkv, D) of B frames lie behind each other; a frame's counts come from device
// memory or are the same for all frames.  The G = H / Hkv query heads that share a key head are ROWS beside each other: row
// r of a frame and key head is query r / G, head hk G + r % G.  So a single query with shared heads still fills a tile, and the
// gradients of shared keys are sums over rows like any other.
//
// All products run on 32 x 32 MFMA tiles in one register layout.  A product C = A B leaves lane (l32, half) with column l32 and
// rows 8 (i / 4) + 4 half + i % 4 (i = 0..15) of C.  Eight consecutive i are a B operand of the next product whose k index runs
// in that order, so scores turn into probabilities and into the next operand without leaving the lane; the other operand is
// read from LDS in the same k order (16-bit: the transposing read; 32-bit: plain reads).
#pragma once
#include "glx_elem.h"

#define XA_KEYS 64            // keys of a staged tile

typedef float xf16 __attribute__((ext_vector_type(16)));
typedef float xf4 __attribute__((ext_vector_type(4)));
typedef short xs4 __attribute__((ext_vector_type(4)));
typedef short xs8 __attribute__((ext_vector_type(8)));

struct XaArgs {
  const void *q, *k, *v, *o, *go;
  void *out, *dq, *dk, *dv;
  __bf16 *rest;                     // (Nq, H, D) what the rounding of a 16-bit out left, or NULL
  float *lse, *delta;               // (Nq, H); lse in base 2, +inf where no key is left
  float *part;                      // splits' partial results
  const unsigned char* mask;        // (Nk) or NULL
  const int *qcnt, *kcnt;           // (B) or NULL: Lq, Lk
  long long sq, hq, sk, hk, sv, hv, sg, hg;      // elements between rows and between heads of q, k, v, go
  long long nq, nk;
  int frames, lq, lk, heads, kvheads, group, dim, splits;
  int dma;                          // bits: rows of q, k, v, go are whole 16-byte chunks
  float scale, scale2;              // scale2 = scale log2(e)
};

// waves per SIMD that the registers are kept for: two where LDS holds two blocks (else the compiler takes all 512 for one)
template <typename T, int DP>
constexpr int xa_waves(int row_waves) {
  return 4 * (row_waves == 1 ? 128 : 64) * DP * (int)sizeof(T) <= 80 * 1024 ? 2 : 1;
}

// ------------------------------------------------------------------------------------------------ operands
template <typename T> struct XaFrag { typedef T vec __attribute__((ext_vector_type(8))); };

__device__ __forceinline__ void xa_mma(xf16& c, const XaFrag<__bf16>::vec& a, const XaFrag<__bf16>::vec& b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void xa_mma(xf16& c, const XaFrag<_Float16>::vec& a, const XaFrag<_Float16>::vec& b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void xa_mma(xf16& c, const XaFrag<float>::vec& a, const XaFrag<float>::vec& b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
}

// A staged tile: rows of DP values without padding, the 16-byte chunks of a row in an order of the row's own.  Reads along the
// rows take one chunk of 16 consecutive rows at a time, transposing reads four chunks (64 bytes) of 4 consecutive rows: chunk c
// of row r lies at c ^ swap(r) so that both cover all 64 banks.  (Rows padded by 16 bytes left the transposing reads with
// four-way conflicts: dK and dV of 4096 x 16384, 2 x 8 heads of 128, bf16, 2271 us instead of 1831.)
template <typename T, int DP> struct XaTile {
  static constexpr int LD = DP * (int)sizeof(T), E = 16 / (int)sizeof(T), CPR = DP / E;
  static __device__ __forceinline__ int swap(int r) {
    if (sizeof(T) == 4) return DP % 64 == 0 ? r & 15 : (r >> 1) & 7;
    return ((r >> 2) & 3) ^ (DP == 128 ? (r & 3) << 2 : DP == 64 ? (r & 2) << 1 : 0);
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * LD + (c ^ swap(r)) * 16; }
};

// eight values along a row: the operand whose k index is d; row = l32, k = 16 ks + 8 half + 0..7
template <typename T, int DP>
__device__ __forceinline__ typename XaFrag<T>::vec xa_along(const char* tile, int row, int ks, int half) {
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const typename XaFrag<T>::vec*>(tile + XaTile<T, DP>::at(row, ks * 2 + half));
  } else {
    const xf4 a = *reinterpret_cast<const xf4*>(tile + XaTile<T, DP>::at(row, ks * 4 + half * 2));
    const xf4 b = *reinterpret_cast<const xf4*>(tile + XaTile<T, DP>::at(row, ks * 4 + half * 2 + 1));
    return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
}
// eight values down the rows row0 + 4 half + {0..3, 8..11}, column d0 + l32: the operand whose k index is the row
template <typename T, int DP>
__device__ __forceinline__ typename XaFrag<T>::vec xa_down(const char* tile, int row0, int d0, int lane) {
  typedef XaTile<T, DP> Tile;
  const int half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    // a 16-lane group reads 4 rows x 16 columns and every lane gets a column's four values
    typedef xs4 __attribute__((address_space(3))) * lds_p;
    const int row = row0 + half * 4 + ((lane >> 2) & 3), c = d0 / 8 + ((lane >> 3) & 2) + ((lane >> 1) & 1), b = (lane & 1) * 8;
    const xs4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(tile + Tile::at(row, c) + b));
    const xs4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(tile + Tile::at(row + 8, c) + b));
    const xs8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(typename XaFrag<T>::vec, v);
  } else {
    const int c = (d0 + (lane & 31)) >> 2, b = (lane & 3) * 4;
    typename XaFrag<T>::vec v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float*>(tile + Tile::at(row0 + half * 4 + (i >> 2) * 8 + (i & 3), c) + b);
    return v;
  }
}
// + the sum of an operand's eight values
__device__ __forceinline__ float xa_total(const XaFrag<__bf16>::vec& p, float l) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const b2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2_f32_bf16(b2{p[i], p[i + 1]}, one, l, false);
  return l;
}
__device__ __forceinline__ float xa_total(const XaFrag<_Float16>::vec& p, float l) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
  for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2(h2{p[i], p[i + 1]}, one, l, false);
  return l;
}
__device__ __forceinline__ float xa_total(const XaFrag<float>::vec&, float l) { return l; }
// accumulators 8 c .. 8 c + 7 as an operand
template <typename T>
__device__ __forceinline__ typename XaFrag<T>::vec xa_pack(const xf16& s, int c) {
  typename XaFrag<T>::vec v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)s[c * 8 + i];
  return v;
}
// eight values of a row in global memory, d = 16 ks + 8 half .., zeros beyond D
template <typename T>
__device__ __forceinline__ typename XaFrag<T>::vec xa_row(const T* p, int d, int D) {
  if (d + 8 <= D) return GlxVec<T, 8>::load(p + d);
  typename XaFrag<T>::vec v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = d + i < D ? p[d + i] : (T)0.f;
  return v;
}

// The compiler places an operand's read in front of its product and waits for it there; with one or two waves per SIMD that
// leaves the matrix units idle most of the time.  So the loops below are written as steps -- one or two products, the reads for
// the step XA_AHEAD later, a share of the exponentials -- that are not reordered among each other.
#define XA_AHEAD 2
#define XA_STEP() __builtin_amdgcn_sched_barrier(0)

// ------------------------------------------------------------------------------------------------ staging
// ROWS rows of a tensor into a tile.  Rows that are whole 16-byte chunks go straight from memory to LDS (no registers, no LDS
// writes; a lane fetches the chunk that belongs at its place): `place` keeps the thread's offsets within a tile, `issue` starts the
// transfers of the rows below n and lets the places behind them repeat the last one, `settle` waits for the thread's own transfers
// and clears the places of rows that are not there or masked -- so those never reach a product, whatever they hold.  Other rows
// take the way through registers, element by element where they are ragged.  rowoff(r): elements from the tile's base to row r.
template <typename T, int DP, int ROWS>
struct XaLoad {
  static constexpr int E = XaTile<T, DP>::E, CPR = XaTile<T, DP>::CPR, N = ROWS * CPR / 256;
  static_assert(ROWS * CPR % 256 == 0, "whole rounds of the block");
  typedef typename GlxVec<T, E>::vec vec;
  int off[N];                 // bytes
  static __device__ __forceinline__ int row_of(int i) { return ((int)threadIdx.x + i * 256) / CPR; }
  static __device__ __forceinline__ int chunk_of(int i) {
    const int r = row_of(i);
    return ((int)threadIdx.x + i * 256 - r * CPR) ^ XaTile<T, DP>::swap(r);
  }
  template <typename F>
  __device__ __forceinline__ void place(F rowoff, int D) {
#pragma unroll
    for (int i = 0; i < N; ++i) off[i] = (int)((rowoff(row_of(i)) + (chunk_of(i) * E < D ? chunk_of(i) * E : 0)) * (int)sizeof(T));
  }
  template <typename F, typename V>
  __device__ __forceinline__ void issue(char* tile, const T* base, F rowoff, V valid, int n, int D, bool dma) const {
    if (dma) {
      const unsigned to = (unsigned)(unsigned long long)(const __attribute__((address_space(3))) char*)tile + (threadIdx.x >> 6) * 1024;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int o = off[i];
        if (n < ROWS) {
          const int r = row_of(i) < n ? row_of(i) : n - 1, c = chunk_of(i) * E < D ? chunk_of(i) * E : 0;
          o = (int)((rowoff(r) + c) * (int)sizeof(T));
        }
        // (no register is written, and the compiler, which would wait for all transfers in front of any transposing read, does
        // not see them: `settle` waits.  64 lanes x 16 bytes from base + o to LDS at the wave's place.)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     ::"v"(o), "s"(base), "s"(__builtin_amdgcn_readfirstlane(to + i * 4096))
                     : "memory");
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        const int r = row_of(i), d = chunk_of(i) * E;
        vec v = {};
        if (r < n && valid(r)) {
          const T* p = base + rowoff(r) + d;
          if (d + E <= D) {
            v = GlxVec<T, E>::load(p);
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (d + e < D) v[e] = p[e];
          }
        }
        *reinterpret_cast<vec*>(tile + (threadIdx.x + i * 256) * 16) = v;
      }
    }
  }
  template <typename V>
  __device__ __forceinline__ void settle(char* tile, V valid, bool all) const {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (all) return;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!valid(row_of(i))) *reinterpret_cast<vec*>(tile + (threadIdx.x + i * 256) * 16) = vec{};
  }
  // behind `settle`, of rows that came straight from memory: clears the channels from D on, which repeat the row's first ones.  A
  // product's zeros on the other side make nothing of them unless they are infinite
  __device__ __forceinline__ void trim(char* tile, int D) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (chunk_of(i) * E >= D) *reinterpret_cast<vec*>(tile + (threadIdx.x + i * 256) * 16) = vec{};
  }
};

// ------------------------------------------------------------------------------------------------ frames
struct XaPlace { long long q0, k0; int nq, nk, tile; };      // tile: index within the frame, -1: nothing there

// which frame holds the tile `t` when every frame has ceil(size / unit) tiles, size = its rows (queries x G) or its keys; the
// rows behind the last frame count as a frame whose other side is empty.  Counts are clamped into the tensors.
__device__ __forceinline__ XaPlace xa_find(const XaArgs& a, long long t, int unit, bool keys) {
  XaPlace p = {0, 0, 0, 0, -1};
  if (!a.qcnt) {
    const long long size = keys ? a.lk : (long long)a.lq * a.group, per = (size + unit - 1) / unit;
    if (per == 0) return p;
    const long long b = t / per;
    if (b >= a.frames) return p;
    p.q0 = b * a.lq; p.k0 = b * a.lk; p.nq = a.lq; p.nk = a.lk; p.tile = (int)(t - b * per);
    return p;
  }
  const int lane = threadIdx.x & 63;
  long long tiles0 = 0, q0 = 0, k0 = 0;
  for (int f0 = 0; f0 < a.frames; f0 += 64) {
    const int f = f0 + lane;
    long long cq = f < a.frames ? a.qcnt[f] : 0, ck = f < a.frames ? a.kcnt[f] : 0;
    cq = cq < 0 ? 0 : (cq > a.nq ? a.nq : cq);
    ck = ck < 0 ? 0 : (ck > a.nk ? a.nk : ck);
    long long sq = cq, sk = ck;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long x = __shfl_up(sq, o, 64), y = __shfl_up(sk, o, 64);
      if (lane >= o) { sq += x; sk += y; }
    }
    // (exclusive prefix, clamped to what is left of the tensors)
    long long eq = q0 + sq - cq, ek = k0 + sk - ck;
    eq = eq > a.nq ? a.nq : eq; ek = ek > a.nk ? a.nk : ek;
    cq = cq > a.nq - eq ? a.nq - eq : cq;
    ck = ck > a.nk - ek ? a.nk - ek : ck;
    const long long size = keys ? ck : cq * a.group, n = (size + unit - 1) / unit;
    long long sn = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long x = __shfl_up(sn, o, 64);
      if (lane >= o) sn += x;
    }
    const bool here = t >= tiles0 + sn - n && t < tiles0 + sn;
    const unsigned long long hit = __ballot(here);
    if (hit) {
      const int l = __ffsll((long long)hit) - 1;
      p.q0 = __shfl(eq, l, 64); p.k0 = __shfl(ek, l, 64);
      p.nq = (int)__shfl(cq, l, 64); p.nk = (int)__shfl(ck, l, 64);
      p.tile = (int)(t - __shfl(tiles0 + sn - n, l, 64));
      return p;
    }
    tiles0 += __shfl(sn, 63, 64);
    q0 = __shfl(eq + cq, 63, 64);
    k0 = __shfl(ek + ck, 63, 64);
  }
  const long long left = keys ? a.nk - k0 : a.nq - q0, size = keys ? left : left * a.group, n = (size + unit - 1) / unit;
  if (t >= tiles0 + n) return p;
  p.q0 = q0; p.k0 = k0; p.tile = (int)(t - tiles0);
  (keys ? p.nk : p.nq) = (int)left;
  return p;
}

__device__ __forceinline__ long long xa_uniform(long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long long)v >> 32));
  return (long long)((unsigned long long)hi << 32 | lo);
}
// xa_find in scalar registers: what follows from the place -- bases, loop bounds, branches -- is then the wave's, not a lane's
__device__ __forceinline__ XaPlace xa_place(const XaArgs& a, long long t, int unit, bool keys) {
  const XaPlace p = xa_find(a, t, unit, keys);
  return {xa_uniform(p.q0), xa_uniform(p.k0), __builtin_amdgcn_readfirstlane(p.nq), __builtin_amdgcn_readfirstlane(p.nk),
          __builtin_amdgcn_readfirstlane(p.tile)};
}

// bit j: key k0 + j exists (j < n) and is not masked; the same in every lane
__device__ __forceinline__ unsigned long long xa_valid(const unsigned char* mask, long long k0, int n) {
  const int lane = threadIdx.x & 63;
  return __ballot(lane < n && (!mask || mask[k0 + lane] != 0));
}

// host: rows of `tile` consecutive places start at 16-byte boundaries, are whole chunks and lie within 31 bits of each other
static inline bool xa_chunked(const void* p, long long row, long long head, int dim, int dtype) {
  const long long e = (long long)glx_elem_size(dtype);
  return ((uintptr_t)p & 15) == 0 && dim * e % 16 == 0 && row * e % 16 == 0 && head * e % 16 == 0 && row >= 0 && head >= 0
         && row * e < (1ll << 22) && head * e < (1ll << 22);
}

// host: upper bound of the tiles that xa_place hands out
static inline long long xa_tiles(long long n, int frames, int per_frame, bool counts, int unit) {
  return counts ? n / unit + frames + 1 : (long long)frames * ((per_frame + (long long)unit - 1) / unit);
}
