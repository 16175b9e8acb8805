// Orthogonalised updates (glenet_amd/optim.py): Newton-Schulz steps on a list of matrices of any shapes, few launches for all.
// Matrices of up to 16 rows have a kernel of their own, further down; what follows is about the others.
//
//   X = G / (|G|_F + eps), transposed where G has more rows than columns (X: m x n, m <= n);  per step
//   A = X X^T,  X <- a X + (b A + c A^2) X  =  P X,  P = a I + b A + c A^2
//
// The next step's Gram matrix is P A P, and every P is a polynomial of the first A: a SEGMENT of s steps runs on m x m matrices
// alone (P = aI + bA + cA^2;  H = P A;  A <- H P;  Q <- P Q) and touches X twice, A = X X^T before and X <- Q X behind.  With
// symmetric products formed once per pair of tiles a segment costs 3 m^2 n + (4 s - 3) m^3 multiply-adds instead of
// s (3 m^2 n + m^3): the same for square matrices, s times less work on X for wide ones.  What limits s is rounding: a
// perturbation of A in directions of small singular values grows by a^2 = 11.9 per step until the next look at X.  Measured
// against 64 bits over six gradients with decaying spectra, in the Frobenius norm and as a multiple of what plain fp32 products leave
// (1e-6 to 3e-6): fp32 in segments of one step 0.4 to 0.8, of three 0.4 to 1.3 (single ones of 300 x 1500 up to 1.9), and below the
// limits that follow 1.1 to 2.0 (200 x 300 1.7, 129 x 1032 2.0).  So fp32 takes segments of three above 192 rows and from 4 : 1 on
// (1000 x 4400: 440 us, in segments of one 634; 200 x 300 would not gain), fp16, whose rounding covers both, three above 128 rows and
// from 1.25 : 1 on (1000 x 3600: 347 and 471 us; 512 x 600 188 and 179, the other way), bf16 five there (290 and 471 us; 2000 x 2400
// 1078 and 936; its error up to 1.24 times its rounding's), and the rest one.
//
// Products: every operand is held as two fp16 planes of value * 2^k (hi + lo: 22 bits down to 2^-25 of the scale), and a
// product is three MFMAs hi hi + hi lo + lo hi into fp32.  The scales 2^k come from bounds of the spectral norms that follow
// from the coefficients (the eigenvalues start in [0, 1]) and from |X_0| = |G| / (|G| + eps), so nothing overflows and a
// gradient far below eps keeps its precision (down to norms of 1e-36).
// Zero padding to whole tiles is exact: it stays zero in A and X.
//
// 4096 x 4096 bf16: 3.54 to 3.7 ms by the box.  A split product of the size of Q X takes 446 us (925 TFLOP/s of fp16 products; a large
// library product reaches 1119), a single one 212 us (649: its 64 KB stages wait for their way from L2 to LDS).  256 x 256 fp32: 15 products
// of 8 us each, all latency.
#include "glx_elem.h"

#include <math.h>
#include <vector>

#define NS_K 64                // the k range of a split comes in multiples of this
#define NS_OPS 39              // products of one launch (kernel arguments: 96 bytes each)
#define NS_MATS 40             // matrices of one prologue launch
#define NS_SMALLS 64           // matrices of one launch of the small ones
#define NS_AHEAD 4             // 16-column pieces that each of their 16 waves has on their way
#define NS_STEPS 64            // at most
#define NS_PARTS 1024          // partial sums of squares per matrix, at most
#define NS_BYTES (1ull << 30)  // workspace of the matrices that run together: a list beyond it runs in groups, one behind the other

typedef _Float16 nh8 __attribute__((ext_vector_type(8)));
typedef _Float16 nh4 __attribute__((ext_vector_type(4)));
typedef float nf16 __attribute__((ext_vector_type(16)));
typedef float nf4 __attribute__((ext_vector_type(4)));

enum { NS_PLANES, NS_PARTIAL, NS_XPLANES, NS_FINAL };

// out = epilogue(alpha A B^T): A (mp, K), B (np, K) planes, lo plane behind the hi plane.  Places in the workspace in units of
// 256 bytes, 0: none (the first unit stays empty)
struct NsOp {
  unsigned a, b, d;            // d: NS_PLANES: + beta D, D (mp, mp) planes
  unsigned out, out2;          // NS_PLANES: planes (mp, mp); NS_PARTIAL: fp32 [splits][mp][mp]; NS_XPLANES: planes (mp, np) and
                               // their transpose (np, mp)
  unsigned xin, xout;          // scales of the X planes that are read (`xpow` of the operands) / written, floats
  float alpha, beta, diag, scale;
  int mp, np, K, m, n;
  long long ldd;               // NS_FINAL: elements between the caller's rows
  void* dst;                   // ... its matrix
  unsigned short splits, kper; // kper: k elements of a split, in NS_K
  unsigned char kind, sym, tall, dtype, xpow, xstep, xnext;
};
struct NsOps { int first[NS_OPS]; NsOp op[NS_OPS]; int count; char* ws; };       // first[k]: first block of op k

struct NsMat {
  const void* src; long long ld;       // the caller's matrix, `rows` x `cols`
  _Float16* x; _Float16* xt;           // planes (mp, np) and (np, mp)
  double* parts; float* xscale;        // sums of squares; the scale of X's planes in front of every step
  int rows, cols, mp, np, tall, nparts;
};
// xb[s], qb[s]: bounds of |X| in front of step s, and of |X| / |X_0|
struct NsMats { int first[NS_MATS], tfirst[NS_MATS]; NsMat mat[NS_MATS]; int count, dtype, steps; double eps; float xb[NS_STEPS], qb[NS_STEPS]; };
static_assert(sizeof(NsMats) <= 4032 && sizeof(NsOps) <= 4032, "kernel arguments");

// the entry whose blocks hold this one: the first blocks side by side, one read for a wave (kernel arguments lie in host memory;
// a search through the entries themselves costs a round trip each)
__device__ __forceinline__ int ns_entry(const int* first, int count) {
  const int lane = threadIdx.x & 63;
  return __popcll(__ballot(lane < count && (int)blockIdx.x >= first[lane < count ? lane : 0])) - 1;
}
// elements between the rows of planes of k columns: rows of a power of two bytes would all start in the same cache channels
__host__ __device__ __forceinline__ int ns_ld(int k) { return k % 256 == 0 ? k + 64 : k; }
__device__ __forceinline__ void ns_split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}
__device__ __forceinline__ float ns_elem(const void* p, long long i, int dtype) {
  return dtype == GLX_F32 ? ((const float*)p)[i] : dtype == GLX_BF16 ? (float)((const __bf16*)p)[i] : (float)((const _Float16*)p)[i];
}

// ------------------------------------------------------------------------------------------------ |G|_F and the planes of X
__global__ __launch_bounds__(256) void k_ns_norm(NsMats s) {
  const int k = ns_entry(s.first, s.count);
  const NsMat& t = s.mat[k];
  const int part = blockIdx.x - s.first[k];
  double sum = 0.0;
  auto add = [&](auto* src) {
    typedef GlxVec<__remove_cvref(decltype(*src)), 4> V;
    const bool dense = t.ld == t.cols;
    const long long runs = dense ? 1 : t.rows, len = dense ? (long long)t.rows * t.cols : t.cols;
    // one run: the parts stride over it; else over the rows
    for (long long r = dense ? 0 : part; r < runs; r += dense ? 1 : t.nparts) {
      const long long first = ((dense ? (long long)part * 256 : 0) + threadIdx.x) * 4, step = (dense ? (long long)t.nparts : 1) * 1024;
#pragma unroll 4
      for (long long e = first; e < len; e += step) {
        if (e + 4 <= len) {
          const auto v = V::load(src + r * t.ld + e);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += (double)(float)v[i] * (double)(float)v[i];
        } else {
          for (long long i = e; i < len; ++i) sum += (double)(float)src[r * t.ld + i] * (double)(float)src[r * t.ld + i];
        }
      }
    }
  };
  if (s.dtype == GLX_F32) add((const float*)t.src);
  else if (s.dtype == GLX_BF16) add((const __bf16*)t.src);
  else add((const _Float16*)t.src);
  __shared__ double red[256];
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) t.parts[part] = red[0];
}

// a 64 x 64 tile of X: read along the caller's rows, written as planes of X and of its transpose
__global__ __launch_bounds__(256) void k_ns_planes(NsMats s) {
  __shared__ float tile[64][65];
  __shared__ double red[256];
  const int k = ns_entry(s.tfirst, s.count);
  const NsMat& t = s.mat[k];
  double mine = 0.0;
  for (int i = threadIdx.x; i < t.nparts; i += 256) mine += t.parts[i];
  red[threadIdx.x] = mine;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  const int b = blockIdx.x - s.tfirst[k], tiles_n = t.np / 64;
  const double norm = sqrt(red[0]), rho = norm / (norm + s.eps);
  // the planes hold G 2^k with |G| 2^k in [2^14, 2^15): 16-bit values exactly, in the hi plane alone
  const int k0 = norm > 0.0 ? 14 - ilogb(norm) : 60, kx = k0 > 127 ? 127 : (k0 < -120 ? -120 : k0);
  const float up = ldexpf(1.f, kx);
  if (b == 0 && (int)threadIdx.x < s.steps) {
    // X = planes / xscale; later X in front of step st: min(xb, qb rho) 2^e in [2^14, 2^15).  (|G| = 1e-36 beside eps = 1e-7 has
    // e = 110; xscale^2 is infinite from 2^64 on, which makes A, below 2^-100 there, 0)
    const int st = threadIdx.x;
    const float bound = fminf(s.xb[st], (float)(s.qb[st] * rho));
    const int e = bound > 0.f ? 14 - ilogbf(bound) : 60;
    t.xscale[st] = st == 0 ? (float)((double)up * (norm + s.eps)) : ldexpf(1.f, e > 120 ? 120 : e);
  }
  const int i0 = b / tiles_n * 64, j0 = b % tiles_n * 64;      // of X
  const int c = threadIdx.x & 63;
#pragma unroll 4
  for (int r = threadIdx.x >> 6; r < 64; r += 4) {
    const int row = t.tall ? j0 + r : i0 + r, col = t.tall ? i0 + c : j0 + c;       // of the caller's matrix
    const float v = row < t.rows && col < t.cols ? ns_elem(t.src, row * t.ld + col, s.dtype) * up : 0.f;
    if (t.tall) tile[c][r] = v; else tile[r][c] = v;
  }
  __syncthreads();
  const int ldn = ns_ld(t.np), ldm = ns_ld(t.mp);
  const long long plane = (long long)t.mp * ldn, tplane = (long long)t.np * ldm;
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int q = threadIdx.x + it * 256, r = q >> 3, c8 = (q & 7) * 8;
    nh8 h, l, th, tl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 u, v;
      ns_split(tile[r][c8 + e], u, v);
      h[e] = u; l[e] = v;
      ns_split(tile[c8 + e][r], u, v);
      th[e] = u; tl[e] = v;
    }
    const long long o = (long long)(i0 + r) * ldn + j0 + c8, ot = (long long)(j0 + r) * ldm + i0 + c8;
    *reinterpret_cast<nh8*>(t.x + o) = h;
    *reinterpret_cast<nh8*>(t.xt + ot) = th;
    if (s.dtype == GLX_F32) {
      *reinterpret_cast<nh8*>(t.x + plane + o) = l;
      *reinterpret_cast<nh8*>(t.xt + tplane + ot) = tl;
    }
  }
}

// ------------------------------------------------------------------------------------------------ the products
// A block forms a TILE x TILE tile.  k comes in steps of KS that go from memory to LDS without registers, STAGES of them ahead (a
// product is bound by the round trips of what is in flight: four stages bring 256 x 256 in one); the four waves share a step
// along k, each for the whole tile, so that an operand read from LDS serves two or four products, and their sums are joined through
// LDS at the end, each wave finishing a quarter.  (With a quarter of the tile per wave the
// 64-wide form read twice as much from LDS as the matrix units could take.)  The order of a staged row's 16-byte chunks is rotated
// by the row, so that the 32 rows an operand read touches spread over the banks.  PROD products per pair of operands: 3 both split
// (4: with lo lo), 2 where B's lo plane is empty, 1 where neither is used.
template <int TILE, int PROD, int STAGES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void k_ns_gemm(NsOps s) {
  constexpr int KS = 64, C = KS / 8, RB = KS * 2;                    // k elements of a stage, its chunks and bytes per row
  constexpr int PA = PROD > 1 ? 2 : 1, PB = PROD > 2 ? 2 : 1;        // planes of the operands
  constexpr int F = TILE / 32, H = TILE / 64;                        // 32-wide parts: of the tile, of a quarter of it
  constexpr int CH = TILE * C / 256, LOADS = (PA + PB) * CH;         // transfers per thread: of a plane, of a stage
  constexpr int PLANE = TILE * RB, STAGE = (PA + PB) * PLANE;
  constexpr int PIECES = TILE == 64 ? 4 : 2, JOIN = PIECES * 4 * H * H * 4096, BYTES = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  const int entry = ns_entry(s.first, s.count);
  const NsOp& t = s.op[entry];
  int b = blockIdx.x - s.first[entry];
  const int tm = t.mp / TILE, tn = t.np / TILE;
  const int per = t.sym ? tm * (tm + 1) / 2 : tm * tn, split = b / per;
  b -= split * per;
  int ti, tj;
  if (t.sym) {                                                       // row ti holds the tiles tj <= ti
    ti = (int)((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
    while (ti * (ti + 1) / 2 > b) --ti;
    tj = b - ti * (ti + 1) / 2;
  } else {
    ti = b / tn; tj = b - ti * tn;
  }
  auto at = [&](unsigned place) { return s.ws + (size_t)place * 256; };
  const float xin = t.xin ? ((const float*)at(t.xin))[t.xstep] : 1.f, alpha = t.alpha / (t.xpow == 2 ? xin * xin : xin);
  const float scale = t.xout ? ((const float*)at(t.xout))[t.xnext] : t.scale;
  const int kper = t.kper * NS_K, k0 = split * kper, k1 = k0 + kper < t.K ? k0 + kper : t.K;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l32 = lane & 31;
  const int ld = ns_ld(t.K);
  const _Float16* src[PA + PB];
#pragma unroll
  for (int p = 0; p < PA; ++p) src[p] = (const _Float16*)at(t.a) + ((long long)p * t.mp + ti * TILE) * ld;
#pragma unroll
  for (int p = 0; p < PB; ++p) src[PA + p] = (const _Float16*)at(t.b) + ((long long)p * t.np + tj * TILE) * ld;
  auto swap = [](int r, int ch) { return (ch ^ r) & 7; };
  // memory -> LDS: a lane fetches the chunk that belongs at its place (the compiler does not see these transfers)
  int off[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int q = threadIdx.x + c * 256, r = q / C;
    off[c] = (r * ld + swap(r, q) * 8) * 2;
  }
  auto fetch = [&](int n, int x, int slot = -1) {                    // transfer x of stage n
    const unsigned to = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem
                        + (slot < 0 ? n % STAGES : slot) * STAGE + (wave << 10);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 ::"v"(off[x % CH]), "s"(src[x / CH] + k0 + n * KS), "s"(to + x / CH * PLANE + x % CH * 4096)
                 : "memory");
  };
  nf16 acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = (nf16)(0.f);
  const int stages = (k1 - k0) / KS;
  // 64-wide: every slot is filled at once, and again as it falls free.  128-wide: a slot stays free, the transfers for it go out
  // between the products (one after the other they hold a wave up for as long as the products take), behind the last stage
  // repeating it into slots that are not read again
  constexpr bool BETWEEN = TILE == 128;
  for (int n = 0; n < STAGES - BETWEEN && n < stages; ++n)
#pragma unroll
    for (int x = 0; x < LOADS; ++x) fetch(n, x);
  for (int n = 0; n < stages; ++n) {
    // stage n is there once at most the later ones are on their way; its slot's last readers have passed the barrier of n - 1
    if (BETWEEN ? stages >= STAGES - 1 : n > 0 && n + STAGES - 2 < stages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * LOADS) : "memory");
    else if (!BETWEEN && n == 0 && stages >= STAGES) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (!BETWEEN && n > 0 && n + STAGES - 1 < stages) {
#pragma unroll
      for (int x = 0; x < LOADS; ++x) fetch(n + STAGES - 1, x);
    }
    const int from = n + STAGES - 1 < stages ? n + STAGES - 1 : stages - 1, slot = (n + STAGES - 1) % STAGES;
    const char* at = smem + (n % STAGES) * STAGE;
    const int ch = wave * 2 + half;
    nh8 fa[2][PA], fb[F][PB];
    auto rows = [&](int i) {
#pragma unroll
      for (int p = 0; p < PA; ++p)
        fa[i & 1][p] = *reinterpret_cast<const nh8*>(at + p * PLANE + (i * 32 + l32) * RB + swap(l32, ch) * 16);
    };
    rows(0);
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int p = 0; p < PB; ++p)
        fb[j][p] = *reinterpret_cast<const nh8*>(at + (PA + p) * PLANE + (j * 32 + l32) * RB + swap(l32, ch) * 16);
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if (i + 1 < F) rows(i + 1);
#pragma unroll
      for (int q = PROD - 1; q >= 0; --q) {                          // lo lo, hi lo, lo hi, hi hi: smallest first
        constexpr int GROUPS = F * PROD;
        const int g = i * PROD + PROD - 1 - q;
        __builtin_amdgcn_sched_barrier(0);
        if (BETWEEN) {
#pragma unroll
          for (int x = g * LOADS / GROUPS; x < (g + 1) * LOADS / GROUPS; ++x) fetch(from, x, slot);
        }
#pragma unroll
        for (int j = 0; j < F; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i & 1][q == 3 || q == 1 ? PA - 1 : 0], fb[j][q >= 2 ? PB - 1 : 0], acc[i][j], 0, 0, 0);
      }
    }
  }
  if (BETWEEN) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // the waves' sums, all quarters of the tile at once (128-wide: two and two); wave w keeps quarter w
  const int wi = wave >> 1, wj = wave & 1;
  nf16 sum[H][H];
  float* join = (float*)smem;
#pragma unroll
  for (int r = 0; r < 4; r += PIECES) {
    __syncthreads();
#pragma unroll
    for (int q = r; q < r + PIECES; ++q)
      if (wave != q) {
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
          for (int j = 0; j < H; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const nf16& v = acc[(q >> 1) * H + i][(q & 1) * H + j];
              *reinterpret_cast<nf4*>(join + (((((q - r) * 4 + wave) * H + i) * H + j) * 4 + g) * 256 + lane * 4) =
                  nf4{v[g * 4], v[g * 4 + 1], v[g * 4 + 2], v[g * 4 + 3]};
            }
      }
    __syncthreads();
#pragma unroll
    for (int q = r; q < r + PIECES; ++q)
      if (wave == q) {
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
          for (int j = 0; j < H; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const nf16& own = acc[(q >> 1) * H + i][(q & 1) * H + j];
              nf4 v = nf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int w = 0; w < 4; ++w)
                v += w == q ? nf4{own[g * 4], own[g * 4 + 1], own[g * 4 + 2], own[g * 4 + 3]}
                            : *reinterpret_cast<const nf4*>(join + (((((q - r) * 4 + w) * H + i) * H + j) * 4 + g) * 256 + lane * 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) sum[i][j][g * 4 + e] = v[e];
            }
      }
  }
  // a lane's accumulators: column l32, rows 8 g + 4 half + 0..3 of the 32 x 32 part
#pragma unroll
  for (int i = 0; i < H; ++i)
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int row0 = ti * TILE + (wi * H + i) * 32 + half * 4, col = tj * TILE + (wj * H + j) * 32 + l32;
      if (t.kind == NS_PARTIAL) {
        float* o = (float*)at(t.out) + (long long)split * t.mp * t.mp;
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[(long long)(row0 + g * 8 + e) * t.mp + col] = sum[i][j][g * 4 + e] * alpha;
      } else if (t.kind == NS_FINAL) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = row0 + g * 8 + e;
            if (row >= t.m || col >= t.n) continue;
            const float v = sum[i][j][g * 4 + e] * alpha;
            const long long to = t.tall ? (long long)col * t.ldd + row : (long long)row * t.ldd + col;
            if (t.dtype == GLX_F32) ((float*)t.dst)[to] = v;
            else if (t.dtype == GLX_BF16) ((__bf16*)t.dst)[to] = (__bf16)v;
            else ((_Float16*)t.dst)[to] = (_Float16)v;
          }
      } else {
        const int ldm = ns_ld(t.mp), ldo = t.kind == NS_PLANES ? ldm : ns_ld(t.np);
        const long long po = (long long)t.mp * ldo, px = (long long)(t.kind == NS_PLANES ? t.mp : t.np) * ldm;
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = sum[i][j][e] * alpha;
        if (t.d) {                                             // (D is symmetric: its column's four values lie side by side)
          const _Float16* d = (const _Float16*)at(t.d) + (long long)col * ldm + row0;
          nh4 dh[4], dl[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            dh[g] = *reinterpret_cast<const nh4*>(d + g * 8);
            dl[g] = *reinterpret_cast<const nh4*>(d + (long long)t.mp * ldm + g * 8);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            v[e] += t.beta * ((float)dh[e >> 2][e & 3] + (float)dl[e >> 2][e & 3]);
            if (row0 + (e >> 2) * 8 + (e & 3) == col) v[e] += t.diag;
          }
        }
        // the planes themselves, and X's transposed planes or a symmetric product's mirrored tile (the diagonal's holds both)
        const bool own = t.kind == NS_XPLANES || ti != tj;
        _Float16* o = (_Float16*)at(t.out);
        _Float16* x = (_Float16*)at(t.kind == NS_XPLANES ? t.out2 : t.out) + (long long)col * ldm + row0;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          nh4 h, l;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            _Float16 u, w;
            ns_split(v[g * 4 + e] * scale, u, w);
            h[e] = u; l[e] = w;
            if (own) {
              _Float16* to = o + (long long)(row0 + g * 8 + e) * ldo + col;
              to[0] = u; to[po] = w;
            }
          }
          *reinterpret_cast<nh4*>(x + g * 8) = h;
          *reinterpret_cast<nh4*>(x + px + g * 8) = l;
        }
      }
    }
}

// the splits' sum of a Gram matrix (64-wide tiles on and below the diagonal were formed) as planes of the whole matrix: a block per 16
// rows of a tile, and the mirrored columns through LDS
__global__ __launch_bounds__(256) void k_ns_join(NsOps s) {
  __shared__ float tile[16][68];
  const int k = ns_entry(s.first, s.count);
  const NsOp& t = s.op[k];
  const int b = blockIdx.x - s.first[k], tri = b >> 2;
  int ti = (int)((sqrtf(8.f * tri + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= tri) ++ti;
  while (ti * (ti + 1) / 2 > tri) --ti;
  const int tj = tri - ti * (ti + 1) / 2, r0 = ti * 64 + (b & 3) * 16, c0 = tj * 64, ld = ns_ld(t.mp);
  const long long plane = (long long)t.mp * t.mp, lo = (long long)t.mp * ld;
  _Float16* out = (_Float16*)(s.ws + (size_t)t.out * 256);
  const int r = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
  const float* p = (const float*)(s.ws + (size_t)t.a * 256) + (long long)(r0 + r) * t.mp + c0 + c;
  nf4 v = nf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int q = 0; q < t.splits; ++q) v += *reinterpret_cast<const nf4*>(p + q * plane);
  auto put = [&](long long to, nf4 x) {
    nh4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      _Float16 u, w;
      ns_split(x[e] * t.scale, u, w);
      h[e] = u; l[e] = w;
    }
    *reinterpret_cast<nh4*>(out + to) = h;
    *reinterpret_cast<nh4*>(out + lo + to) = l;
  };
  put((long long)(r0 + r) * ld + c0 + c, v);
  if (ti == tj) return;
  *reinterpret_cast<nf4*>(&tile[r][c]) = v;
  __syncthreads();
  const int col = threadIdx.x >> 2, rr = (threadIdx.x & 3) * 4;
  put((long long)(c0 + col) * ld + r0 + rr, nf4{tile[rr][col], tile[rr + 1][col], tile[rr + 2][col], tile[rr + 3][col]});
}

// ------------------------------------------------------------------------------------------------ matrices of up to 16 rows
// One block per matrix, all of it in one launch and in 64 bits: A = X X^T on the fp64 matrix units (one value per lane is both
// operands), the steps on the 16 x 16 polynomials, X <- Q X.  Few singular values leave nothing to average: here a
// matrix is 2e-8 to 4e-8 off, a twentieth of what plain fp32 arithmetic leaves, and on the split products above its some 15
// launches were all latency.  Bound by the fp64 matrix units (14 us of 56 at 16 x 4096) and one CU's loads.
typedef double nd4 __attribute__((ext_vector_type(4)));
struct NsSmall { const void* src; void* dst; long long ld_src, ld_dst; int rows, cols; };
struct NsSmalls { NsSmall mat[NS_SMALLS]; double c[3], eps; int steps, dtype; };
static_assert(sizeof(NsSmalls) <= 4032, "kernel arguments");

__global__ __launch_bounds__(1024) void k_ns_small(NsSmalls s) {
  __shared__ double part[16][16][17], A[16][17], P[16][17], H[16][17], Q[2][16][17];
  const NsSmall& t = s.mat[blockIdx.x];
  const bool tall = t.rows > t.cols;
  const int m = tall ? t.cols : t.rows, n = tall ? t.rows : t.cols;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, kq = lane >> 4;
  const int r = threadIdx.x >> 4 & 15, c = threadIdx.x & 15;
  const bool first = threadIdx.x < 256;                        // a thread per entry of the 16 x 16 matrices
  auto run = [&](auto* src) {
    typedef __remove_cvref(decltype(*src)) T;
    const long long down = tall ? 1 : t.ld_src, along = tall ? t.ld_src : 1;
    // of X, before the division by its norm (no branch around the load: many are on their way at once)
    auto load = [&](int row, int col) { return (float)src[(row < m ? row : 0) * down + (col < n ? col : 0) * along]; };
    auto there = [&](int row, int col, float v) { return row < m && col < n ? (double)v : 0.0; };
    nd4 acc = {0.0, 0.0, 0.0, 0.0};
    for (int k0 = wave * 16; k0 < n; k0 += 256 * NS_AHEAD) {
      float v[NS_AHEAD][4];
#pragma unroll
      for (int a = 0; a < NS_AHEAD; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) v[a][u] = load(i, k0 + a * 256 + kq * 4 + u);
#pragma unroll
      for (int a = 0; a < NS_AHEAD; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const double x = there(i, k0 + a * 256 + kq * 4 + u, v[a][u]);
          acc = __builtin_amdgcn_mfma_f64_16x16x4f64(x, x, acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) part[wave][u * 4 + kq][i] = acc[u];
    __syncthreads();
    if (first) {
      double v = 0.0;
#pragma unroll
      for (int w = 0; w < 16; ++w) v += part[w][r][c];
      A[r][c] = v;
    }
    __syncthreads();
    double square = 0.0;
#pragma unroll
    for (int u = 0; u < 16; ++u) square += A[u][u];            // |G|_F^2
    const double inv = 1.0 / (sqrt(square) + s.eps);
    __syncthreads();
    if (first) {
      A[r][c] = A[r][c] * inv * inv;
      Q[0][r][c] = r == c ? 1.0 : 0.0;
    }
    __syncthreads();
    auto product = [&](const double (*x)[17], const double (*y)[17]) {
      double v = 0.0;
#pragma unroll
      for (int u = 0; u < 16; ++u) v += x[r][u] * y[u][c];
      return v;
    };
    int q = 0;
    for (int step = 0; step < s.steps; ++step, q ^= 1) {
      if (first) P[r][c] = (r == c ? s.c[0] : 0.0) + s.c[1] * A[r][c] + s.c[2] * product(A, A);
      __syncthreads();
      if (first) {
        Q[q ^ 1][r][c] = product(P, Q[q]);
        H[r][c] = product(P, A);
      }
      __syncthreads();
      if (first) A[r][c] = product(H, P);
      __syncthreads();
    }
    double z[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = Q[q][i][u * 4 + kq] * inv;
    for (int j0 = wave * 16; j0 < n; j0 += 256 * NS_AHEAD) {
      float v[NS_AHEAD][4];
#pragma unroll
      for (int a = 0; a < NS_AHEAD; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) v[a][u] = load(u * 4 + kq, j0 + a * 256 + i);
#pragma unroll
      for (int a = 0; a < NS_AHEAD; ++a) {
        const int col = j0 + a * 256 + i;
        nd4 x = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int u = 0; u < 4; ++u) x = __builtin_amdgcn_mfma_f64_16x16x4f64(z[u], there(u * 4 + kq, col, v[a][u]), x, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = u * 4 + kq;
          if (row < m && col < n) ((T*)t.dst)[tall ? col * t.ld_dst + row : row * t.ld_dst + col] = (T)(float)x[u];
        }
      }
    }
  };
  if (s.dtype == GLX_F32) run((float*)t.src);
  else if (s.dtype == GLX_BF16) run((__bf16*)t.src);
  else run((_Float16*)t.src);
}

// ------------------------------------------------------------------------------------------------ host: programs
struct NsPlan {                // one matrix
  int rows, cols, m, n, mp, np, tile, xtile, tall, seg, splits, kper, nparts;       // tile: of symmetric products, xtile: of Q X
  size_t x, xt[2], g, h, p[2], q[2], part, parts, xscale;              // byte offsets in the workspace
};

static float ns_scale(double bound) { return (float)exp2(floor(log2(32768.0 / bound))); }

// the largest eigenvalues that the coefficients allow, step by step: lambda <- lambda p(lambda)^2 from [0, 1]
static bool ns_bounds(int steps, const double* c, std::vector<double>& lam, std::vector<double>& pmax, std::vector<double>& hmax) {
  if (!isfinite(c[0]) || !isfinite(c[1]) || !isfinite(c[2])) return false;
  double top = 1.01;           // (A's eigenvalues are at most 1 up to its own rounding)
  lam.push_back(top);
  for (int s = 0; s < steps; ++s) {
    double pm = 0, hm = 0, next = 0;
    for (int i = 0; i <= 2048; ++i) {
      const double l = top * i / 2048, p = c[0] + c[1] * l + c[2] * l * l;
      pm = fmax(pm, fabs(p)); hm = fmax(hm, fabs(l * p)); next = fmax(next, l * p * p);
    }
    // (between the samples: a polynomial of degree 5 moves by far less than 1 % of its maximum)
    pmax.push_back(pm * 1.01 + 1e-6); hmax.push_back(hm * 1.01 + 1e-6);
    top = next * 1.02 + 1e-6;
    if (!(top < 64.0) || !(pm < 64.0)) return false;
    lam.push_back(top);
  }
  return true;
}

static int ns_padded(int v, int tile) { return (v + tile - 1) / tile * tile; }

// (16 x 64: 13 us in one launch, 81 on the tiles; x 801: 20 and 119; x 4096: 56 and 118; x 16384: 191 and 139)
static bool ns_small(const glx_matrix& a) { return (a.rows < a.cols ? a.rows : a.cols) <= 16 && a.rows <= 8192 && a.cols <= 8192; }

// the plan of one matrix and its places in the workspace from `at` on.  Steep: segments of one step
static NsPlan ns_plan(int rows, int cols, int dtype, int steps, bool steep, size_t& at) {
  NsPlan p = {};
  p.rows = rows; p.cols = cols; p.tall = rows > cols;
  p.m = p.tall ? cols : rows; p.n = p.tall ? rows : cols;
  // 128-wide tiles where they still fill the card: they read half as much from LDS per product
  const int pad = p.m > 1024 ? 128 : 64;
  p.mp = ns_padded(p.m, pad); p.np = ns_padded(p.n, pad);
  const long long wide = p.mp / 128, across = p.np / 128;
  p.tile = pad == 128 && wide * (wide + 1) / 2 >= 200 ? 128 : 64;
  p.xtile = pad == 128 && wide * across >= 200 ? 128 : 64;
  p.seg = dtype == GLX_BF16 ? 5 : 3;
  // (fp32 rows up to 192: 129 x 1032 comes out 2.0 times as far off as plain fp32 products in segments of three, 0.6 times in ones;
  // 160 x 800 takes 155 and 158 us)
  if (p.m <= (dtype == GLX_F32 ? 192 : 128) || (dtype == GLX_F32 ? p.n < 4ll * p.m : 4ll * p.n <= 5ll * p.m) || steep) p.seg = 1;
  if (p.seg > steps) p.seg = steps;
  const int t = p.mp / p.tile;
  const long long tiles = (long long)t * (t + 1) / 2, ksteps = p.np / NS_K;
  // (only where a quarter of the compute units would have a tile: every part is read again by the join)
  long long splits = p.tile == 64 && tiles <= 64 ? 256 / tiles : 1;
  if (splits > ksteps / 8) splits = ksteps / 8;         // 512 k elements a split, at least: a join costs as much as those
  if (splits < 1) splits = 1;
  p.kper = (int)((ksteps + splits - 1) / splits) * NS_K;
  p.splits = (int)((p.np + p.kper - 1) / p.kper);
  const long long total = (long long)p.m * p.n;
  p.nparts = (int)((total + 4095) / 4096);
  if (p.nparts > NS_PARTS) p.nparts = NS_PARTS;
  const size_t ldn = ns_ld(p.np), ldm = ns_ld(p.mp), X = p.mp * ldn * 4, XT = p.np * ldm * 4, S = p.mp * ldm * 4;
  auto take = [&](size_t bytes) { const size_t o = at; at += glx_align(bytes); return o; };
  // X <- Q X reads the transposed planes alone, so X's own are overwritten; H, the second P and the Qs are those of longer segments
  p.x = take(X); p.xt[0] = take(XT); p.xt[1] = p.seg < steps ? take(XT) : p.xt[0];
  p.g = take(S); p.p[0] = take(S);
  if (p.seg > 1) { p.h = take(S); p.p[1] = take(S); p.q[1] = take(S); }
  if (p.seg > 2) p.q[0] = take(S);
  p.part = take(p.splits > 1 ? (size_t)p.mp * p.mp * 4 * p.splits : 256);
  p.parts = take(NS_PARTS * sizeof(double));
  p.xscale = take(NS_STEPS * sizeof(float));
  return p;
}

static int ns_check(const char* who, const glx_matrix* mats, int count, int dtype, int steps) {
  GLX_REQUIRE(count >= 0 && (count == 0 || mats), "%s: null list", who);
  GLX_REQUIRE(glx_elem_ok(dtype), "%s: dtype %d", who, dtype);
  GLX_REQUIRE(steps >= 1 && steps <= NS_STEPS, "%s: %d steps", who, steps);
  for (int i = 0; i < count; ++i)
    GLX_REQUIRE(mats[i].rows >= 1 && mats[i].cols >= 1 && mats[i].rows <= (1 << 20) && mats[i].cols <= (1 << 20)
                && (mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols) <= (1 << 15),
                "%s: matrix %d is %d x %d", who, i, mats[i].rows, mats[i].cols);
  return GLX_OK;
}

// of one matrix, whatever the coefficients
static size_t ns_bytes(const glx_matrix& a, int dtype, int steps) {
  size_t usual = 0, steep = 0;
  ns_plan(a.rows, a.cols, dtype, steps, false, usual);
  ns_plan(a.rows, a.cols, dtype, steps, true, steep);
  return usual > steep ? usual : steep;
}
// the end of the group that begins at matrix i, and its bytes: one matrix at least, more while they fit NS_BYTES
static int ns_group(const glx_matrix* mats, int i, int count, int dtype, int steps, size_t* bytes) {
  *bytes = 256;                                        // (place 0 means none)
  for (const int first = i; i < count; ++i) {
    const size_t b = ns_small(mats[i]) ? 0 : ns_bytes(mats[i], dtype, steps);
    if (i > first && b > 0 && *bytes + b > NS_BYTES) break;
    *bytes += b;
  }
  return i;
}

extern "C" size_t glx_orthogonalize_workspace_bytes(const glx_matrix* mats, int count, int dtype, int steps) {
  if (ns_check("glx_orthogonalize_workspace_bytes", mats, count, dtype, steps) != GLX_OK) return 0;
  size_t most = 256, bytes;
  for (int i = 0; i < count; most = bytes > most ? bytes : most) i = ns_group(mats, i, count, dtype, steps, &bytes);
  return most + 256;
}

struct NsStage {               // what one launch round does, over all matrices
  std::vector<NsOp> gemm[2][4], join;       // by tile; by the products per pair of operands
  void add(int tile, int prods, const NsOp& o) { gemm[tile == 128][prods - 1].push_back(o); }
};

template <int TILE, int STAGES>
static void ns_launch_gemm(const NsOps& s, int blocks, int prods, hipStream_t st) {
  constexpr int MORE = TILE == 128 ? 2 : 1;             // (fewer planes, more stages in the same LDS)
  if (prods == 4) hipLaunchKernelGGL((k_ns_gemm<TILE, 4, STAGES>), dim3(blocks), dim3(256), 0, st, s);
  else if (prods == 3) hipLaunchKernelGGL((k_ns_gemm<TILE, 3, STAGES>), dim3(blocks), dim3(256), 0, st, s);
  else if (prods == 2) hipLaunchKernelGGL((k_ns_gemm<TILE, 2, STAGES + MORE - 1>), dim3(blocks), dim3(256), 0, st, s);
  else hipLaunchKernelGGL((k_ns_gemm<TILE, 1, STAGES * MORE>), dim3(blocks), dim3(256), 0, st, s);
}
static void ns_launch_ops(std::vector<NsOp>& ops, char* ws, int tile, int prods, hipStream_t st) {       // prods = 0: joins
  for (size_t i = 0; i < ops.size(); i += NS_OPS) {
    NsOps s;
    memset(&s, 0, sizeof(s));
    s.ws = ws;
    int blocks = 0;
    for (size_t j = i; j < ops.size() && j < i + NS_OPS; ++j) {
      s.first[s.count] = blocks;
      NsOp& o = s.op[s.count++] = ops[j];
      const int tm = o.mp / tile, tn = o.np / tile;
      blocks += prods == 0 ? tm * (tm + 1) / 2 * 4 : (o.sym ? tm * (tm + 1) / 2 : tm * tn) * o.splits;
    }
    if (prods == 0) hipLaunchKernelGGL(k_ns_join, dim3(blocks), dim3(256), 0, st, s);
    else if (tile == 128) ns_launch_gemm<128, 2>(s, blocks, prods, st);
    else if (blocks > 256) ns_launch_gemm<64, 2>(s, blocks, prods, st);        // two blocks per compute unit
    else ns_launch_gemm<64, 4>(s, blocks, prods, st);
  }
}

static void ns_launch_small(const std::vector<glx_matrix>& mats, int dtype, int steps, const double* c, double eps, hipStream_t st) {
  for (size_t i = 0; i < mats.size(); i += NS_SMALLS) {
    NsSmalls s;
    memset(&s, 0, sizeof(s));
    s.steps = steps; s.dtype = dtype; s.eps = eps;
    for (int k = 0; k < 3; ++k) s.c[k] = c[k];
    int n = 0;
    for (size_t j = i; j < mats.size() && j < i + NS_SMALLS; ++j, ++n)
      s.mat[n] = NsSmall{mats[j].src, mats[j].dst, mats[j].ld_src, mats[j].ld_dst, mats[j].rows, mats[j].cols};
    hipLaunchKernelGGL(k_ns_small, dim3(n), dim3(1024), 0, st, s);
  }
}

struct NsBounds { std::vector<double> lam, p, h; double steepest; };       // of A, P and P A, step by step (ns_bounds)

// the launches of `count` matrices that share one workspace; their plans lie in it from place 0 on
static void ns_run(const glx_matrix* mats, int count, int dtype, int steps, const double* coefficients, double eps, const NsBounds& bound,
                   char* ws, hipStream_t st) {
  const float a = (float)coefficients[0], b = (float)coefficients[1], c = (float)coefficients[2];
  const std::vector<double>&lam = bound.lam, &pmax = bound.p, &hmax = bound.h;
  const double steepest = bound.steepest;
  std::vector<NsPlan> plans;
  size_t at = 256;
  // (a segment's Gram matrix loses its error times the slope squared per step: coefficients steeper than the usual ones, whose
  // 3.4445 keeps five bfloat16 steps below half a step of the result, take segments of one step)
  for (int i = 0; i < count; ++i) plans.push_back(ns_plan(mats[i].rows, mats[i].cols, dtype, steps, steepest > 4.0, at));
  auto qbound = [&](int s0, int s) { double v = 1; for (int i = s0; i <= s; ++i) v *= pmax[i]; return v; };

  for (int i = 0; i < count; i += NS_MATS) {           // |G|_F, then the planes
    NsMats s;
    memset(&s, 0, sizeof(s));
    s.dtype = dtype; s.eps = eps; s.steps = steps;
    double growth = 1.0;
    for (int k = 0; k < steps; ++k) {
      s.xb[k] = (float)sqrt(lam[k]); s.qb[k] = (float)fmin(growth, 1e30);
      growth *= pmax[k];
    }
    int nb = 0, tb = 0;
    for (int j = i; j < count && j < i + NS_MATS; ++j) {
      const NsPlan& p = plans[j];
      s.first[s.count] = nb; s.tfirst[s.count] = tb;
      NsMat& t = s.mat[s.count++];
      t.src = mats[j].src; t.ld = mats[j].ld_src;
      t.x = (_Float16*)(ws + p.x); t.xt = (_Float16*)(ws + p.xt[0]); t.parts = (double*)(ws + p.parts); t.xscale = (float*)(ws + p.xscale);
      t.rows = p.rows; t.cols = p.cols; t.mp = p.mp; t.np = p.np; t.tall = p.tall; t.nparts = p.nparts;
      nb += p.nparts; tb += p.mp / 64 * (p.np / 64);
    }
    hipLaunchKernelGGL(k_ns_norm, dim3(nb), dim3(256), 0, st, s);
    hipLaunchKernelGGL(k_ns_planes, dim3(tb), dim3(256), 0, st, s);
  }

  // every matrix's program as a list of stages; stage k of all matrices runs together
  std::vector<NsStage> stages;
  for (int i = 0; i < count; ++i) {
    const NsPlan& p = plans[i];
    // bfloat16: single products in the last two steps, where what they lose is no longer amplified (it comes to 1e-3 of the
    // result: 4096 x 4096 is 1.86e-3 off, 1.98e-3 where all singular values are alike, with split ones 1.66e-3, its rounding; 3.65
    // and 4.7 ms); segments of one step only, and matrices whose time is the products (smaller ones lose as much -- 24 x 360 2.0e-3
    // in all -- and gain nothing)
    auto last = [&](int s1) {
      return dtype == GLX_BF16 && p.seg == 1 && p.m > 1024 && s1 > steps - 2 && steps >= 4 && steepest <= 4.0;
    };
    // lo lo too: fp32 matrices on 64-wide tiles, whose time is latency and LDS (24 x 360: 0.7 to 0.8 of a plain fp32 product's
    // error, without 0.9)
    const int full = dtype == GLX_F32 && p.tile == 64 && p.xtile == 64 ? 4 : 3;
    size_t k = 0;
    auto stage = [&]() -> NsStage& {
      if (k == stages.size()) stages.emplace_back();
      return stages[k++];
    };
    auto planes = [](size_t o) { return (unsigned)(o / 256); };
    auto square = [&](size_t A, float as, size_t B, float bs, size_t out, float scale) {       // out = A B, symmetric
      NsOp o = {};
      o.a = planes(A); o.b = planes(B); o.out = planes(out);
      o.alpha = 1.f / (as * bs); o.scale = scale;
      o.mp = p.mp; o.np = p.mp; o.K = p.mp; o.kper = (unsigned short)(p.mp / NS_K); o.splits = 1; o.kind = NS_PLANES; o.sym = 1;
      return o;
    };
    size_t xt = p.xt[0], xt2 = p.xt[1];
    for (int s0 = 0; s0 < steps; s0 += p.seg) {
      const int s1 = s0 + p.seg < steps ? s0 + p.seg : steps;
      const unsigned xs = planes(p.xscale);
      float gs = ns_scale(lam[s0]);
      {                                                // A = X X^T
        NsOp o = {};
        o.a = o.b = planes(p.x);
        o.alpha = 1.f; o.scale = gs; o.xin = xs; o.xpow = 2; o.xstep = (unsigned char)s0;
        o.mp = o.np = p.mp; o.K = p.np; o.kper = (unsigned short)(p.kper / NS_K); o.splits = (unsigned short)p.splits; o.sym = 1;
        const int prods = last(s1) || (s0 == 0 && dtype != GLX_F32) ? 1 : full;
        if (p.splits > 1) {
          o.kind = NS_PARTIAL; o.out = planes(p.part);
          stage().add(p.tile, prods, o);
          NsOp j = {};
          j.a = planes(p.part); j.out = planes(p.g); j.scale = gs; j.mp = j.np = p.mp; j.splits = (unsigned short)p.splits;
          stage().join.push_back(j);
        } else {
          o.kind = NS_PLANES; o.out = planes(p.g);
          stage().add(p.tile, prods, o);
        }
      }
      size_t q = p.q[0];
      float qs = 0.f;
      for (int s = s0; s < s1; ++s) {
        const float ps = ns_scale(pmax[s]), hs = ns_scale(hmax[s]);
        const size_t P = p.p[(s - s0) & 1];
        NsOp o = square(p.g, gs, p.g, gs, P, ps);      // P = a I + b A + c A A
        o.alpha *= c; o.d = planes(p.g); o.beta = b / gs; o.diag = a;
        stage().add(p.tile, last(s1) ? 1 : full, o);
        if (s == s0) {
          q = P; qs = ps;
        } else {                                       // (beside H where a step follows)
          const float nqs = ns_scale(qbound(s0, s));
          const size_t nq = p.q[(s - s0) & 1];
          stage().add(p.tile, full, square(P, ps, q, qs, nq, nqs));
          q = nq; qs = nqs;
          --k;
        }
        if (s + 1 < s1) {
          stage().add(p.tile, full, square(P, ps, p.g, gs, p.h, hs));
          const float ngs = ns_scale(lam[s + 1]);
          stage().add(p.tile, full, square(p.h, hs, P, ps, p.g, ngs));
          gs = ngs;
        } else if (s > s0) {
          ++k;
        }
      }
      {                                                // X <- Q X
        NsOp o = {};
        o.a = planes(q); o.b = planes(xt);
        o.alpha = 1.f / qs; o.xin = xs; o.xpow = 1; o.xstep = (unsigned char)s0;
        o.mp = p.mp; o.np = p.np; o.K = p.mp; o.kper = (unsigned short)(p.mp / NS_K); o.splits = 1;
        if (s1 == steps) {
          o.kind = NS_FINAL; o.dst = mats[i].dst; o.ldd = mats[i].ld_dst;
          o.m = p.m; o.n = p.n; o.tall = (unsigned char)p.tall; o.dtype = (unsigned char)dtype;
        } else {
          o.kind = NS_XPLANES; o.out = planes(p.x); o.out2 = planes(xt2); o.xout = xs; o.xnext = (unsigned char)s1;
        }
        stage().add(p.xtile, last(s1) ? 1 : s0 == 0 && dtype != GLX_F32 ? 2 : full, o);
        const size_t y = xt; xt = xt2; xt2 = y;
      }
    }
  }
  for (auto& g : stages) {
    for (int t = 0; t < 2; ++t) {
      for (int n = 0; n < 4; ++n) ns_launch_ops(g.gemm[t][n], ws, t ? 128 : 64, n + 1, st);
    }
    ns_launch_ops(g.join, ws, 64, 0, st);
  }
}

extern "C" int glx_orthogonalize(const glx_matrix* list, int listed, int dtype, int steps, const double* coefficients, double eps,
                                 void* workspace, size_t workspace_bytes, void* stream) try {
  if (int rc = ns_check("glx_orthogonalize", list, listed, dtype, steps)) return rc;
  GLX_REQUIRE(coefficients && eps >= 0.0, "glx_orthogonalize: bad coefficients or eps");
  NsBounds bound;
  GLX_REQUIRE(ns_bounds(steps, coefficients, bound.lam, bound.p, bound.h),
              "glx_orthogonalize: these coefficients let singular values grow beyond the arithmetic's range");
  bound.steepest = 1.0;
  for (double p : bound.p) bound.steepest = fmax(bound.steepest, p);
  if (listed == 0) return GLX_OK;
  std::vector<glx_matrix> mats, small;
  size_t need = 256, bytes;
  for (int i = 0; i < listed; need = bytes > need ? bytes : need) i = ns_group(list, i, listed, dtype, steps, &bytes);
  for (int i = 0; i < listed; ++i) {
    GLX_REQUIRE(list[i].src && list[i].dst && list[i].ld_src >= list[i].cols && list[i].ld_dst >= list[i].cols,
                "glx_orthogonalize: matrix %d: null pointer or rows that overlap", i);
    (ns_small(list[i]) ? small : mats).push_back(list[i]);
  }
  GLX_REQUIRE(need < (1ull << 40), "glx_orthogonalize: a matrix needs a workspace of %zu bytes", need);
  if (!workspace || workspace_bytes < need) {
    glx_set_error("glx_orthogonalize: workspace %zu < %zu bytes", workspace_bytes, need);
    return GLX_EWORKSPACE;
  }
  GLX_REQUIRE(((uintptr_t)workspace & 15) == 0, "glx_orthogonalize: the workspace must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  ns_launch_small(small, dtype, steps, coefficients, eps, st);
  const int count = (int)mats.size();
  for (int i = 0, to; i < count; i = to) {
    to = ns_group(mats.data(), i, count, dtype, steps, &bytes);
    ns_run(mats.data() + i, to - i, dtype, steps, coefficients, eps, bound, (char*)workspace, st);
  }
  GLX_LAUNCH_CHECK();
  return GLX_OK;
} catch (const std::exception& e) {
  glx_set_error("glx_orthogonalize: %s", e.what());
  return GLX_EINVAL;
}
