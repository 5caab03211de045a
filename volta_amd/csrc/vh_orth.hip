// vh_orth.hip -- the orthogonalised update: a few steps of the quintic Newton-Schulz
// iteration that takes a matrix's singular values towards 1 and keeps its singular
// vectors, and the optimiser step around it.
//
// With X0 = G / (|G|_F + eps), m <= n (a tall G is taken transposed), each step is
//   A = X X^T,  B = b A + c A A,  X <- a X + B X        (a, b, c) = (3.4445, -4.7750, 2.0315)
// three matrix products of m x m x n, m x m x m and m x m x n; A and B are symmetric, so
// of the first two only the tiles on and below the diagonal are computed.  Bound by the
// matrix cores for large matrices, by the launches and each product's depth for small.
//
// Numbers.  The singular values stay below 1.21, so everything fits fp16 with a fixed
// power-of-two scale, and fp16's 11 bits are 8 times as fine as bf16's at the same MFMA
// rate.  X is held as two fp16 planes, hi + lo (22 bits).
//  * fp32 matrices: every operand is a pair of planes and every product three MFMAs
//    (hi hi + hi lo + lo hi): the fp32 result at a third of the fp16 rate, where the
//    fp32 MFMA has a sixteenth.  Against 64 bits it is as far off as products in fp32
//    (512 x 512: 6.3e-6 both; singular values that start near 0 grow 485-fold, and
//    with them what rounding left there).
//  * bf16 matrices: one MFMA of hi planes, fp32 sums.  What each rounding costs: that of A
//    the most (its diagonal, near 1, is rounded alike in a whole row: 3.5e-3 off 64 bits
//    in the end), so the diagonals of A and B stay in fp32 and out of the products
//    (1.1e-3); a X comes from hi + lo: from hi alone, what rounding puts into the
//    directions that X lacks grows with the smallest singular values (rank 1: 9e-2
//    off; 2e-4 so), while B X does not let it through -- if the diagonal of B meets the same
//    hi as the rest of B does.  bf16 outputs are off by 1.65e-3 for their own rounding.
//    Small matrices (kFineElems) are computed as fp32 ones.
#include "vh_kernels.hpp"
#include "vh_tiles.hpp"

namespace vh {

namespace {

using namespace tiles;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
// Scales of the planes: X up to 1.21 * 2^13, A and B up to 3 * 2^13, both under 65504; lo's
// smallest step is 2^-24 / 2^13.
constexpr float kSX = 8192.f, kSA = 8192.f;

struct Planes {
  _Float16 *hi, *lo;
};

// hi + lo = v to 22 bits.  v is made a value of its own first: where the compiler folds the
// product that it comes from into the conversion, hi is rounded once in one place and
// twice in the other, and a tie in ten thousand leaves lo beside another hi.
__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  asm volatile("" : "+v"(v));
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

enum { kGram, kSquare, kApply, kLast };  // A = X X^T; B = b A + c A A; X' = a X + B X; the same, to the output

struct OrthArgs {
  const _Float16 *a[2], *b[2];  // hi and lo planes of the product's operands
  const float* diag;            // kSquare, kApply: the diagonal of A, of B
  const _Float16 *x[2];         // kSquare: A off its diagonal; kApply, kLast: X
  _Float16* out[2];
  float* diag_out;              // kGram, kSquare
  int rows;                     // of diag
  int K, lda, ldb, ldo;         // K a multiple of 64; ldo of x and out
  int tiles_m, tiles_n, tiles;  // tiles: blocks that have one
  long za, zb, zo, zd;          // from one matrix of a batch to the next (elements)
  int a_bytes, b_bytes;         // of one plane of one matrix
  // kLast
  void* dst;                    // [rows][cols] (fp32 if SPLIT, else bf16): dst = decay dst + step X'
  int tall, m, n;               // m x n of the iteration: tall, dst is n x m
  long zdst;
  float decay, step;
};

// 8 consecutive values of the output: dst = decay dst + step v, the first `n` of them
template <typename T>
__device__ __forceinline__ void write_out(const OrthArgs& g, size_t at, const float (&v)[8], int n) {
  using S = typename Elem<T>::storage;
  S* p = static_cast<S*>(g.dst) + at;
  S o[8];
  if (n >= 8) {
    if (g.decay != 0.f) __builtin_memcpy(o, p, sizeof(o));
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = Elem<T>::from_f32(g.decay != 0.f ? g.decay * Elem<T>::to_f32(o[e]) + g.step * v[e] : g.step * v[e]);
    __builtin_memcpy(p, o, sizeof(o));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = Elem<T>::from_f32(g.decay != 0.f ? g.decay * Elem<T>::to_f32(p[e]) + g.step * v[e] : g.step * v[e]);
  }
}

__device__ __forceinline__ void store8(_Float16* hi, _Float16* lo, const float (&v)[8]) {
  f16x8 h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    _Float16 a, b;
    split(v[e], a, b);
    h[e] = a;
    l[e] = b;
  }
  *reinterpret_cast<f16x8*>(hi) = h;
  if (lo) *reinterpret_cast<f16x8*>(lo) = l;
}

// what the lanes of a wave wrote to LDS before, they read after
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One BM x BN tile by NW waves of WM x WN each; where the tile has fewer than NW such
// parts, KS groups of waves share K.  Outputs are whole tiles (the planes are padded), so
// stores are not checked; where one plane has fewer rows of padding than a tile of the
// other, the copies' range check reads zeros past its end.  SPLIT: three MFMAs of the planes, from stages
// that hold both of each operand; where those would not fit (192 x 192 on), as three stages
// of the same k.
template <int BM, int BN, int WM, int WN, int NW, int NB, int MODE, bool SPLIT>
__global__ __launch_bounds__(NW * 64) void orth_kernel(OrthArgs g) {
  using TB = MnTile<bf16, BN>;
  constexpr bool BT = MODE >= kApply;  // X as stored: [K][n]
  using T = std::conditional_t<SPLIT, float, bf16>;
  constexpr int FM = WM / 32, FN = WN / 32, NWN = BN / WN;
  constexpr int WPG = (BM / WM) * (BN / WN), KS = NW / WPG;
  constexpr bool BOTH = SPLIT && BM < 192;  // both planes in a stage
  constexpr int PL = BOTH ? 2 : 1, P = SPLIT && !BOTH ? 3 : 1;
  constexpr int AC = BM / 8 / WPG, BC = BN / 8 / WPG, GP = (BM + BN) * 8, GS = GP * PL;
  static_assert(WPG * KS == NW && AC * WPG == BM / 8 && BC * WPG == BN / 8, "waves");
  extern __shared__ __attribute__((aligned(16))) u32x4g S[];

  const int tid = threadIdx.x, lane = tid & 63, row_l = lane & 31, half_l = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), grp = wv / WPG, wave = wv % WPG;
  const int wm = (wave / NWN) * WM, wn = (wave % NWN) * WN;
  const int lb = xcd_block((int)gridDim.x), z = blockIdx.z;  // a grid of whole eights: an XCD's blocks are neighbours
  if (lb >= g.tiles) return;
  int tm, tn;
  if constexpr (MODE <= kSquare) {  // tiles on and below the diagonal, in squares of 4 x 4
    int left = lb, row = 0;
    for (;; row += 4) {
      const int r = min(4, g.tiles_m - row), full = row * r;
      if (left < full) {  // square left / (4 r) of this row of squares
        const int q = left / (4 * r), in = left - q * 4 * r;
        tm = row + in / 4;
        tn = q * 4 + in % 4;
        break;
      }
      left -= full;
      if (left < r * (r + 1) / 2) {  // the one on the diagonal
        int i = 0;
        while (left > i) left -= ++i;
        tm = row + i;
        tn = row + left;
        break;
      }
      left -= r * (r + 1) / 2;
    }
  } else {  // groups of 8 row tiles share their columns of X in L2
    const int grp8 = lb / (8 * g.tiles_n), gm = min(g.tiles_m - grp8 * 8, 8), in = lb - grp8 * 8 * g.tiles_n;
    tm = grp8 * 8 + in % gm;
    tn = in / gm;
  }
  const int m0 = tm * BM, n0 = tn * BN;

  // copy instruction c: 64 units.  K-major: rows 8c .. 8c+7; MN-major: k rows (64 / UR) c ..
  int ua[AC], ub[BC];
#pragma unroll
  for (int i = 0; i < AC; ++i) {
    const int r = 8 * (wave + WPG * i) + (lane >> 3), u = (lane & 7) ^ ((r >> 1) & 7);
    ua[i] = ((m0 + r) * g.lda + 8 * u) * 2;
  }
#pragma unroll
  for (int i = 0; i < BC; ++i) {
    const int c = wave + WPG * i;
    if constexpr (BT) {
      const int kr = TB::RPI * c + lane / TB::UR, u = (lane % TB::UR) ^ TB::swz(kr);
      ub[i] = (kr * g.ldb + n0 + 8 * u) * 2;
    } else {
      const int r = 8 * c + (lane >> 3), u = (lane & 7) ^ ((r >> 1) & 7);
      ub[i] = ((n0 + r) * g.ldb + 8 * u) * 2;
    }
  }
  const __amdgpu_buffer_rsrc_t ar[2] = {rsrc_g(g.a[0] + z * g.za, g.a_bytes), rsrc_g(g.a[SPLIT] + z * g.za, g.a_bytes)};
  const __amdgpu_buffer_rsrc_t br[2] = {rsrc_g(g.b[0] + z * g.zb, g.b_bytes), rsrc_g(g.b[SPLIT] + z * g.zb, g.b_bytes)};
  const int nst = g.K / 64 * P;  // stages: P of each 64 k
  auto issue = [&](u32x4g* st, int sk) {
    const int s = sk * KS + grp;  // this group's stage; past the last one its copies read zeros
    const int kq = P == 3 ? s / 3 : s, p = P == 3 ? s - 3 * kq : 0, k0 = kq * 64;
    const int over = (nst - 1 - s) & kOORg;
    const int ask = k0 * 2, bsk = BT ? k0 * g.ldb * 2 : k0 * 2;
#pragma unroll
    for (int q = 0; q < PL; ++q) {
      const uint32_t la = lds_byte_addr(st) + (grp * GS + q * GP) * 16;
      const __amdgpu_buffer_rsrc_t ra = q || (P == 3 && p == 2) ? ar[1] : ar[0], rb = q || (P == 3 && p == 1) ? br[1] : br[0];
#pragma unroll
      for (int i = 0; i < AC; ++i) lds_copy16(ra, (ua[i] + ask) | over, 0, la + (wave + WPG * i) * 1024);
#pragma unroll
      for (int i = 0; i < BC; ++i) lds_copy16(rb, (ub[i] + bsk) | over, 0, la + BM * 128 + (wave + WPG * i) * 1024);
    }
  };
  struct Frags {
    bf16x8 a[PL][FM], b[PL][FN];  // bits of 8 fp16
  };
  auto read = [&](const u32x4g* st, int kk, Frags& f) {
#pragma unroll
    for (int q = 0; q < PL; ++q) {
      const char* at = reinterpret_cast<const char*>(st + grp * GS + q * GP);
      const char* bt = at + BM * 128;
#pragma unroll
      for (int i = 0; i < FM; ++i) f.a[q][i] = read_k<bf16>(at, wm + 32 * i, kk, lane);
      if constexpr (BT) {
        read_mn<bf16, BN, FN>(bt, wn, kk, lane, f.b[q]);
      } else {
#pragma unroll
        for (int j = 0; j < FN; ++j) f.b[q][j] = read_k<bf16>(bt, wn + 32 * j, kk, lane);
      }
    }
  };
  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
  auto mma = [&](const Frags& f) {
#pragma unroll
    for (int q = 0; q < 2 * PL - 1; ++q)  // hi hi, hi lo, lo hi
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const f16x8 a = __builtin_bit_cast(f16x8, f.a[q >> 1][i]), b = __builtin_bit_cast(f16x8, f.b[q & 1][j]);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc[i][j], 0, 0, 0);
        }
  };

  // copies of the next NB - 1 stages in flight, reads of the next step ahead of this one's MFMAs
  Frags fa, fb;
  const int ns = (nst + KS - 1) / KS;
#pragma unroll
  for (int i = 0; i < NB - 1; ++i)
    if (i < ns) issue(S + i * KS * GS, i);
  stage_sync<NB, (AC + BC) * PL>(ns - 1);
  read(S, 0, fa);
  for_stages<NB>(ns, [&](auto BUF, int s) {
    constexpr int B = decltype(BUF)::value;
    const u32x4g* cur = S + B * KS * GS;
    const u32x4g* nxt = S + (B + 1) % NB * KS * GS;
    if (s + NB - 1 < ns) issue(S + (B + NB - 1) % NB * KS * GS, s + NB - 1);
#pragma unroll
    for (int kk = 1; kk < 4; kk += 2) {
      read(cur, kk, fb);
      __builtin_amdgcn_sched_barrier(0);
      mma(fa);
      __builtin_amdgcn_sched_barrier(0);
      if (kk + 1 < 4) {
        read(cur, kk + 1, fa);
      } else if (s + 1 < ns) {
        stage_sync<NB, (AC + BC) * PL>(ns - 2 - s);
        read(nxt, 0, fa);
      }
      __builtin_amdgcn_sched_barrier(0);
      mma(fb);
      __builtin_amdgcn_sched_barrier(0);
    }
  });

  if constexpr (KS > 1) {  // the groups' sums, added in group order
    float* red = reinterpret_cast<float*>(S);
    constexpr int TILE = FM * FN * 1024;
    static_assert((KS - 1) * WPG * TILE * 4 <= NB * KS * GS * 16, "group sums exceed the stages");
    __syncthreads();
    if (grp > 0) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            red[((grp - 1) * WPG + wave) * TILE + ((i * FN + j) * 16 + v) * 64 + lane] = acc[i][j][v];
    }
    __syncthreads();
    if (grp == 0)
#pragma unroll
      for (int q = 0; q < KS - 1; ++q)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] += red[(q * WPG + wave) * TILE + ((i * FN + j) * 16 + v) * 64 + lane];
  }

  // Epilogue, 32 rows of the wave's part at a time through its own LDS: lanes come to hold
  // 8 consecutive columns of a row (16-byte loads and stores of the planes), and for the
  // tile across the diagonal or a tall output 8 consecutive rows of a column.  Both
  // walks and the accumulators' are free of bank conflicts with an odd row pitch.
  constexpr int EP = WN + 1, UPR = WN / 8;
  static_assert(WPG * 32 * EP * 4 <= NB * KS * GS * 16, "epilogue rows exceed the stages");
  __syncthreads();  // the stages, or the groups' sums, are read
  if (grp > 0) return;
  float* e = reinterpret_cast<float*>(S) + wave * 32 * EP;
  // (asking for x ahead of the main loop, or a part a stage, changed no size by more than 2 %)
  const _Float16 *xh = MODE == kGram ? nullptr : g.x[0] + z * g.zo, *xl = MODE == kGram ? nullptr : g.x[1] + z * g.zo;
  _Float16 *oh = MODE == kLast ? nullptr : g.out[0] + z * g.zo, *ol = MODE == kLast ? nullptr : g.out[1] + z * g.zo;
  const float* diag = MODE == kGram ? nullptr : g.diag + z * g.zd;
  float* dout = MODE <= kSquare ? g.diag_out + z * g.zd : nullptr;
  const bool across = MODE <= kSquare ? tm != tn : MODE == kLast && g.tall;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int r0 = m0 + wm + 32 * i, c0 = n0 + wn;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) e[((v >> 2) * 8 + half_l * 4 + (v & 3)) * EP + 32 * j + row_l] = acc[i][j][v];
    wave_sync();
#pragma unroll
    for (int k = 0; k < 32 * UPR / 64; ++k) {
      const int u = k * 64 + lane, lr = u / UPR, lc = u % UPR * 8, r = r0 + lr, c = c0 + lc;
      const size_t o = (size_t)r * g.ldo + c;
      float v[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = e[lr * EP + lc + t];
      if constexpr (MODE == kGram) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          if (r == c + t) dout[r] = v[t] * (1.f / (kSX * kSX));
          v[t] = r == c + t ? 0.f : v[t] * (kSA / (kSX * kSX));
        }
        store8(oh + o, SPLIT ? ol + o : nullptr, v);
      } else if constexpr (MODE == kSquare) {
        const f16x8 h = *reinterpret_cast<const f16x8*>(xh + o);
        f16x8 l = {};
        if (SPLIT) l = *reinterpret_cast<const f16x8*>(xl + o);
        const float di = diag[r];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float x = SPLIT ? (float)h[t] + (float)l[t] : (float)h[t];  // scaled by kSA, as v comes to be
          v[t] = (kB + kC * (di + diag[c + t])) * x + v[t] * (kC / kSA);
          if (r == c + t) {
            dout[r] = v[t] * (1.f / kSA) + di * (kB + kC * di);
            v[t] = 0.f;
          }
        }
        store8(oh + o, SPLIT ? ol + o : nullptr, v);
      } else {
        const f16x8 h = *reinterpret_cast<const f16x8*>(xh + o);
        const f16x8 l = *reinterpret_cast<const f16x8*>(xl + o);
        const float di = r < g.rows ? diag[r] : 0.f;  // X may have more rows of zeros than B
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float x = (float)h[t] + (float)l[t];
          v[t] = kA * x + (di * (SPLIT ? x : (float)h[t]) + v[t] * (1.f / kSA));  // scaled by kSX
        }
        if constexpr (MODE == kApply) {
          store8(oh + o, ol + o, v);
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t) v[t] *= 1.f / kSX;
          if (!across && r < g.m && c < g.n) write_out<T>(g, z * g.zdst + (size_t)r * g.n + c, v, g.n - c);
        }
      }
      if ((MODE <= kSquare || MODE == kLast) && across) {
#pragma unroll
        for (int t = 0; t < 8; ++t) e[lr * EP + lc + t] = v[t];
      }
    }
    if ((MODE <= kSquare || MODE == kLast) && across) {
      wave_sync();
#pragma unroll
      for (int k = 0; k < 32 * UPR / 64; ++k) {
        const int u = k * 64 + lane, lc = u % WN, lr = u / WN * 8, r = r0 + lr, c = c0 + lc;
        float v[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = e[(lr + t) * EP + lc];
        if constexpr (MODE <= kSquare) {
          const size_t o = (size_t)c * g.ldo + r;
          store8(oh + o, SPLIT ? ol + o : nullptr, v);
        } else if (c < g.n && r < g.m) {
          write_out<T>(g, z * g.zdst + (size_t)c * g.m + r, v, g.m - r);
        }
      }
    }
    wave_sync();
  }
}

// ---------------------------------------------------------------- the first planes
struct LoadArgs {
  const void* g;      // the gradient
  float* mom;         // momentum, or null: the matrix is g itself
  float beta;
  int nesterov;
  double* part;       // [batch][parts] sums of squares
  int parts, rows, cols;
  long z;             // elements of a matrix
  _Float16* out[2];
  int ld;             // their row
  long zo;
  float eps;
};

// 8 consecutive elements of a matrix of p.z, from i on; zeros past its end (`n` of them are in it)
template <typename T>
__device__ __forceinline__ void read8(const typename Elem<T>::storage* p, long n, float (&v)[8]) {
  typename Elem<T>::storage o[8];
  if (n >= 8) {
    __builtin_memcpy(o, p, sizeof(o));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = Elem<T>::to_f32(o[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? Elem<T>::to_f32(p[e]) : 0.f;
  }
}
// What is orthogonalised, once the momentum is the new one
template <typename T>
__device__ __forceinline__ void update8(const LoadArgs& p, size_t i, long n, float (&v)[8]) {
  using S = typename Elem<T>::storage;
  if (!p.mom || p.nesterov) read8<T>(static_cast<const S*>(p.g) + i, n, v);
  if (p.mom) {
    float m[8];
    read8<float>(p.mom + i, n, m);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p.nesterov ? v[e] + p.beta * m[e] : m[e];
  }
}

// What takes a matrix of Frobenius norm sqrt(s) to planes of norm kSX: factor times two to the power k.  As
// one fp32 it would be infinite from entries of 1e-37 on and lose bits for norms past 1e41; in two,
// an entry is scaled by the power, which is exact, then rounded once.  Where there is nothing to divide by,
// zeros stay zeros.
struct Scale {
  float factor;
  int k;
  __device__ __forceinline__ float operator()(float v) const { return __builtin_amdgcn_ldexpf(v, k) * factor; }
};
__device__ __forceinline__ Scale scale_of(double s, float eps) {
  const double norm = sqrt(s) + (double)eps, d = norm == 0.0 ? 0.0 : (double)kSX / norm;
  return {(float)__builtin_amdgcn_frexp_mant(d), __builtin_amdgcn_frexp_exp(d)};
}

// mom = beta mom + v; v = what is orthogonalised
__device__ __forceinline__ void new_momentum8(const LoadArgs& p, size_t i, long n, float (&v)[8]) {
  float m[8];
  float* q = p.mom + i;
  read8<float>(q, n, m);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    m[e] = p.beta * m[e] + v[e];
    v[e] = p.nesterov ? v[e] + p.beta * m[e] : m[e];
  }
  if (n >= 8) {
    __builtin_memcpy(q, m, 32);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) q[e] = m[e];
  }
}

// The sum of squares of block blockIdx.x's share of a matrix, in double (no overflow, no
// loss in a long sum); with a momentum, mom = beta mom + g first.
template <typename T>
__global__ __launch_bounds__(256) void orth_norm_kernel(LoadArgs p) {
  using S = typename Elem<T>::storage;
  __shared__ double red[4];
  const size_t base = (size_t)blockIdx.z * p.z;
  double s = 0;
#pragma unroll 2
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 8; i < p.z; i += (long)gridDim.x * 2048) {
    float v[8];
    const long n = p.z - i;
    read8<T>(static_cast<const S*>(p.g) + base + i, n, v);
    if (p.mom) new_momentum8(p, base + i, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)v[e] * v[e];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) p.part[(size_t)blockIdx.z * p.parts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// A 64 x 64 tile of X0 = G / (|G| + eps) as planes, G transposed if tall, zeros outside.
template <typename T, bool TALL>
__global__ __launch_bounds__(256) void orth_load_kernel(LoadArgs p) {
  __shared__ double red[4];
  __shared__ float tile[TALL ? 64 : 1][65];
  const size_t base = (size_t)blockIdx.z * p.z;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const int r0 = TALL ? j0 : i0, c0 = TALL ? i0 : j0, lr = threadIdx.x >> 3, lc = (threadIdx.x & 7) * 8;
  float v[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = r0 + lr + 32 * k, c = c0 + lc;
    if (r < p.rows && c < p.cols) {
      update8<T>(p, base + (size_t)r * p.cols + c, p.cols - c, v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
    }
    if (TALL)
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[lr + 32 * k][lc + e] = v[k][e];
  }
  double s = 0;
  for (int i = threadIdx.x; i < p.parts; i += 256) s += p.part[(size_t)blockIdx.z * p.parts + i];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const Scale f = scale_of((red[0] + red[1]) + (red[2] + red[3]), p.eps);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = lr + 32 * k;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = f(TALL ? tile[lc + e][r] : v[k][e]);
    const size_t o = blockIdx.z * p.zo + (size_t)(i0 + r) * p.ld + j0 + lc;
    store8(p.out[0] + o, p.out[1] + o, v[k]);
  }
}

// ---------------------------------------------------------------- small matrices
// A matrix that fits one CU's LDS goes through all its steps in one block: the planes of
// X in chunks of 64 columns (MP rows of 128 bytes, the K-major tile of vh_tiles.hpp, read
// along its rows for A and by transposing reads for B X), A's and B's in one place after
// the other.  MP / 32 squared waves; a wave computes the 32 x 32 part of A and B that is
// its own, and of X every (MP / 32)-th one of its row: the waves of one column part meet
// at a barrier between reading X there and writing X' over it.
// Its steps are latency (64 x 64 fp32: 5 us each); the launches of the products above cost
// 4 us each, 17 of them.
struct SmallArgs {
  LoadArgs l;
  void* dst;
  int m, n, np, tall, steps;
  float decay, step;
};

// byte of element (i, j) of planes in chunks of MP rows
template <int MP>
__device__ __forceinline__ int small_at(int i, int j) {
  return (j >> 6) * MP * 128 + i * 128 + ((((j & 63) >> 3) ^ ((i >> 1) & 7)) * 16) + (j & 7) * 2;
}

// B operand of X' = B X: k rows 16 kk .. +15 of the 32 columns from col0 on of a chunk
__device__ __forceinline__ f16x8 small_read_x(const char* chunk, int col0, int kk, int lane) {
  typedef short v4i16 __attribute__((ext_vector_type(4)));
  typedef short v8i16 __attribute__((ext_vector_type(8)));
  const int kr = 16 * kk + 8 * (lane >> 5) + ((lane & 15) >> 2);
  const int u = (col0 >> 3) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  auto at = [&](int r) {
    return (__attribute__((address_space(3))) v4i16*)((const __attribute__((address_space(3))) char*)chunk + r * 128 +
                                                      ((u ^ ((r >> 1) & 7)) * 16) + 8 * (lane & 1));
  };
  const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(kr)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(kr + 4));
  const v8i16 w = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(f16x8, w);
}

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// 4 consecutive columns of the planes (BOTH: lo too) from byte `at` on
template <bool BOTH>
__device__ __forceinline__ void small_put4(char* const (&pl)[2], int at, const float (&v)[4]) {
  f16x4 h, o;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    _Float16 x, y;
    split(v[t], x, y);
    h[t] = x;
    o[t] = y;
  }
  *reinterpret_cast<f16x4*>(pl[0] + at) = h;
  if (BOTH) *reinterpret_cast<f16x4*>(pl[1] + at) = o;
}

// lanes hold rows, registers columns: register 4 q + t of a part whose columns start at c0 is
// column c0 + 8 q + 4 (lane / 32) + t
template <bool SPLIT>
__device__ __forceinline__ void small_mma(f32x16& acc, const f16x8 (&a)[2], const f16x8 (&b)[2]) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[0], a[0], acc, 0, 0, 0);
  if (SPLIT) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[1], a[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[0], a[1], acc, 0, 0, 0);
  }
}
// 16 k from k on of 32 rows of a plane
template <int MP>
__device__ __forceinline__ f16x8 small_read_a(const char* plane, int row0, int k, int lane) {
  return __builtin_bit_cast(f16x8, read_k<bf16>(plane + (k >> 6) * MP * 128, row0, (k & 63) >> 4, lane));
}

// The wave's part of B = b A + c A A (scaled by kSA, without its diagonal, which goes to db)
template <bool SPLIT, int MP>
__device__ __forceinline__ void small_square(char* const (&A)[2], const float* da, float* db, f32x16& acc, int wi, int aj,
                                             int lane) {
  f16x8 a[2], b[2];
#pragma unroll
  for (int k = 0; k < MP; k += 16) {
#pragma unroll
    for (int q = 0; q < (SPLIT ? 2 : 1); ++q) {
      a[q] = small_read_a<MP>(A[q], wi * 32, k, lane);
      b[q] = small_read_a<MP>(A[q], aj, k, lane);
    }
    small_mma<SPLIT>(acc, a, b);
  }
  const int ri = wi * 32 + (lane & 31);
  const float di = da[ri];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = aj + 8 * q + 4 * (lane >> 5), at = small_at<MP>(ri, c);
    const f16x4 h = *reinterpret_cast<const f16x4*>(A[0] + at);
    f16x4 o = {};
    if (SPLIT) o = *reinterpret_cast<const f16x4*>(A[1] + at);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float v = (kB + kC * (di + da[c + t])) * ((float)h[t] + (float)o[t]) + acc[4 * q + t] * (kC / kSA);
      if (ri == c + t) db[ri] = v * (1.f / kSA) + di * (kB + kC * di);
      acc[4 * q + t] = ri == c + t ? 0.f : v;
    }
  }
}

// acc = a X + B X (scaled by kSX) of a part of X, from the product of B off its diagonal;
// c: the lane's first column
template <bool SPLIT, int MP>
__device__ __forceinline__ void small_apply(char* const (&X)[2], f32x16& acc, int ri, float di, int c) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int at = small_at<MP>(ri, c + 8 * q);
    const f16x4 h = *reinterpret_cast<const f16x4*>(X[0] + at), o = *reinterpret_cast<const f16x4*>(X[1] + at);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float x = (float)h[t] + (float)o[t];
      acc[4 * q + t] = kA * x + (di * (SPLIT ? x : (float)h[t]) + acc[4 * q + t] * (1.f / kSA));
    }
  }
}

// The groups' sums, in group order, in the first group's registers
template <int MP, int G>
__device__ __forceinline__ void small_group_sum(f32x16& acc, float* sums, int grp, int part, int lane) {
  if constexpr (G > 1) {
    for (int g = 1; g < G; ++g) {
      if (grp == g)
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[(part * 16 + v) * 64 + lane] = acc[v];
      __syncthreads();
      if (grp == 0)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[v] += sums[(part * 16 + v) * 64 + lane];
      __syncthreads();
    }
  }
}

// two planes of X; A's, or the fp32 sums of a group; two diagonals; the waves' sums of squares
template <bool SPLIT, int MP, int G>
constexpr int small_a_bytes() {
  return MP * MP * (SPLIT || G > 1 ? 4 : 2);
}
template <bool SPLIT, int MP, int G>
constexpr int small_lds(int np) {
  return MP * np * 4 + small_a_bytes<SPLIT, MP, G>() + MP * 8 + 256;
}

template <typename T, bool SPLIT, int MP, int G>
__global__ __launch_bounds__(64 * (MP / 32) * (MP / 32) * G) void orth_small_kernel(SmallArgs p) {
  using ST = typename Elem<T>::storage;
  constexpr int W = MP / 32, WAVES = W * W * G, THREADS = 64 * WAVES, PL = SPLIT ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  const int xb = MP * p.np * 2, ab = MP * MP * 2;
  char* X[2] = {sm, sm + xb};
  char* A[2] = {sm + 2 * xb, sm + 2 * xb + (PL - 1) * ab};
  float* sums = reinterpret_cast<float*>(sm + 2 * xb);
  float* da = reinterpret_cast<float*>(sm + 2 * xb + small_a_bytes<SPLIT, MP, G>());
  float* db = da + MP;
  double* red = reinterpret_cast<double*>(db + MP);
  const int tid = threadIdx.x, lane = tid & 63, row_l = lane & 31, half_l = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / (W * W), wi = wave % (W * W) / W, wj = wave % W;
  const LoadArgs& l = p.l;
  const size_t base = (size_t)blockIdx.x * l.z;

  for (int i = tid; i < xb / 8; i += THREADS) reinterpret_cast<u32x4g*>(sm)[i] = u32x4g{0, 0, 0, 0};  // both planes
  // the momentum and the sum of squares; a thread reads its own elements again below
  double s = 0;
#pragma unroll 4
  for (long i = tid * 8; i < l.z; i += THREADS * 8) {
    float v[8];
    const long n = l.z - i;
    read8<T>(static_cast<const ST*>(l.g) + base + i, n, v);
    if (l.mom) new_momentum8(l, base + i, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)v[e] * v[e];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  s = 0;
  for (int w = 0; w < WAVES; ++w) s += red[w];
  const Scale f = scale_of(s, l.eps);
  const int cols = p.tall ? p.m : p.n;  // of the matrix as it lies
  for (long i = tid * 8; i < l.z; i += THREADS * 8) {
    float v[8];
    update8<T>(l, base + i, l.z - i, v);
    int r = (int)i / cols, c = (int)i - r * cols;
    if (!p.tall && cols % 8 == 0) {
      const int at = small_at<MP>(r, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = f(v[e]);
      store8(reinterpret_cast<_Float16*>(X[0] + at), reinterpret_cast<_Float16*>(X[1] + at), v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (i + e < l.z) {
          const int at = p.tall ? small_at<MP>(c, r) : small_at<MP>(r, c);
          _Float16 h, q;
          split(f(v[e]), h, q);
          *reinterpret_cast<_Float16*>(X[0] + at) = h;
          *reinterpret_cast<_Float16*>(X[1] + at) = q;
        }
        if (++c == cols) c = 0, ++r;
      }
    }
  }
  __syncthreads();

  const int ri = wi * 32 + row_l, aj = wj * 32;
  auto col_of = [&](int c0, int q) { return c0 + 8 * q + 4 * half_l; };
  for (int step = 0; step < p.steps; ++step) {
    f32x16 acc = {};
    f16x8 a[2], b[2];
    for (int k = grp * 16; k < p.np; k += 16 * G) {  // A = X X^T
#pragma unroll
      for (int q = 0; q < PL; ++q) {
        a[q] = small_read_a<MP>(X[q], wi * 32, k, lane);
        b[q] = small_read_a<MP>(X[q], aj, k, lane);
      }
      small_mma<SPLIT>(acc, a, b);
    }
    small_group_sum<MP, G>(acc, sums, grp, wi * W + wj, lane);
    if (grp == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = col_of(aj, q);
        float v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          v[t] = acc[4 * q + t] * (kSA / (kSX * kSX));
          if (ri == c + t) {
            da[ri] = acc[4 * q + t] * (1.f / (kSX * kSX));
            v[t] = 0.f;
          }
        }
        small_put4<SPLIT>(A, small_at<MP>(ri, c), v);
      }
    }
    __syncthreads();
    acc = f32x16{};
    if (grp == 0) small_square<SPLIT, MP>(A, da, db, acc, wi, aj, lane);
    __syncthreads();  // A is read
    if (grp == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v[4] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        small_put4<SPLIT>(A, small_at<MP>(ri, col_of(aj, q)), v);
      }
    }
    __syncthreads();
    const float di = db[ri];
    for (int n0 = 0; n0 < p.np; n0 += MP * G) {  // X' = a X + B X, G column parts of MP at a time
      const int j0 = n0 + grp * MP + aj;
      const bool on = j0 < p.np;  // np is a multiple of MP: the same for a group
      acc = f32x16{};
      if (on) {
#pragma unroll
        for (int k = 0; k < MP; k += 16) {
#pragma unroll
          for (int q = 0; q < PL; ++q) {
            a[q] = small_read_a<MP>(A[q], wi * 32, k, lane);
            b[q] = small_read_x(X[q] + (j0 >> 6) * MP * 128, j0 & 63, k >> 4, lane);
          }
          small_mma<SPLIT>(acc, a, b);
        }
        small_apply<SPLIT, MP>(X, acc, ri, di, col_of(j0, 0));
      }
      __syncthreads();
      if (on && step + 1 < p.steps) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v[4] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
          small_put4<true>(X, small_at<MP>(ri, col_of(j0, q)), v);
        }
      } else if (on && ri < p.m) {
        ST* out = static_cast<ST*>(p.dst) + base;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = col_of(j0, v >> 2) + (v & 3);
          if (c < p.n) {
            ST* q = out + (p.tall ? (size_t)c * p.m + ri : (size_t)ri * p.n + c);
            const float x = p.step * (acc[v] * (1.f / kSX));
            *q = Elem<T>::from_f32(p.decay != 0.f ? p.decay * Elem<T>::to_f32(*q) + x : x);
          }
        }
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- short, wide matrices
// m <= 128 and more columns than a CU's LDS holds: a block takes a slice of X's columns,
// and a launch a whole step.  It adds up the slices' parts of A, computes B -- every
// block for itself: 128^3 at most --, then chunk by chunk of its columns X' = a X + B X and
// the part of A' = X' X'^T that they give.  One launch a step instead of three, and the
// long sum over n, which a few tiles of A would go through one after the other, is shared
// out (64 x 4096: 8 to 19 us a step for A alone).
struct SliceArgs {
  LoadArgs l;                  // first: the gradient, its norm's parts; l.out, l.ld, l.zo: X
  const float* part_in;        // [batch][slices][MP * MP] parts of A
  float* part_out;
  void* dst;                   // last: the output
  int m, n, chunks, per, slices, tall;  // chunks of X in all, of a block
  float decay, step;
};

template <bool SPLIT, int MP, int G>
constexpr int slice_lds() {
  return MP * MP * G * 4 + small_a_bytes<SPLIT, MP, G>() + MP * 8 + 256;
}

// FIRST: X from the gradient, no step.  LAST: X' to the output, no A'.
template <bool SPLIT, int MP, int G, bool FIRST, bool LAST>
__global__ __launch_bounds__(64 * (MP / 32) * (MP / 32) * G) void orth_slice_kernel(SliceArgs p) {
  using T = std::conditional_t<SPLIT, float, bf16>;
  using ST = typename Elem<T>::storage;
  constexpr int W = MP / 32, WAVES = W * W * G, THREADS = 64 * WAVES, PL = SPLIT ? 2 : 1;
  constexpr int CW = MP * G, XB = MP * CW * 2;  // columns of a chunk, bytes of its planes
  extern __shared__ __attribute__((aligned(16))) char sm[];
  char* X[2] = {sm, sm + XB};
  constexpr int ab = MP * MP * 2;
  char* A[2] = {sm + 2 * XB, sm + 2 * XB + (PL - 1) * ab};
  float* sums = reinterpret_cast<float*>(sm + 2 * XB);
  float* da = reinterpret_cast<float*>(sm + 2 * XB + small_a_bytes<SPLIT, MP, G>());
  float* db = da + MP;
  double* red = reinterpret_cast<double*>(db + MP);
  const int tid = threadIdx.x, lane = tid & 63, row_l = lane & 31, half_l = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / (W * W), wi = wave % (W * W) / W, wj = wave % W;
  const LoadArgs& l = p.l;
  const int z = blockIdx.y;
  const size_t base = (size_t)z * l.z;
  _Float16* gx[2] = {l.out[0] + z * l.zo, l.out[1] + z * l.zo};
  const int ri = wi * 32 + row_l, aj = wj * 32;
  auto col_of = [&](int c0, int q) { return c0 + 8 * q + 4 * half_l; };
  f16x8 a[2], b[2];
  Scale f{};
  float di = 0.f;

  if constexpr (FIRST) {
    double s = 0;
    for (int i = tid; i < l.parts; i += THREADS) s += l.part[(size_t)z * l.parts + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < WAVES; ++w) s += red[w];
    f = scale_of(s, l.eps);
  } else {
    // A: the slices' parts added in order
    const float* part = p.part_in + (size_t)z * p.slices * MP * MP;
    for (int u = tid; u < MP * MP / 4; u += THREADS) {
      f32x4 v = {};
#pragma unroll 8
      for (int q = 0; q < p.slices; ++q) v += reinterpret_cast<const f32x4*>(part + (size_t)q * MP * MP)[u];
      const int r = u / (MP / 4), c = u % (MP / 4) * 4;
      float w[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        w[t] = v[t] * (kSA / (kSX * kSX));
        if (r == c + t) {
          da[r] = v[t] * (1.f / (kSX * kSX));
          w[t] = 0.f;
        }
      }
      small_put4<SPLIT>(A, small_at<MP>(r, c), w);
    }
    __syncthreads();
    f32x16 acc = {};
    if (grp == 0) small_square<SPLIT, MP>(A, da, db, acc, wi, aj, lane);
    __syncthreads();  // A is read
    if (grp == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v[4] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        small_put4<SPLIT>(A, small_at<MP>(ri, col_of(aj, q)), v);
      }
    }
    __syncthreads();
    di = db[ri];
  }

  f32x16 gram = {};
  const int c_end = min((int)(blockIdx.x + 1) * p.per, p.chunks);
  for (int ch = blockIdx.x * p.per; ch < c_end; ++ch) {
    const int n0 = ch * CW;
    if constexpr (FIRST) {
      for (int u = tid; u < MP * CW / 8; u += THREADS) {  // 8 consecutive elements of the gradient
        float v[8];
        const int across = p.tall ? MP / 8 : CW / 8, o = u / across, e0 = u % across * 8;
        const int r = p.tall ? e0 : o, c = p.tall ? n0 + o : n0 + e0;  // of X
        const int left = p.tall ? p.m - r : p.n - c;
        if (left > 0 && r < p.m && c < p.n) {
          update8<T>(l, base + (p.tall ? (size_t)c * p.m + r : (size_t)r * p.n + c), left, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.f;
        }
        if (!p.tall) {
          const int at = small_at<MP>(r, e0);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = f(v[e]);
          store8(reinterpret_cast<_Float16*>(X[0] + at), reinterpret_cast<_Float16*>(X[1] + at), v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = small_at<MP>(r + e, o);
            _Float16 h, q;
            split(f(v[e]), h, q);
            *reinterpret_cast<_Float16*>(X[0] + at) = h;
            *reinterpret_cast<_Float16*>(X[1] + at) = q;
          }
        }
      }
    } else {
#pragma unroll
      for (int u = tid; u < MP * CW / 8; u += THREADS) {
        const int r = u / (CW / 8), c = u % (CW / 8) * 8, at = small_at<MP>(r, c);
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<f16x8*>(X[q] + at) = *reinterpret_cast<const f16x8*>(gx[q] + (size_t)r * l.ld + n0 + c);
      }
    }
    __syncthreads();
    if constexpr (!FIRST) {
      const int j0 = grp * MP + aj;  // X' = a X + B X
      f32x16 acc = {};
#pragma unroll
      for (int k = 0; k < MP; k += 16) {
#pragma unroll
        for (int q = 0; q < PL; ++q) {
          a[q] = small_read_a<MP>(A[q], wi * 32, k, lane);
          b[q] = small_read_x(X[q] + (j0 >> 6) * MP * 128, j0 & 63, k >> 4, lane);
        }
        small_mma<SPLIT>(acc, a, b);
      }
      small_apply<SPLIT, MP>(X, acc, ri, di, col_of(j0, 0));
      __syncthreads();  // X is read
      if constexpr (LAST) {
        ST* out = static_cast<ST*>(p.dst) + base;
        if (ri < p.m)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int c = n0 + col_of(j0, v >> 2) + (v & 3);
            if (c < p.n) {
              ST* q = out + (p.tall ? (size_t)c * p.m + ri : (size_t)ri * p.n + c);
              const float x = p.step * (acc[v] * (1.f / kSX));
              *q = Elem<T>::from_f32(p.decay != 0.f ? p.decay * Elem<T>::to_f32(*q) + x : x);
            }
          }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v[4] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
          small_put4<true>(X, small_at<MP>(ri, col_of(j0, q)), v);
        }
        __syncthreads();
      }
    }
    if constexpr (!LAST) {
      for (int k = grp * 16; k < CW; k += 16 * G) {
#pragma unroll
        for (int q = 0; q < PL; ++q) {
          a[q] = small_read_a<MP>(X[q], wi * 32, k, lane);
          b[q] = small_read_a<MP>(X[q], aj, k, lane);
        }
        small_mma<SPLIT>(gram, a, b);
      }
      for (int u = tid; u < MP * CW / 8; u += THREADS) {
        const int r = u / (CW / 8), c = u % (CW / 8) * 8, at = small_at<MP>(r, c);
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<f16x8*>(gx[q] + (size_t)r * l.ld + n0 + c) = *reinterpret_cast<const f16x8*>(X[q] + at);
      }
      __syncthreads();  // X is read
    }
  }
  if constexpr (!LAST) {
    small_group_sum<MP, G>(gram, sums, grp, wi * W + wj, lane);
    if (grp == 0) {
      float* out = p.part_out + ((size_t)z * p.slices + blockIdx.x) * MP * MP;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(out + ri * MP + col_of(aj, q)) = f32x4{gram[4 * q], gram[4 * q + 1], gram[4 * q + 2], gram[4 * q + 3]};
    }
  }
}

// ---------------------------------------------------------------- launches
template <int BM, int BN, int WM, int WN, int NW, int NB, int MODE, bool SPLIT>
int launch(const OrthArgs& g, int batch, hipStream_t st) {
  auto kern = orth_kernel<BM, BN, WM, WN, NW, NB, MODE, SPLIT>;
  constexpr int KS = NW / ((BM / WM) * (BN / WN)), BYTES = NB * KS * (BM + BN) * 128 * (SPLIT && BM < 192 ? 2 : 1);
  static_assert(BYTES <= 160 * 1024, "LDS");
  VH_LDS_LIMIT_ONCE(kern);
  OrthArgs a = g;
  a.tiles = MODE <= kSquare ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
  kern<<<dim3((unsigned)(a.tiles + 7) / 8 * 8, 1, (unsigned)batch), NW * 64, BYTES, st>>>(a);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

// Tiles.  A product's time goes by its tiles a CU: us of m x m x K (lower half) and m x m x n
// products, one matrix, bf16 (fp32), by tile:
//               32        64 in 2 K groups   64        128        192        256
//   512, 4096   8.4 (19)  13 (35)            16 (44)   27 (68)    --         --     A = X X^T
//   1024, 4096  27 (57)   15 (36)            19 (45)   29 (70)    --         --
//   2304, 2304  --        38 (76)            29 (69)   25 (54)    35 (95)    69      B
//   3456, 3456  --        --                 --        70 (172)   62 (154)   --
//   4096, 4096  --        --                 --       115 (275)   82 (215)   95 (262)
//   5376, 5376  --        --                 --       183 (512)  167 (462)  144 (411)
//   512 x 1024  7.0 (9.8) 5.0 (6.8)          5.2 (7.7) 7.6 (12)   --         --     B X
//   512 x 4096  24 (35)   9.7 (13)           7.1 (11)  8.8 (14)   --         --
//   2048 x 2048 --        39 (92)            33 (76)   28 (57)    --         53 (129)
//   4096 x 4096 --        --                 --       168 (398)   --        138 (364)
// so: the smallest ones (and K split over groups of waves) while they fit the chip at
// once; 64 x 64 while those that a CU holds (three in bf16, two in fp32) nearly do; then
// the least time of rounds of 128 (1), 192 (2: of 4096 rows 253 tiles, where 256 x 256 are
// 136) and 256 (2.6).  192 are for the symmetric products, whose operands both lie along
// K: rows of 192 columns are no whole copy instructions.
enum { kT32 = 32, kT64K = 1, kT64 = 64, kT128 = 128, kT192 = 192, kT256 = 256 };
int tile_rows(int tile) { return tile == kT64K ? 64 : tile; }
// of `rows` x `cols` outputs (`sym`: the tiles on and below the diagonal)
int pick_tile(long rows, long cols, bool sym, long batch, bool fp32) {
  auto tiles = [&](long t) {
    const long a = (rows + t - 1) / t, b = (cols + t - 1) / t;
    return batch * (sym ? a * (a + 1) / 2 : a * b);
  };
  if (tiles(32) <= 256) return kT32;
  if (tiles(64) <= 256) return kT64K;
  if (tiles(64) <= (fp32 ? 512 : 600)) return kT64;
  auto cost = [&](long t, long w) { return (tiles(t) + 255) / 256 * w; };
  const long c128 = cost(128, 5), c192 = sym ? cost(192, 10) : c128 + 1, c256 = cost(256, 13);
  return c256 < std::min(c192, c128 + 1) ? kT256 : c192 <= c128 ? kT192 : kT128;
}

template <int MODE, bool SPLIT>
int product(OrthArgs g, int tile, int rows, int cols, int batch, hipStream_t st) {
  const int t = tile_rows(tile);
  g.tiles_m = rows / t;
  g.tiles_n = cols / t;
  constexpr int NB = SPLIT ? 2 : 3;
  switch (tile) {
    case kT32: return launch<32, 32, 32, 32, 4, NB, MODE, SPLIT>(g, batch, st);
    case kT64K: return launch<64, 64, 32, 32, 8, NB, MODE, SPLIT>(g, batch, st);
    case kT64: return launch<64, 64, 32, 32, 4, NB, MODE, SPLIT>(g, batch, st);
    case kT128: return launch<128, 128, 64, 32, 8, NB, MODE, SPLIT>(g, batch, st);
    case kT192:
      if constexpr (MODE <= kSquare) return launch<192, 192, 96, 32, 12, 3, MODE, SPLIT>(g, batch, st);
      return VH_ERR_UNSUPPORTED;
    default: return launch<256, 256, 128, 64, 8, 2, MODE, SPLIT>(g, batch, st);
  }
}

// Rows of the one-block kernel that takes an m x n matrix (0: none), its columns in *np
int small_rows(long m, long n, int* np) {
  const int mp = m <= 64 ? 64 : 128;
  if (m > 128 || n > (mp == 64 ? 512 : 128)) return 0;
  *np = (int)((n + mp - 1) / mp * mp);
  return mp;
}

template <typename T, bool SPLIT, int MP, int G>
int launch_small(const SmallArgs& a, long batch, hipStream_t st) {
  auto kern = orth_small_kernel<T, SPLIT, MP, G>;
  VH_LDS_LIMIT_ONCE(kern);
  kern<<<dim3((unsigned)batch), 64 * (MP / 32) * (MP / 32) * G, small_lds<SPLIT, MP, G>(a.np), st>>>(a);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

// The slices of m <= 128 rows, wider than the above: chunks of a matrix, of a block, blocks
struct SlicePlan {
  int mp, np, chunks, per, slices;
  size_t per_matrix;
};
bool slice_plan(long m, long n, long batch, SlicePlan* o) {
  if (m > 128) return false;
  o->mp = m <= 64 ? 64 : 128;
  const int cw = o->mp == 64 ? 256 : 128;
  o->chunks = (int)((n + cw - 1) / cw);
  o->np = o->chunks * cw;
  // a block for each CU and chunk, but at most 16 parts of A to add up in every block
  const long most = std::min<long>(16, std::max<long>(1, 256 / batch));
  o->per = (int)((o->chunks + most - 1) / most);
  o->slices = (o->chunks + o->per - 1) / o->per;
  o->per_matrix = (size_t)o->mp * o->np * 4 + (size_t)o->slices * o->mp * o->mp * 8;
  return true;
}

template <bool SPLIT, int MP, int G, bool FIRST, bool LAST>
int launch_slice(const SliceArgs& a, long batch, hipStream_t st) {
  auto kern = orth_slice_kernel<SPLIT, MP, G, FIRST, LAST>;
  VH_LDS_LIMIT_ONCE(kern);
  kern<<<dim3((unsigned)a.slices, (unsigned)batch), 64 * (MP / 32) * (MP / 32) * G, slice_lds<SPLIT, MP, G>(), st>>>(a);
  VH_LAUNCH_CHECK();
  return VH_OK;
}
template <bool SPLIT, int MP, int G>
int run_slices(SliceArgs a, float* (&part)[2], int steps, long batch, hipStream_t st) {
  a.part_out = part[0];
  int r = launch_slice<SPLIT, MP, G, true, false>(a, batch, st);
  for (int s = 0; s < steps && r == VH_OK; ++s) {
    a.part_in = part[s & 1];
    a.part_out = part[(s + 1) & 1];
    r = s + 1 < steps ? launch_slice<SPLIT, MP, G, false, false>(a, batch, st)
                      : launch_slice<SPLIT, MP, G, false, true>(a, batch, st);
  }
  return r;
}

struct OrthPlan {
  long m, n, mp, np, ma;  // X in mp x np, A and B in ma x ma
  int tile_a, tile_x;  // of the m x m products, of the m x n ones
  size_t x_plane, a_plane;
  size_t per_matrix;   // bytes of its planes
};

OrthPlan plan_of(long rows, long cols, long batch, bool fp32) {
  OrthPlan o{};
  o.m = std::min(rows, cols);
  o.n = std::max(rows, cols);
  auto up = [](long v, long t) { return (v + t - 1) / t * t; };
  o.tile_a = pick_tile(o.m, o.m, true, batch, fp32);
  o.tile_x = pick_tile(o.m, o.n, false, batch, fp32);
  // whole tiles of each product's outputs, and whole stages of 64 k
  o.ma = up(o.m, std::max(64, tile_rows(o.tile_a)));
  o.mp = up(o.m, std::max(64, tile_rows(o.tile_x)));
  o.np = up(o.n, std::max(64, tile_rows(o.tile_x)));
  o.x_plane = (size_t)o.mp * o.np;
  o.a_plane = (size_t)o.ma * o.ma;
  o.per_matrix = (o.x_plane + o.a_plane) * 8;
  return o;
}

// bf16 matrices of fewer elements are computed with both planes, as fp32 ones: the roundings of one plane
// average over a matrix's entries, and where there are few, were up to 1.7e-2 of a 2 x 3 result, 3.3e-3 of
// 16 x 16, 2.7e-3 of 32 x 32 (the largest of 2000; 2.4e-3 at 64 x 64, 2.2e-3 at 128 x 128), of which the output's
// rounding is 1.7e-3.  It costs 22 us for 18 (16 of 16 x 16), 49 for 39 (of 2 x 500).
constexpr long kFineElems = 4096;

constexpr size_t kOrthMostWs = (size_t)1 << 30;

// The buffers of `nb` matrices in a workspace, each from a multiple of 256 bytes on
struct OrthCarve {
  size_t off[12], total = 0;
  int n = 0;
  void take(size_t bytes) {
    off[n++] = total;
    total += (bytes + 255) & ~(size_t)255;
  }
};
int norm_parts(long elems) { return (int)std::min<long>(std::max<long>(elems / 2048, 1), 512); }
OrthCarve carve(const SlicePlan& o, long nb, int parts) {  // X hi, lo; A's parts of two steps; the norm's
  OrthCarve c;
  for (int p = 0; p < 2; ++p) c.take((size_t)o.mp * o.np * 2 * nb);
  for (int p = 0; p < 2; ++p) c.take((size_t)o.slices * o.mp * o.mp * 4 * nb);
  c.take((size_t)parts * 8 * nb);
  return c;
}
OrthCarve carve(const OrthPlan& o, long nb, int parts) {  // X and X' hi, lo; A and B hi, lo; their diagonals; the norm's
  OrthCarve c;
  for (int p = 0; p < 4; ++p) c.take(o.x_plane * 2 * nb);
  for (int p = 0; p < 4; ++p) c.take(o.a_plane * 2 * nb);
  for (int p = 0; p < 2; ++p) c.take((size_t)o.ma * 4 * nb);
  c.take((size_t)parts * 8 * nb);
  return c;
}

}  // namespace

// Matrices of a batch that go together: as many as 1 GiB of workspace holds, at least one.
static long orth_chunk(long rows, long cols, long batch, bool fp32) {
  SlicePlan sp;
  const size_t one = slice_plan(std::min(rows, cols), std::max(rows, cols), 1, &sp) ? sp.per_matrix : plan_of(rows, cols, 1, fp32).per_matrix;
  return std::max<long>(1, std::min<long>(std::min<long>(batch, 65535), (long)(kOrthMostWs / one)));
}

bool orth_ok(long rows, long cols) {  // planes of less than 2^31 bytes
  const long mp = rows + 256, np = cols + 256;
  return mp * np < 1L << 30 && std::min(mp, np) * std::min(mp, np) < 1L << 30;
}

// What the turns of a call take: all but the last have orth_chunk's matrices, the last the
// rest, which may go on other tiles, with other padding, or in other slices.
size_t orth_ws(int dtype, long rows, long cols, long batch) {
  const long m = std::min(rows, cols), n = std::max(rows, cols);
  int np;
  if (small_rows(m, n, &np)) return 0;
  const bool fp32 = dtype == VH_F32;
  const long c = orth_chunk(rows, cols, batch, fp32);
  auto need = [&](long nb) {
    SlicePlan sp;
    if (!nb) return (size_t)0;
    return slice_plan(m, n, nb, &sp) ? carve(sp, nb, norm_parts(rows * cols)).total
                                     : carve(plan_of(rows, cols, nb, fp32), nb, norm_parts(rows * cols)).total;
  };
  return std::max(need(c), need(batch % c));
}

template <typename T>
int run_orth(const OrthCall& q, char* ws, hipStream_t st) {
  constexpr bool SPLIT = std::is_same<T, float>::value;
  const long chunk = orth_chunk(q.rows, q.cols, q.batch, SPLIT), z = q.rows * q.cols;
  const bool tall = q.rows > q.cols;
  SmallArgs sa{};
  if (const int mp = small_rows(std::min(q.rows, q.cols), std::max(q.rows, q.cols), &sa.np)) {
    sa.l.g = q.grad;
    sa.l.mom = q.momentum;
    sa.l.beta = q.beta;
    sa.l.nesterov = q.nesterov;
    sa.l.z = z;
    sa.l.eps = q.eps;
    sa.dst = q.out;
    sa.m = (int)std::min(q.rows, q.cols);
    sa.n = (int)std::max(q.rows, q.cols);
    sa.tall = tall;
    sa.steps = q.steps;
    sa.decay = q.decay;
    sa.step = q.step;
    if (mp == 128) return launch_small<T, SPLIT, 128, 1>(sa, q.batch, st);
    if (SPLIT || z >= kFineElems) return sa.np == 64 ? launch_small<T, SPLIT, 64, 1>(sa, q.batch, st) : launch_small<T, SPLIT, 64, 4>(sa, q.batch, st);
    return sa.np == 64 ? launch_small<T, true, 64, 1>(sa, q.batch, st) : launch_small<T, true, 64, 4>(sa, q.batch, st);
  }
  for (long at = 0; at < q.batch; at += chunk) {
    const long nb = std::min(chunk, q.batch - at);
    LoadArgs l{};
    l.g = static_cast<const char*>(q.grad) + (size_t)at * z * sizeof(typename Elem<T>::storage);
    l.mom = q.momentum ? q.momentum + at * z : nullptr;
    l.beta = q.beta;
    l.nesterov = q.nesterov;
    l.parts = norm_parts(z);
    l.rows = (int)q.rows;
    l.cols = (int)q.cols;
    l.z = z;
    l.eps = q.eps;
    void* dst = static_cast<char*>(q.out) + (size_t)at * z * sizeof(typename Elem<T>::storage);
    const auto norm = [&] {
      orth_norm_kernel<T><<<dim3((unsigned)l.parts, 1, (unsigned)nb), 256, 0, st>>>(l);
      VH_LAUNCH_CHECK();
      return (int)VH_OK;
    };
    SlicePlan sp;
    if (slice_plan(std::min(q.rows, q.cols), std::max(q.rows, q.cols), nb, &sp)) {
      SliceArgs a{};
      const OrthCarve w = carve(sp, nb, l.parts);
      for (int p = 0; p < 2; ++p) l.out[p] = (_Float16*)(ws + w.off[p]);
      float* part[2] = {(float*)(ws + w.off[2]), (float*)(ws + w.off[3])};
      l.part = (double*)(ws + w.off[4]);
      l.ld = sp.np;
      l.zo = (long)sp.mp * sp.np;
      a.l = l;
      a.dst = dst;
      a.m = (int)std::min(q.rows, q.cols);
      a.n = (int)std::max(q.rows, q.cols);
      a.chunks = sp.chunks;
      a.per = sp.per;
      a.slices = sp.slices;
      a.tall = tall;
      a.decay = q.decay;
      a.step = q.step;
      int r = norm();
      if (r == VH_OK) r = sp.mp == 64 ? run_slices<SPLIT, 64, 4>(a, part, q.steps, nb, st) : run_slices<SPLIT, 128, 1>(a, part, q.steps, nb, st);
      if (r != VH_OK) return r;
      continue;
    }
    const OrthPlan o = plan_of(q.rows, q.cols, nb, SPLIT);
    const OrthCarve w = carve(o, nb, l.parts);
    _Float16 *x[2][2], *a[2][2];
    for (int i = 0; i < 4; ++i) {
      x[i >> 1][i & 1] = (_Float16*)(ws + w.off[i]);
      a[i >> 1][i & 1] = (_Float16*)(ws + w.off[4 + i]);
    }
    float* diag[2] = {(float*)(ws + w.off[8]), (float*)(ws + w.off[9])};
    l.part = (double*)(ws + w.off[10]);
    l.out[0] = x[0][0];
    l.out[1] = x[0][1];
    l.ld = (int)o.np;
    l.zo = (long)o.x_plane;
    if (const int r = norm()) return r;
    const dim3 grid((unsigned)(o.np / 64), (unsigned)(o.mp / 64), (unsigned)nb);
    if (tall) orth_load_kernel<T, true><<<grid, 256, 0, st>>>(l);
    else orth_load_kernel<T, false><<<grid, 256, 0, st>>>(l);
    VH_LAUNCH_CHECK();
    OrthArgs sq{}, ap{}, gr{};
    const int mp = (int)o.mp, np = (int)o.np, ma = (int)o.ma, mk = (int)((o.m + 63) / 64 * 64);
    for (int s = 0; s < q.steps; ++s) {
      _Float16 **xi = x[s & 1], **xo = x[(s + 1) & 1];
      gr.K = np;
      gr.lda = gr.ldb = np;
      gr.ldo = ma;
      gr.za = gr.zb = (long)o.x_plane;
      gr.zo = (long)o.a_plane;
      gr.zd = gr.rows = ma;
      gr.a_bytes = gr.b_bytes = (int)(o.x_plane * 2);
      sq = ap = gr;
      for (int p = 0; p < 2; ++p) {
        gr.a[p] = gr.b[p] = xi[p];
        gr.out[p] = a[0][p];
        sq.a[p] = sq.b[p] = sq.x[p] = a[0][p];
        sq.out[p] = a[1][p];
        ap.a[p] = a[1][p];
        ap.b[p] = ap.x[p] = xi[p];
        ap.out[p] = xo[p];
      }
      gr.diag_out = diag[0];
      sq.diag = diag[0];
      sq.diag_out = diag[1];
      ap.diag = diag[1];
      sq.K = ap.K = mk;
      sq.lda = sq.ldb = ap.lda = ma;
      sq.za = sq.zb = ap.za = (long)o.a_plane;
      sq.a_bytes = sq.b_bytes = ap.a_bytes = (int)(o.a_plane * 2);
      ap.ldo = np;
      ap.zo = (long)o.x_plane;
      int r = product<kGram, SPLIT>(gr, o.tile_a, ma, ma, (int)nb, st);
      if (r == VH_OK) r = product<kSquare, SPLIT>(sq, o.tile_a, ma, ma, (int)nb, st);
      if (r != VH_OK) return r;
      if (s + 1 < q.steps) {
        r = product<kApply, SPLIT>(ap, o.tile_x, mp, np, (int)nb, st);
      } else {
        ap.dst = dst;
        ap.tall = tall;
        ap.m = (int)o.m;
        ap.n = (int)o.n;
        ap.zdst = z;
        ap.decay = q.decay;
        ap.step = q.step;
        r = product<kLast, SPLIT>(ap, o.tile_x, mp, np, (int)nb, st);
      }
      if (r != VH_OK) return r;
    }
  }
  return VH_OK;
}

// The plan of a turn of nb matrices: padded rows and columns, and whether each product has
// whole tiles and stages, every buffer an aligned place of its own, and every offset 31 bits
bool orth_info(int dtype, long rows, long cols, long batch, long nb) {
  const long m = std::min(rows, cols), n = std::max(rows, cols);
  const size_t bytes = orth_ws(dtype, rows, cols, batch);
  int np;
  if (const int mp = small_rows(m, n, &np)) return mp >= m && np >= n && np % mp == 0 && !bytes;
  SlicePlan sp;
  if (slice_plan(m, n, nb, &sp)) {
    const OrthCarve w = carve(sp, nb, norm_parts(rows * cols));
    return sp.mp >= m && sp.np >= n && (long)sp.slices * sp.per >= sp.chunks && (long)(sp.slices - 1) * sp.per < sp.chunks &&
           w.total <= bytes;
  }
  const OrthPlan o = plan_of(rows, cols, nb, dtype == VH_F32);
  const int ta = tile_rows(o.tile_a), tx = tile_rows(o.tile_x);
  return o.mp >= m && o.np >= n && o.ma >= m && o.ma % ta == 0 && o.mp % tx == 0 && o.np % tx == 0 && o.ma % 64 == 0 &&
         o.mp % 64 == 0 && o.np % 64 == 0 && o.x_plane * 2 < (size_t)1 << 31 && o.a_plane * 2 < (size_t)1 << 31 &&
         // rows past a plane's end: their offsets neither wrap round nor fall into it
         (size_t)(std::max(o.ma, o.mp)) * std::max(o.np, o.ma) * 2 < (size_t)1 << 32 && (o.tile_x != kT192) &&
         carve(o, nb, norm_parts(rows * cols)).total <= bytes;
}
long orth_turn(int dtype, long rows, long cols, long batch) { return orth_chunk(rows, cols, batch, dtype == VH_F32); }

template int run_orth<float>(const OrthCall&, char*, hipStream_t);
template int run_orth<bf16>(const OrthCall&, char*, hipStream_t);

}  // namespace vh
