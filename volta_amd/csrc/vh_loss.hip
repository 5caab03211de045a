// vh_loss.hip -- losses over a vocabulary and their gradients: token
// log-probabilities, the clipped policy loss with its KL term, the preference loss
// over pairs of sequences.
//
// With z_v = x_v / T of a row of logits, m = max z, s = sum exp(z - m), the taken
// token's log-probability is logp = z_tok - m - log s, and a loss L of the
// log-probabilities has dL/dx_v = dL/dlogp / T * (1[v = tok] - exp(z_v - m) / s).
// Nothing here multiplies matrices: the passes are bound by memory.  m, s and every
// sum are fp32 or wider; the gradient is rounded once, to the logits' type.
//
// Measured: the policy loss of 2048 rows of 32003 bf16, a quarter masked, in 64 us (3.5 TB/s
// read and written), of 4096 rows of 131072 in 435 (4.3); the preference loss of 3010 rows of
// 50021 in 66 + 6 + 102: its gradient needs every row's log-probability first, so the
// logits are read a second time (0.3 GB: more than the caches keep); 48 rows of 1000 in 6 + 2.3.
//
// Rows are walked as vh_rows.hpp has it, with 64-bit row offsets: the logits may pass
// 2^31 elements.
#include "vh_kernels.hpp"
#include "vh_rows.hpp"

namespace vh {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.925963033500941e-8f;
constexpr float kNegInf = -__builtin_huge_valf();

// exp(z - m) of a row whose largest value is m.  The difference is taken first: scaled
// by log2 e apart, two large values would lose it.  log2 e in fp32 is 1.3e-8 of itself short, the
// same way in every entry of every row: 4e-8 of a sum, which added up over the rows of a sequence
// to 2e-6 of a preference loss.  The second multiplication costs the bf16 passes 1 to 8 %; an
// entry of the gradient (grad_unit), rounded by itself, goes without.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(fmaf(d, kLog2e, d * kLog2eRest)); }

// Running maximum and sum of exponentials.  The maximum leaves NaN out (fmaxf); the
// sum takes it in, so a row with a NaN or an infinity ends as NaN.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float finite_or_0(float m) { return m == kNegInf ? 0.f : m; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m), f = finite_or_0(m);
  return {m, a.s * exp_of(a.m - f) + b.s * exp_of(b.m - f)};
}

template <typename T>
__device__ __forceinline__ void add_unit(MaxSum& a, const Unit<T>& u, float inv_t) {
#pragma clang fp contract(off)  // z is rounded as it is in m: the largest exponential is 1
  constexpr int VE = Unit<T>::VE;
  float z[VE], m = a.m;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    z[e] = u.get(e) * inv_t;
    m = fmaxf(m, z[e]);
  }
  const float f = finite_or_0(m);
  float s = a.s * exp_of(a.m - f);
#pragma unroll
  for (int e = 0; e < VE; ++e) s += exp_of(z[e] - f);
  a = {m, s};
}

// Of the whole row, in every one of its THREADS threads the same: the two sides of a join are
// rounded differently (the first product within a multiply-add), so the lanes of a wave end with
// sums that differ in their last bits.  The first lane's is taken, which in each wave
// is joined in the same order.
template <int THREADS>
__device__ __forceinline__ MaxSum block_join(MaxSum a, MaxSum* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const MaxSum b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o)};
    a = join(a, b);
  }
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    constexpr int W = THREADS / 64;
    a = red[threadIdx.x & (W - 1)];
#pragma unroll
    for (int o = W / 2; o; o >>= 1) {
      const MaxSum b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o)};
      a = join(a, b);
    }
  }
  auto first = [](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); };
  return {first(a.m), first(a.s)};
}

__device__ __forceinline__ bool tok_ok(long tok, int V) {
  return tok >= 0 && tok < V;
}

// logp of a row's token, from its logit, beyond fp32: what is left of z and log s, around 10
// each, is subtracted again (old_logp, the other sequence's sum), and losses over few
// rows are differences of ratios: in fp32 the last bits of 10 were 1e-5 of such a loss.
// log s = k log 2 + log f with f in 0.7 .. 1.4, whose logarithm is off by 3e-8 in fp32 (one in
// double, and the ratio's exponential, before the gradient took 15 % of 8192 rows of 8192).
// NaN for a token outside the vocabulary (z is NaN then).
__device__ __forceinline__ double logp_of(float z, MaxSum a) {
  float f = __builtin_amdgcn_frexp_mantf(a.s);
  int k = __builtin_amdgcn_frexp_expf(a.s);
  if (f < 0.70710678f) f *= 2.f, --k;
  return ((double)z - (double)a.m) - ((double)k * 0.69314718055994531 + (double)logf(f));
}

// dL/dx of one element: c (1[v = tok] - exp(z - m) / s) with cs = -c / s
__device__ __forceinline__ float grad_one(float x, float inv_t, float m, float cs, float c, bool taken) {
#pragma clang fp contract(off)
  const float g = __builtin_amdgcn_exp2f((x * inv_t - m) * kLog2e) * cs;
  return taken ? g + c : g;
}

// Of a unit, elements `at` .. of the row.  tok as an int: -1 for one outside the vocabulary.
template <typename T>
__device__ __forceinline__ void grad_unit(Unit<T>& u, int at, float inv_t, float m, float cs, float c, int tok) {
  const int t = tok - at;
#pragma unroll
  for (int e = 0; e < Unit<T>::VE; ++e) u.set(e, grad_one(u.get(e), inv_t, m, cs, c, e == t));
}

// ---------------------------------------------------------------- the policy loss
// Ratios and KL terms past fp32 count as its largest value in the gradient, as does the
// row's coefficient: infinite, they would turn an advantage of 0 and every entry of
// probability 0 into NaN.  A NaN stays one.
constexpr float kMost = 3.402823466e38f;
__device__ __forceinline__ float finite(float v) { return fabsf(v) > kMost ? copysignf(kMost, v) : v; }
__device__ __forceinline__ float exp_finite(float v) { return finite(expf(v)); }

struct PolicyArgs {
  const void* logits;
  long ld;
  const long* tokens;
  const float *old_logp, *adv, *ref_logp;  // ref_logp may be null
  const uint8_t* mask;                     // may be null
  const float* count;                      // device: max(1, rows that count), or null: counted here
  void* grad;                              // may be null
  long ldg;
  float* logp;
  double* term;  // [rows] the rows' losses, before the division by their count
  int rows, vocab;
  float lo, hi, kl, inv_t, grad_scale;
};

__device__ __forceinline__ int count_mask(const uint8_t* mask, int rows, int tid, int threads) {
  int n = 0;
#pragma unroll 4
  for (int i = tid; i < rows; i += threads) n += mask[i] != 0;
#pragma unroll
  for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
  return n;  // of the wave
}

__global__ __launch_bounds__(1024) void mask_count_kernel(const uint8_t* mask, int rows, float* out) {
  __shared__ int part[16];
  const int n = count_mask(mask, rows, threadIdx.x, 1024);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int s = 0;
    for (int w = 0; w < 16; ++w) s += part[w];
    *out = (float)max(s, 1);
  }
}

// The row's first THREADS * NU units are in registers from the pass that finds m and s to the
// one that writes the gradient: the logits are read once.  Such a unit starts at element
// 16 bytes times its number, but the last one at the row's last 16 bytes: its loads and stores
// are whole, the elements that it shares with the unit before are left out of the sum
// and written twice with the same value.  Units beyond those (a row longer than the block
// holds) are read again.  grad may be the logits themselves: a thread writes only what
// it has in registers, or units that it alone has read, after every thread has read the
// token's logit.
// THREADS = 64: a wave a row, four rows a block, no barrier.
// (Rows of 131072 bf16 fill a CU's registers, which so reads and writes in turns: 4.3 TB/s.
// Blocks that stay and load the next row's units behind this one's stores would do both at
// once, but the compiler holds both rows: 200 spilled registers, 2.3 TB/s.)
template <typename T, int THREADS, int NU>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void policy_kernel(PolicyArgs p) {
  using S = typename Elem<T>::storage;
  constexpr int VE = Unit<T>::VE, RPB = THREADS < 256 ? 256 / THREADS : 1;
  __shared__ MaxSum red[THREADS / 64];
  __shared__ int cnt[THREADS / 64];
  const int tid = threadIdx.x % THREADS, V = p.vocab;
  const int units = (V + VE - 1) / VE, last = max(V - VE, 0), shared = units * VE - V;
  const long row = (long)blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / THREADS : 0);
  if (row >= p.rows) return;  // whole waves, and only where a row is a wave
  const S* x = static_cast<const S*>(p.logits) + (size_t)row * p.ld;
  S* g = p.grad ? static_cast<S*>(p.grad) + (size_t)row * p.ldg : nullptr;
  if (p.mask && !p.mask[row]) {  // the row's logits are not read
    if (tid == 0) {
      p.logp[row] = 0.f;
      p.term[row] = 0.f;
    }
    if (g) {
      Unit<T> zero;
      zero.raw = u32x4r{0, 0, 0, 0};
      for (int u = tid; u < units; u += THREADS) zero.template store<true>(g, u, V);
    }
    return;
  }
  Unit<T> r[NU];
  auto load_unit = [&](Unit<T>& v, const S* x, int i) {
    if (V >= VE) v.raw = load_once(x + min((i * THREADS + tid) * VE, last));
    else v.load(x, 0, V, kNegInf);  // a vocabulary of less than a unit: every thread has it
  };
#pragma unroll
  for (int i = 0; i < NU; ++i)
    if (i * THREADS < units) load_unit(r[i], x, i);
  float count = (float)p.rows;
  if (p.mask && p.count) count = *p.count;
  if (p.mask && !p.count) {
    int n = count_mask(p.mask, p.rows, tid, THREADS);
    if constexpr (THREADS > 64) {
      if ((tid & 63) == 0) cnt[tid >> 6] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) n += cnt[w];
    }
    count = (float)max(n, 1);
  }
  const long tok64 = p.tokens[row];
  const int tok = tok_ok(tok64, V) ? (int)tok64 : -1;
  const float zt = tok >= 0 ? Elem<T>::to_f32(x[tok]) * p.inv_t : __builtin_nanf("");
  const float old = p.old_logp[row], adv = p.adv[row];
  MaxSum a = {kNegInf, 0.f};
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if ((i + 1) * THREADS < units) {  // not the last unit, nor any past it
      add_unit<T>(a, r[i], p.inv_t);
    } else if (i * THREADS < units) {
      const int u = i * THREADS + tid, from = u < units - 1 ? 0 : u < units && V >= VE ? shared : u == 0 ? 0 : VE;
      Unit<T> v = r[i];
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e < from) v.set(e, kNegInf);
      add_unit<T>(a, v, p.inv_t);
    }
  }
  for (int u = NU * THREADS + tid; u < units; u += THREADS) {
    Unit<T> v;
    v.load(x, u, V, kNegInf);
    add_unit<T>(a, v, p.inv_t);
  }
  a = block_join<THREADS>(a, red);
  const double logp = logp_of(zt, a);
  const float ratio = exp_finite((float)(logp - (double)old));
  const float plain = ratio * adv, clipped = fminf(fmaxf(ratio, 1.f - p.lo), 1.f + p.hi) * adv;
  float d = plain <= clipped ? -plain : 0.f;  // the loss's slope in logp
  if (isnan(plain)) d = plain;  // min and max leave a NaN out
  if (p.ref_logp && p.kl != 0.f) d += p.kl * (1.f - exp_finite((float)((double)p.ref_logp[row] - logp)));
  // The row's loss behind its gradient, by one wave: in double, for the loss is a small
  // difference of terms where advantages cancel, and of a few rows the terms' last bits in
  // fp32 were 4e-6 of it.
  auto loss_term = [&] {
    if (tid) return;
    const double r = exp(logp - (double)old), full = adv == 0.f && r > 0.0 ? 0.0 : r * adv;
    double term = -fmin(full, fmin(fmax(r, 1.0 - (double)p.lo), 1.0 + (double)p.hi) * adv);
    if (isnan(full)) term = full;
    if (p.ref_logp && p.kl != 0.f) {
      const double q = (double)p.ref_logp[row] - logp;
      term += p.kl * (exp(q) - q - 1.0);
    }
    p.logp[row] = (float)logp;
    p.term[row] = term;
  };
  if (!g) return loss_term();
  const float c = finite(d * p.inv_t * p.grad_scale / count), cs = -c / a.s, m = finite_or_0(a.m);
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if ((i + 1) * THREADS < units) {
      const int at = (i * THREADS + tid) * VE;
      grad_unit<T>(r[i], at, p.inv_t, m, cs, c, tok);
      store_once(g + at, r[i].raw);
    } else if (i * THREADS < units) {
      const int u = i * THREADS + tid, at = min(u * VE, last);
      grad_unit<T>(r[i], at, p.inv_t, m, cs, c, tok);
      if (V < VE) {
        if (u == 0) r[i].store(g, 0, V);
      } else if (u < units) {
        store_once(g + at, r[i].raw);
      }
    }
  }
  for (int u = NU * THREADS + tid; u < units; u += THREADS) {
    Unit<T> v;
    v.load(x, u, V, kNegInf);
    grad_unit<T>(v, u * VE, p.inv_t, m, cs, c, tok);
    v.template store<true>(g, u, V);
  }
  loss_term();
}

// loss = the mean of the n terms that the mask keeps (the others are 0), in double and in a
// fixed order
__device__ __forceinline__ void mean_terms(const double* term, const uint8_t* mask, long n, float* loss, double* red) {
  double s = 0, count = 0;  // of terms; 1 for each row that counts
  for (long i = threadIdx.x; i < n; i += blockDim.x) {
    s += term[i];
    count += !mask || mask[i] ? 1.0 : 0.0;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    s += __shfl_xor(s, o);
    count += __shfl_xor(count, o);
  }
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = s;
    red[16 + (threadIdx.x >> 6)] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0, c = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
      t += red[w];
      c += red[16 + w];
    }
    *loss = (float)(t / fmax(c, 1.0));
  }
}
__global__ __launch_bounds__(1024) void term_mean_kernel(const double* term, const uint8_t* mask, long n, float* loss) {
  __shared__ double red[32];
  mean_terms(term, mask, n, loss, red);
}

// ---------------------------------------------------------------- log-probabilities
struct RowArgs {
  const void* logits;
  long ld;
  const long* tokens;
  const uint8_t* mask;  // may be null
  float* logp;          // 0 where the mask is
  double* logp64;       // in place of logp, with stat
  MaxSum* stat;
  int rows, vocab;
  float inv_t;
};

// A row's m, s and its token's log-probability; the row is read once.  THREADS = 64: a wave
// a row, four rows a block.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void row_stat_kernel(RowArgs p) {
  using S = typename Elem<T>::storage;
  constexpr int VE = Unit<T>::VE, RPB = THREADS < 256 ? 256 / THREADS : 1;
  __shared__ MaxSum red[THREADS / 64];
  const int row = blockIdx.x * RPB + (RPB > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS) : 0);
  if (row >= p.rows) return;  // whole waves, and only where a row is a wave
  const int tid = threadIdx.x % THREADS, V = p.vocab, whole = V / VE;
  if (p.mask && !p.mask[row]) {
    if (tid == 0 && p.stat) p.logp64[row] = 0.0;
    else if (tid == 0) p.logp[row] = 0.f;
    return;
  }
  const S* x = static_cast<const S*>(p.logits) + (size_t)row * p.ld;
  MaxSum a = {kNegInf, 0.f};
  const bool rest = V % VE && tid == whole % THREADS;  // the row's last unit, not a whole one
  Unit<T> end;
  if (rest) end.load(x, whole, V, kNegInf);
  int u = tid;
  for (; u + 3 * THREADS < whole; u += 4 * THREADS) {  // four loads in flight
    Unit<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) __builtin_memcpy(&v[i].raw, x + (size_t)(u + i * THREADS) * VE, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) add_unit<T>(a, v[i], p.inv_t);
  }
  if (u < whole) {  // and three: past the row's end the last whole unit is asked for again
    Unit<T> v[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) __builtin_memcpy(&v[i].raw, x + (size_t)min(u + i * THREADS, whole - 1) * VE, 16);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (u + i * THREADS < whole) add_unit<T>(a, v[i], p.inv_t);
  }
  if (rest) add_unit<T>(a, end, p.inv_t);
  a = block_join<THREADS>(a, red);
  if (tid == 0) {
    const long tok = p.tokens[row];
    const double logp = logp_of(tok_ok(tok, V) ? Elem<T>::to_f32(x[tok]) * p.inv_t : __builtin_nanf(""), a);
    if (p.stat) {
      p.logp64[row] = logp;
      p.stat[row] = a;
    } else {
      p.logp[row] = (float)logp;
    }
  }
}

// ---------------------------------------------------------------- the preference loss
struct PairArgs {
  const long* offsets;  // [2 pairs + 1]
  const double* logp;   // [rows]
  const float* ref;     // [2 pairs]
  float* seq_logp;      // [2 pairs]
  float* coef;          // [2 pairs] dLoss/dlogp of the sequence's rows
  double* term;         // [pairs]
  int pairs;
  long rows;
  float beta, smooth;
};

// One block of two waves per pair: wave 0 sums the chosen sequence, wave 1 the rejected
// one.  In double, of rows in double: the sums are hundreds or thousands of nats, their
// difference a few, and fp32 rows of 10 nats were 1e-6 of the loss of 3010 of them.
__global__ __launch_bounds__(128) void pair_kernel(PairArgs p) {
  __shared__ double sum[2];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, s = blockIdx.x + w * p.pairs;
  const long lo = max(p.offsets[s], 0L), hi = min(p.offsets[s + 1], p.rows);
  double t = 0;
  for (long i = lo + lane; i < hi; i += 64) t += p.logp[i];
#pragma unroll
  for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
  if (lane == 0) {
    sum[w] = t - p.ref[s];
    p.seq_logp[s] = (float)t;
  }
  __syncthreads();
  if (threadIdx.x) return;
  const double z = (double)p.beta * (sum[0] - sum[1]), e = p.smooth;
  // -log sigmoid(z) = max(-z, 0) + log(1 + t) with t = e^-|z|, and both sigmoids from 1 / (1 + t) and t / (1 + t).
  // An infinite margin (a token of probability 0): a label's share of 0 is none, not 0 infinity.
  const double t1 = exp(-fabs(z)), l = log1p(t1), big = 1.0 / (1.0 + t1), small = t1 * big;
  p.term[blockIdx.x] = (e < 1 ? (1 - e) * (fmax(-z, 0.0) + l) : 0.0) + (e > 0 ? e * (fmax(z, 0.0) + l) : 0.0);
  // e sigmoid(z) - (1 - e) sigmoid(-z): a difference of sigmoid(z) and 1 - e loses what is left of a
  // decided pair's slope (1e-3 of it at z = 30, all of it at 37)
  const double d = p.beta / p.pairs * (e * (z < 0 ? small : big) - (1 - e) * (z < 0 ? big : small));
  p.coef[blockIdx.x] = (float)d;
  p.coef[blockIdx.x + p.pairs] = (float)-d;
}

struct PairGradArgs {
  const void* logits;
  long ld;
  const long *tokens, *offsets;
  const uint8_t* mask;
  const MaxSum* stat;
  const float* coef;
  const double* term;
  void* grad;  // may be null: only the loss is written then
  long ldg;
  float* loss;
  int pairs, vocab;
  long rows;
  float inv_t, grad_scale;
};

// Block 0 adds up the loss; every other one writes a part of a row's gradient.  A row
// of no sequence and a masked one get zeros.  Rows go from the last to the first: the
// last ones read by row_stat_kernel are still in the caches.  Units start at the row's first
// 16-byte boundary, the elements before it (`head`) go to a lane each: off the boundary, where
// most rows of odd width are, each wave's loads and stores take a cache line more.  (The sums of
// row_stat_kernel and policy_kernel start at the row's first element all the same, so that
// a row's log-probability has the same bits wherever the row lies: 3010 rows of 50021
// bf16 are read in 65 us for 49 from the boundary.)
template <typename T, int THREADS>
__global__ __launch_bounds__(256) void pair_grad_kernel(PairGradArgs p) {
  using S = typename Elem<T>::storage;
  constexpr int VE = Unit<T>::VE, RPB = 256 / THREADS;
  __shared__ double red[32];
  if (blockIdx.x == 0) {
    if (blockIdx.y == 0) mean_terms(p.term, nullptr, p.pairs, p.loss, red);
    return;
  }
  const int tid = threadIdx.x % THREADS;
  const long row = p.rows - 1 - ((blockIdx.x - 1L) * RPB + (RPB > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS) : 0));
  if (row < 0) return;
  const S* row_x = static_cast<const S*>(p.logits) + (size_t)row * p.ld;
  S* row_g = static_cast<S*>(p.grad) + (size_t)row * p.ldg;
  const int head = p.vocab < 2 * VE ? 0 : (int)((16 - ((uintptr_t)row_x & 15)) & 15) / (int)sizeof(S);
  const int V = p.vocab - head, units = (V + VE - 1) / VE;
  const S* x = row_x + head;
  S* g = row_g + head;
  const bool heads = blockIdx.y == 0 && tid < head;
  // the last sequence that starts at or before the row, among 2 pairs + 1 bounds
  int lo = 0, hi = 2 * p.pairs;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.offsets[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  const bool in = lo < 2 * p.pairs && p.offsets[lo] <= row && (!p.mask || p.mask[row]);
  const int step = THREADS * gridDim.y;
  if (!in) {
    Unit<T> zero;
    zero.raw = u32x4r{0, 0, 0, 0};
    if (heads) row_g[tid] = Elem<T>::from_f32(0.f);
    for (int u = blockIdx.y * THREADS + tid; u < units; u += step) zero.template store<true>(g, u, V);
    return;
  }
  const MaxSum a = p.stat[row];
  const long tok64 = p.tokens[row];
  const int tok = tok_ok(tok64, p.vocab) ? (int)tok64 : -1;
  float c = p.coef[lo] * p.inv_t * p.grad_scale;
  if (tok < 0) c = __builtin_nanf("");
  const float cs = -c / a.s, m = finite_or_0(a.m);
  if (heads) row_g[tid] = Elem<T>::from_f32(grad_one(Elem<T>::to_f32(row_x[tid]), p.inv_t, m, cs, c, tok == tid));
  int u = blockIdx.y * THREADS + tid;
  for (; u + 3 * step < units; u += 4 * step) {
    Unit<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i].template load<true>(x, u + i * step, V, kNegInf);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      grad_unit<T>(v[i], head + (u + i * step) * VE, p.inv_t, m, cs, c, tok);
      v[i].template store<true>(g, u + i * step, V);
    }
  }
  for (; u < units; u += step) {
    Unit<T> v;
    v.template load<true>(x, u, V, kNegInf);
    grad_unit<T>(v, head + u * VE, p.inv_t, m, cs, c, tok);
    v.template store<true>(g, u, V);
  }
}

template <typename T, int THREADS, int NU>
int launch_policy(const PolicyArgs& p, hipStream_t st) {
  constexpr int RPB = THREADS < 256 ? 256 / THREADS : 1;
  const long blocks = (p.rows + RPB - 1L) / RPB;
  policy_kernel<T, THREADS, NU><<<dim3((unsigned)blocks), THREADS * RPB, 0, st>>>(p);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

}  // namespace

size_t policy_loss_ws(long rows) { return (size_t)(rows + 32) * 8; }

template <typename T>
int run_policy_loss(const PolicyLossCall& q, float* ws, hipStream_t st) {
  float* count = ws;
  double* term = reinterpret_cast<double*>(ws + 64);
  if (q.rows) {
    PolicyArgs p{q.logits, q.ld, static_cast<const long*>(q.tokens), q.old_logp, q.adv, q.ref_logp,
                 static_cast<const uint8_t*>(q.mask), nullptr, q.grad, q.ldg, q.logp, term, (int)q.rows, (int)q.vocab,
                 q.lo, q.hi, q.kl, 1.f / q.temperature, q.grad_scale};
    const long units = (q.vocab + Elem<T>::vec - 1) / Elem<T>::vec;
    // few rows: a block counts the mask itself, with eight loads a thread at most and a launch less (1024 rows
    // of 1000 units 12.0 us, 13.3 with the launch; 2048: 19.4 and 18.3; 64 rows of 250: 7.6 and 9.1, 512: 9.7 and 9.4)
    if (q.mask && q.rows > (units <= 512 ? 64 : units <= 2048 ? 1024 : 2048)) {
      mask_count_kernel<<<1, 1024, 0, st>>>(p.mask, p.rows, count);
      VH_LAUNCH_CHECK();
      p.count = count;
    }
    // Threads and units a thread, so that a row just fits them.  A wave a row up to 512 units: 20000 rows of
    // 250 fp32 units 39 us, by 256 threads 61; of 480 bf16 units 70 and 95; 256 threads up to 2048: of 1000 bf16
    // units 149, by 512 threads 205; 512 up to 8192: 6000 rows of 8000 bf16 units 338, by 1024 threads 426.
    // Few rows leave CUs idle then and the longer chain costs up to 2.5 us (48 rows of 480 bf16 units 9.9
    // for 7.4, of 250 8.2 for 7.0), but the rule does not go by the rows: a row's sum has the same bits
    // among any number of them.
    int r;
    if (units <= 256) r = launch_policy<T, 64, 4>(p, st);
    else if (units <= 512) r = launch_policy<T, 64, 8>(p, st);
    else if (units <= 1024) r = launch_policy<T, 256, 4>(p, st);
    else if (units <= 2048) r = launch_policy<T, 256, 8>(p, st);
    else if (units <= 4096) r = launch_policy<T, 512, 8>(p, st);
    else if (units <= 8192) r = launch_policy<T, 512, 16>(p, st);
    else r = launch_policy<T, 1024, 16>(p, st);
    if (r != VH_OK) return r;
  }
  term_mean_kernel<<<1, 1024, 0, st>>>(term, static_cast<const uint8_t*>(q.mask), q.rows, q.loss);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

// Two units a thread and less: a wave a row, four rows a block (20000 rows of 1000 bf16: log-probabilities
// 22.6 -> 11.6 us, the preference loss 73 -> 54; at three units and few rows the longer chain
// costs more, 100 rows of 1000 fp32 3.1 -> 4.2).  Then 256 threads a row, 512 past 2048 units
// (2048 rows of 32003 bf16: 26 us, 32 in 1024 threads) and 1024 past 8192 (4096 of 131072: 179, 188 in 512).
constexpr long kWaveUnits = 128;
template <typename T>
int run_row_stat(const void* logits, long ld, const void* tokens, const void* mask, float* logp, double* logp64, void* stat,
                 long rows, long vocab, float temperature, hipStream_t st) {
  if (!rows) return VH_OK;
  const RowArgs p{logits, ld, static_cast<const long*>(tokens), static_cast<const uint8_t*>(mask), logp, logp64,
                  static_cast<MaxSum*>(stat), (int)rows, (int)vocab, 1.f / temperature};
  const long units = (vocab + Elem<T>::vec - 1) / Elem<T>::vec;
  if (units <= kWaveUnits) row_stat_kernel<T, 64><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, st>>>(p);
  else if (units <= 2048) row_stat_kernel<T, 256><<<dim3((unsigned)rows), 256, 0, st>>>(p);
  else if (units <= 8192) row_stat_kernel<T, 512><<<dim3((unsigned)rows), 512, 0, st>>>(p);
  else row_stat_kernel<T, 1024><<<dim3((unsigned)rows), 1024, 0, st>>>(p);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

size_t preference_loss_ws(long rows, long pairs) { return (size_t)rows * 16 + (size_t)pairs * 16; }

template <typename T>
int run_preference_loss(const PreferenceLossCall& q, float* ws, hipStream_t st) {
  MaxSum* stat = reinterpret_cast<MaxSum*>(ws);
  double *logp = reinterpret_cast<double*>(stat + q.rows), *term = logp + q.rows;
  float* coef = reinterpret_cast<float*>(term + q.pairs);
  const int r = run_row_stat<T>(q.logits, q.ld, q.tokens, q.mask, nullptr, logp, stat, q.rows, q.vocab, q.temperature, st);
  if (r != VH_OK) return r;
  const PairArgs pa{static_cast<const long*>(q.offsets), logp, q.ref_logp, q.seq_logp, coef, term, (int)q.pairs,
                    q.rows, q.beta, q.smooth};
  if (q.pairs) {
    pair_kernel<<<dim3((unsigned)q.pairs), 128, 0, st>>>(pa);
    VH_LAUNCH_CHECK();
  }
  const PairGradArgs pg{q.logits, q.ld, static_cast<const long*>(q.tokens), static_cast<const long*>(q.offsets),
                        static_cast<const uint8_t*>(q.mask), stat, coef, term, q.grad, q.ldg, q.loss, (int)q.pairs,
                        (int)q.vocab, q.rows, 1.f / q.temperature, q.grad_scale};
  // rows split until there are about 4 blocks a CU, 4 units a thread at least
  const long units = (q.vocab + Elem<T>::vec - 1) / Elem<T>::vec;
  long split = 1;
  while (split < 64 && q.rows * split < 1024 && units >= split * 2 * 1024) split *= 2;
  const long blocks = !q.grad ? 1 : units <= kWaveUnits ? (q.rows + 3) / 4 + 1 : q.rows + 1;
  if (units <= kWaveUnits) pair_grad_kernel<T, 64><<<dim3((unsigned)blocks), 256, 0, st>>>(pg);
  else pair_grad_kernel<T, 256><<<dim3((unsigned)blocks, (unsigned)(q.grad ? split : 1)), 256, 0, st>>>(pg);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

#define VH_INST(T)                                                                                             \
  template int run_policy_loss<T>(const PolicyLossCall&, float*, hipStream_t);                                 \
  template int run_preference_loss<T>(const PreferenceLossCall&, float*, hipStream_t);                         \
  template int run_row_stat<T>(const void*, long, const void*, const void*, float*, double*, void*, long, long, float, \
                               hipStream_t);
VH_INST(float)
VH_INST(bf16)
#undef VH_INST

}  // namespace vh
