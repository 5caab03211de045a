// vh_norm.hip -- the norms around a block, fused with its gate and residual scale.
//
// For rows x (the residual stream) and b (the block's output) of D elements:
//   u = b / rms(b) * w_post          rms(v) = sqrt(mean(v^2) + eps)
//   y = x + scale * gate * u         the new residual stream
//   n = y / rms(y) * w_next          the next block's input
// and backwards, with bh = b / rms(b), yh = y / rms(y), from dy and dn:
//   h = dn * w_next,  g = dy + (h - yh mean(h yh)) / rms(y)     = dx
//   k = scale * gate * g * w_post,  db = (k - bh mean(k bh)) / rms(b)
//   dgate = scale * g * u,  dw_post = scale * gate * g * bh,  dw_next = dn * yh
// summed over the rows that share them.  Without w_post, u = b; without w_next there is
// no n; without a gate, 1.  n and the gradients come from y before its rounding (it is
// built again from x and b, which the backward reads anyway), so each output is
// rounded once.
//
// Bound by memory: the forward reads x and b and writes y and n, the backward reads dy,
// dn, x and b and writes dx and db, each once; a row stays in its threads' registers
// between the two reductions that it needs.  A thread has 16 elements forward, 8 backward
// (three sums for each beside the row's tensors): up to 1024 or 512 elements a wave takes a row by itself
// (no barrier), wider rows take several.  8192 rows of 4096 bf16, gates of 1024 rows each:
// 54 us forward (5.0 TB/s), 88 backward (4.7 TB/s) and 5 to add up its partial sums; 1000
// rows of 1531 fp32: 9, 16 and 5, where a row's two sums and two trips to memory, one
// after the other, are the time; one row of 4096: 4.3 forward, the same.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "vh_kernels.hpp"
#include "vh_rows.hpp"

namespace vh {

namespace {

// rows are at most kNormMostWidth elements
template <typename T, typename S>
__device__ __forceinline__ void load(Unit<T>& v, const S* row, int u, int n, float fill) {
  v.template load<false, true>(row, u, n, fill);
}
template <typename T, typename S>
__device__ __forceinline__ void store(const Unit<T>& v, S* row, int u, int n) {
  v.template store<false, true>(row, u, n);
}

struct NormArgs {
  const void *x, *b, *gate, *wp, *wn;  // gate, wp, wn may be null
  void *y, *n;                         // n null without wn
  float* rstd;                         // [2][rows]: 1 / rms(b) (1 without wp), 1 / rms(y)
  long rows, per;                      // rows of a gate row
  int d;
  float scale, eps;
};

struct NormGradArgs {
  const void *dy, *dn, *x, *b, *gate, *wp, *wn;
  const float* rstd;
  void *dx, *db, *dgate;
  float *pp, *pn, *pg;  // partial sums [spans][d] of dw_post, dw_next; of dgate [spans][d] (null: dgate is written whole)
  long rows, per;       // rows of a gate row
  long span;            // rows of a block
  int per_group;        // blocks of a gate row's rows; 0: a block takes whole ones
  int groups;           // rows that a block has at once
  int d;
  float scale;
};

// Sum over the threads of a row: a wave's by shuffles, a block's through red.  Sums that
// follow one another take the two sets in turn: a set is written again only past the
// barrier of the sum between, which no wave reaches before it has read the set.  A row
// has `waves` waves, its own the first of them; red holds two sets of 16 and 15 more,
// which only lanes past the row's waves read.
constexpr int kRed = 48;
template <bool WAVE>
__device__ __forceinline__ float row_sum(float v, float* red, int set, int waves, int first) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) red[set * 16 + (threadIdx.x >> 6)] = v;
    __syncthreads();
    v = red[set * 16 + first + (threadIdx.x & 15)];
    if ((int)(threadIdx.x & 15) >= waves) v = 0.f;
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor(v, o);
  }
  return v;
}

// NU units a thread.  MOST 64: a wave a row, four rows a block; else a block of at most
// MOST threads a row.
template <typename T, int MOST, int NU>
__global__ __launch_bounds__(MOST < 256 ? 256 : MOST) void norm_kernel(NormArgs p) {
  using S = typename Elem<T>::storage;
  constexpr bool WAVE = MOST == 64;
  constexpr int VE = Unit<T>::VE, RPB = WAVE ? 4 : 1;
  __shared__ float red[kRed];
  const int TPR = WAVE ? 64 : (int)blockDim.x, t = WAVE ? threadIdx.x & 63 : threadIdx.x, d = p.d;
  const long row = (long)blockIdx.x * RPB + (WAVE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (row >= p.rows) return;  // whole waves, and only where a row is a wave
  const S* x = static_cast<const S*>(p.x) + row * d;
  const S* b = static_cast<const S*>(p.b) + row * d;
  const S* gate = p.gate ? static_cast<const S*>(p.gate) + row / p.per * d : nullptr;
  const S *wp = static_cast<const S*>(p.wp), *wn = static_cast<const S*>(p.wn);
  const int units = (d + VE - 1) / VE;
  Unit<T> bu[NU], xu[NU], gu[NU], pu[NU], nu[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = i * TPR + t;
    if (u < units) {
      load(bu[i], b, u, d, 0.f);
      load(xu[i], x, u, d, 0.f);
      if (gate) load(gu[i], gate, u, d, 0.f);
      if (wp) load(pu[i], wp, u, d, 0.f);
      if (wn) load(nu[i], wn, u, d, 0.f);
    }
  }
  float rb = 1.f;
  if (wp) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (i * TPR + t < units)
#pragma unroll
        for (int e = 0; e < VE; ++e) s += bu[i].get(e) * bu[i].get(e);
    s = row_sum<WAVE>(s, red, 0, TPR >> 6, 0);
    rb = 1.f / sqrtf(s / (float)d + p.eps);
  }
  float y[NU][VE], s = 0.f;
#pragma unroll
  for (int i = 0; i < NU; ++i)
    if (i * TPR + t < units) {
      Unit<T> yu;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        float v = bu[i].get(e) * rb;
        if (wp) v *= pu[i].get(e);
        if (gate) v *= gu[i].get(e);
        v = xu[i].get(e) + p.scale * v;
        y[i][e] = v;
        s += v * v;
        yu.set(e, v);
      }
      store(yu, static_cast<S*>(p.y) + row * d, i * TPR + t, d);
    }
  float ry = 1.f;
  if (wn) {
    s = row_sum<WAVE>(s, red, 1, TPR >> 6, 0);
    ry = 1.f / sqrtf(s / (float)d + p.eps);
#pragma unroll
    for (int i = 0; i < NU; ++i)
      if (i * TPR + t < units) {
        Unit<T> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o.set(e, y[i][e] * ry * nu[i].get(e));
        store(o, static_cast<S*>(p.n) + row * d, i * TPR + t, d);
      }
  }
  if (t == 0) {
    p.rstd[row] = rb;
    p.rstd[p.rows + row] = ry;
  }
}

// Threads that the backward's registers leave room for, in rows of `threads`, `per` elements
// a thread: 128 registers each for 1024, 168 for 768
constexpr int norm_most_threads(int vec, int threads) {
  return threads > 768 || vec == 8 ? 1024 : 768;
}

// A block takes `span` consecutive rows, `groups` at a time, and keeps the sums over them of
// dw_post, dw_next and dgate in registers (its columns' owner in a group is the same thread for every row).  Spans
// either lie within one gate row's rows (pg: a partial of dgate each) or are whole
// multiples of them (dgate is written as each ends).  TOKEN: a gate row for each row, read
// and its gradient written with it.
// A row is four loads, two sums over it one after the other, two stores: what hides that chain
// is the next row's loads in flight meanwhile (AHEAD) and other rows beside it.  So one
// block fills a CU with as many row groups as the registers allow, which also makes one set
// of partial sums of what would be several blocks' (8192 rows of 4096 bf16, with the sums:
// a row a block of 512 threads 95 us, two in 1024 threads 71; 16000 of 1531: 117 and 75).
// Rows past 8192 elements (WIDE) would need three sums and four tensors of 16 elements a
// thread: two of the sums are in LDS, each thread's own, and what is used once is loaded where
// it is used (1000 rows of 12000 fp32: 293 us when they spilled, 121 so).
template <typename T, int MOST, int NU, bool TOKEN>
__global__ __launch_bounds__(MOST == 64 ? norm_most_threads(Elem<T>::vec, 64) : MOST) void norm_grad_kernel(NormGradArgs p) {
  using S = typename Elem<T>::storage;
  constexpr bool WAVE = MOST == 64, AHEAD = MOST <= 768 || (Unit<T>::VE == 8 && NU == 1);
  constexpr int VE = Unit<T>::VE, Q = VE / 4;
  constexpr bool WIDE = MOST == 1024 && NU * VE == 16, KEEP = !WIDE;
  extern __shared__ float4 shared[];  // kRed floats of row_sum, then the sums
  float* red = reinterpret_cast<float*>(shared);
  float4* lds = shared + kRed / 4;
  float* part = reinterpret_cast<float*>(lds);
  const int RPB = p.groups, TPR = WAVE ? 64 : (int)blockDim.x / RPB, d = p.d;
  // whole waves of a group: its row and what hangs on it in scalar registers
  const int rg = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR), t = threadIdx.x - rg * TPR;
  const int all_units = (d + VE - 1) / VE;
  const bool wp = p.wp != nullptr, wn = p.wn != nullptr;
  // a weight or gate that is not there is 1
  auto load_or_1 = [&](Unit<T>& v, const void* src, long row, int u) {
    if (src && u < all_units) {
      load(v, static_cast<const S*>(src) + row * d, u, d, 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) v.set(e, 1.f);
    }
  };
  Unit<T> pk[KEEP ? NU : 1], nk[KEEP ? NU : 1], gk[KEEP ? NU : 1];
  float sp[WIDE ? 1 : NU][VE], sn[WIDE ? 1 : NU][VE], sg[NU][VE];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if constexpr (KEEP) {
      load_or_1(pk[i], p.wp, 0, i * TPR + t);
      load_or_1(nk[i], p.wn, 0, i * TPR + t);
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      sg[i][e] = 0.f;
      if constexpr (!WIDE) sp[i][e] = sn[i][e] = 0.f;
    }
    if constexpr (WIDE)
#pragma unroll
      for (int h = 0; h < Q; ++h)
        lds[(i * Q + h) * TPR + t] = lds[((NU + i) * Q + h) * TPR + t] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  auto weight = [&](Unit<T> (&kept)[KEEP ? NU : 1], const void* src, long row, int i) {
    if constexpr (KEEP) return kept[i];
    Unit<T> v;
    load_or_1(v, src, row, i * TPR + t);
    return v;
  };
  // a unit of the row that Row keeps, or of a wide row, loaded where it is used
  auto element = [&](const auto& kept, const void* src, long row, int i) {
    if constexpr (!WIDE) return kept[i];
    Unit<T> v;
    load(v, static_cast<const S*>(src) + row * d, i * TPR + t, d, 0.f);
    return v;
  };
  // unit i of the sums for dw_post (0) and dw_next (1) += v
  auto add_up = [&](int which, int i, const float (&v)[VE]) {
    if constexpr (WIDE) {
#pragma unroll
      for (int h = 0; h < Q; ++h) {
        float4& a = lds[((which * NU + i) * Q + h) * TPR + t];
        a = make_float4(a.x + v[h * 4], a.y + v[h * 4 + 1], a.z + v[h * 4 + 2], a.w + v[h * 4 + 3]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) (which ? sn[i][e] : sp[i][e]) += v[e];
    }
  };
  // the block's sum of v: its row groups' added in order, then store(unit, element, sum)
  auto flush = [&](float (&v)[NU][VE], auto store) {
    if (!WIDE && RPB > 1) {
      if (rg)
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
          for (int e = 0; e < VE; ++e) part[((rg - 1) * NU * VE + i * VE + e) * TPR + t] = v[i][e];
      __syncthreads();
      if (!rg)
        for (int w = 0; w < RPB - 1; ++w)
#pragma unroll
          for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) v[i][e] += part[(w * NU * VE + i * VE + e) * TPR + t];
      __syncthreads();
      if (rg) return;
    }
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = i * TPR + t;
      if (u < all_units) store(i, u);
    }
  };
  auto to_partial = [&](float (&v)[NU][VE], float* dst) {
    flush(v, [&](int i, int u) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (u * VE + e < d) dst[(size_t)blockIdx.x * d + u * VE + e] = v[i][e];
    });
  };
  struct Row {
    Unit<T> b[NU], dn[NU], x[WIDE ? 1 : NU], dy[WIDE ? 1 : NU], g[TOKEN && !WIDE ? NU : 1];
    float rb, ry;
  };
  auto load_row = [&](Row& q, long row) {
    q.rb = p.rstd[row];
    q.ry = p.rstd[p.rows + row];
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = i * TPR + t;
      if (u < all_units) {
        load(q.b[i], static_cast<const S*>(p.b) + row * d, u, d, 0.f);
        if (wn) load(q.dn[i], static_cast<const S*>(p.dn) + row * d, u, d, 0.f);
        if constexpr (!WIDE) {
          if (wn) load(q.x[i], static_cast<const S*>(p.x) + row * d, u, d, 0.f);
          if (p.dy) load(q.dy[i], static_cast<const S*>(p.dy) + row * d, u, d, 0.f);
          if constexpr (TOKEN) load(q.g[i], static_cast<const S*>(p.gate) + row * d, u, d, 0.f);
        }
      }
    }
  };
  long first = (long)blockIdx.x * p.span, last = min(first + p.span, p.rows);
  if (p.per_group) {
    const long gr = blockIdx.x / p.per_group;
    first = gr * p.per + (long)(blockIdx.x - gr * p.per_group) * p.span;
    last = min(first + p.span, (gr + 1) * p.per);
  }
  const float inv_d = 1.f / (float)d;
  int set = 0;
  for (long at = first; at < last;) {
    const bool group = !TOKEN && p.gate;
    const long end = group ? min(last, (at / p.per + 1) * p.per) : last;
    const long gate_row = at / p.per;
    if constexpr (!TOKEN && KEEP)
#pragma unroll
      for (int i = 0; i < NU; ++i) load_or_1(gk[i], p.gate, gate_row, i * TPR + t);
    Row q, next;
    if (AHEAD && at + rg < end) load_row(q, at + rg);
    // the block's rows in step (a row's sums have the block's barriers): a group past the
    // last row has no units
    for (long base = at; base < end; base += RPB) {
      const long row = base + rg;
      const int units = row < end ? all_units : 0;
      if (!AHEAD && units) load_row(q, row);
      if (AHEAD && row + RPB < end) load_row(next, row + RPB);
      float g[NU][VE];
      float s = 0.f;
      if (wn) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
          if (i * TPR + t < units) {
            const Unit<T> pu = weight(pk, p.wp, 0, i), nu = weight(nk, p.wn, 0, i);
            Unit<T> gu;
            if constexpr (TOKEN) gu = element(q.g, p.gate, row, i);
            else gu = weight(gk, p.gate, gate_row, i);
            const Unit<T> xu = element(q.x, p.x, row, i);
            float w[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const float v = q.b[i].get(e) * q.rb * pu.get(e) * gu.get(e) * p.scale;
              const float yh = (xu.get(e) + v) * q.ry, dn = q.dn[i].get(e);
              w[e] = dn * yh;
              g[i][e] = yh;
              s += dn * nu.get(e) * yh;
            }
            add_up(1, i, w);
            if constexpr (WIDE) __builtin_amdgcn_sched_barrier(0);  // a unit's loads after the last one's registers
          }
        s = row_sum<WAVE>(s, red, set, TPR >> 6, rg * (TPR >> 6)) * inv_d;
        set ^= 1;
      }
      float k = 0.f;
#pragma unroll
      for (int i = 0; i < NU; ++i)
        if (i * TPR + t < units) {
          const Unit<T> pu = weight(pk, p.wp, 0, i), nu = weight(nk, p.wn, 0, i);
          Unit<T> gu;
          if constexpr (TOKEN) gu = element(q.g, p.gate, row, i);
          else gu = weight(gk, p.gate, gate_row, i);
          Unit<T> o, og, dyu;
          if (p.dy) dyu = element(q.dy, p.dy, row, i);
          float w[VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            float v = p.dy ? dyu.get(e) : 0.f;
            if (wn) v += q.ry * (q.dn[i].get(e) * nu.get(e) - g[i][e] * s);
            o.set(e, v);
            v *= p.scale;
            const float bh = q.b[i].get(e) * q.rb;
            const float dg = v * (bh * pu.get(e));
            if constexpr (TOKEN) og.set(e, dg);
            else sg[i][e] += dg;
            v *= gu.get(e);
            w[e] = v * bh;
            v *= pu.get(e);
            k += v * bh;
            g[i][e] = v;
          }
          add_up(0, i, w);
          store(o, static_cast<S*>(p.dx) + row * d, i * TPR + t, d);
          if constexpr (TOKEN) store(og, static_cast<S*>(p.dgate) + row * d, i * TPR + t, d);
          if constexpr (WIDE) __builtin_amdgcn_sched_barrier(0);
        }
      if (wp) {
        k = row_sum<WAVE>(k, red, set, TPR >> 6, rg * (TPR >> 6)) * inv_d;
        set ^= 1;
      }
#pragma unroll
      for (int i = 0; i < NU; ++i)
        if (i * TPR + t < units) {
          Unit<T> o;
#pragma unroll
          for (int e = 0; e < VE; ++e) o.set(e, wp ? q.rb * (g[i][e] - q.b[i].get(e) * q.rb * k) : g[i][e]);
          store(o, static_cast<S*>(p.db) + row * d, i * TPR + t, d);
        }
      if (AHEAD) q = next;
    }
    if (group && !p.pg) {
      const long gr = at / p.per;
      flush(sg, [&](int i, int u) {
        Unit<T> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o.set(e, sg[i][e]);
        store(o, static_cast<S*>(p.dgate) + gr * d, u, d);
      });
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) sg[i][e] = 0.f;
    }
    at = end;
  }
  if (p.pg) to_partial(sg, p.pg);
  if constexpr (WIDE) {
    auto kept = [&](int which, float* dst) {
      float v[NU][VE];
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int h = 0; h < Q; ++h) {
          const float4 a = lds[((which * NU + i) * Q + h) * TPR + t];
          v[i][h * 4] = a.x;
          v[i][h * 4 + 1] = a.y;
          v[i][h * 4 + 2] = a.z;
          v[i][h * 4 + 3] = a.w;
        }
      to_partial(v, dst);
    };
    if (wp) kept(0, p.pp);
    if (wn) kept(1, p.pn);
  } else {
    if (wp) to_partial(sp, p.pp);
    if (wn) to_partial(sn, p.pn);
  }
}

// out[r][c] = the sum over z < n of part[r * n + z][c]: blocks of 64 columns, 16 waves of
// every sixteenth z each, added in a fixed order.
struct NormSumArgs {
  const float* part[3];
  void* out[3];
  int n[3];  // partials of an output row
  int d;
};
template <typename T>
__global__ __launch_bounds__(1024) void norm_sum_kernel(NormSumArgs p) {
  using S = typename Elem<T>::storage;
  const int which = blockIdx.z;
  const float* part = p.part[which];
  if (!part) return;
  const int n = p.n[which], c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  if (which < 2 && blockIdx.y) return;  // the weights have one row, the gate gridDim.y
  const float* q = part + (size_t)blockIdx.y * n * p.d + c;
  __shared__ float red[16][64];
  float s = 0.f;
  if (c < p.d) {
#pragma unroll 8
    for (int z = w; z < n; z += 16) s += q[(size_t)z * p.d];
  }
  red[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < p.d) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) sum += red[v][threadIdx.x];
    static_cast<S*>(p.out[which])[(size_t)blockIdx.y * p.d + c] = Elem<T>::from_f32(sum);
  }
}

// Threads of a row in whole waves, `per` elements each (64: a wave by itself)
int norm_threads(long d, int per) { return std::max(1, (int)((d + 64 * per - 1) / (64 * per))) * 64; }
// Elements a thread of the backward
int norm_grad_per(long d) { return d <= 8192 ? 8 : 16; }
// Rows that a block of the backward has at once
int norm_groups(long d, int vec) {
  const int threads = norm_threads(d, norm_grad_per(d));
  return norm_most_threads(vec, threads) / threads;
}

}  // namespace

template <typename T>
int run_residual_norm(const ResidualNormCall& q, hipStream_t st) {
  constexpr int NU = 16 / Elem<T>::vec;
  const NormArgs p{q.x, q.b, q.gate, q.wp, q.wn, q.y, q.n, q.rstd, q.rows, q.gate ? q.rows / q.gate_rows : q.rows, (int)q.d, q.scale, q.eps};
  const int threads = norm_threads(q.d, 16);
  const dim3 rows((unsigned)q.rows);
  if (threads == 64) norm_kernel<T, 64, NU><<<dim3((unsigned)((q.rows + 3) / 4)), 256, 0, st>>>(p);
  else if (threads <= 512) norm_kernel<T, 512, NU><<<rows, threads, 0, st>>>(p);
  else norm_kernel<T, 1024, NU><<<rows, threads, 0, st>>>(p);
  VH_LAUNCH_CHECK();
  return VH_OK;
}

// How the rows are shared out: up to a block a CU, which then has the CU's registers to itself
// (a second one waits, and its partial sums cost a row's traffic or two: twice as many
// blocks took 3 to 25 % longer), and a step of its row groups each at least.  With fewer
// gate rows than that, a span is a part of a gate row's rows; otherwise whole ones.
NormPlan residual_norm_plan(int dtype, long rows, long d, long gate_rows) {
  const long target = 256, at_once = norm_groups(d, dtype == VH_F32 ? 4 : 8);
  if (gate_rows == rows) gate_rows = 0;  // a gate row with each row: nothing to add up
  const long groups = gate_rows ? gate_rows : 1, per = rows / groups;
  NormPlan o{};
  if (groups * 2 <= target) {
    const long spans = std::max(1L, std::min(target / groups, per / at_once));
    o.span = (per + spans - 1) / spans;
    o.per_group = (per + o.span - 1) / o.span;
    o.spans = o.per_group * groups;
    o.partial_gate = gate_rows != 0 && o.per_group > 1;
  } else {
    const long k = (groups + target - 1) / target;
    o.span = k * per;
    o.spans = (rows + o.span - 1) / o.span;
    o.per_group = 0;
    o.partial_gate = false;
  }
  return o;
}

size_t residual_norm_ws(int dtype, long rows, long d, long gate_rows) {
  const NormPlan o = residual_norm_plan(dtype, rows, d, gate_rows);
  return (size_t)o.spans * d * 4 * (o.partial_gate ? 3 : 2);
}

template <typename T>
int run_residual_norm_backward(const ResidualNormGradCall& q, float* ws, hipStream_t st) {
  constexpr int dtype = Elem<T>::vec == 4 ? VH_F32 : VH_BF16;
  const NormPlan o = residual_norm_plan(dtype, q.rows, q.d, q.gate ? q.gate_rows : 0);
  const bool token = q.gate && q.gate_rows == q.rows;
  const size_t one = (size_t)o.spans * q.d;
  NormGradArgs p{q.dy, q.dn, q.x, q.b, q.gate, q.wp, q.wn, q.rstd, q.dx, q.db, q.dgate, ws, ws + one,
                 o.partial_gate ? ws + 2 * one : nullptr, q.rows, q.gate && !token ? q.rows / q.gate_rows : q.rows, o.span, (int)o.per_group,
                 norm_groups(q.d, Elem<T>::vec), (int)q.d, q.scale};
  const dim3 grid((unsigned)o.spans);
  const int threads = norm_threads(q.d, norm_grad_per(q.d)), block = threads * p.groups;
  auto launch = [&](auto MOST, auto PER) {
    constexpr int most = decltype(MOST)::value, per = decltype(PER)::value, n = per / Elem<T>::vec;
    // the row groups' sums, or of the widest rows two sums of every column
    constexpr bool wide = most == 1024 && per == 16;
    const size_t lds = kRed * 4 + (size_t)threads * per * 4 * (wide ? 2 : p.groups - 1);
    if (token) {
      auto kern = norm_grad_kernel<T, most, n, true>;
      if constexpr (wide) VH_LDS_LIMIT_ONCE(kern);
      kern<<<grid, block, lds, st>>>(p);
    } else {
      auto kern = norm_grad_kernel<T, most, n, false>;
      if constexpr (wide) VH_LDS_LIMIT_ONCE(kern);
      kern<<<grid, block, lds, st>>>(p);
    }
  };
  using I64 = std::integral_constant<int, 64>;
  using I1024 = std::integral_constant<int, 1024>;
  using I8 = std::integral_constant<int, 8>;
  using I16 = std::integral_constant<int, 16>;
  if (threads == 64) launch(I64{}, I8{});
  else if (q.d > 8192) launch(I1024{}, I16{});
  else if (Elem<T>::vec == 8 || block > 768) launch(I1024{}, I8{});
  else if constexpr (Elem<T>::vec == 4) launch(std::integral_constant<int, 768>{}, I8{});
  VH_LAUNCH_CHECK();
  if (q.wp || q.wn || p.pg) {
    const NormSumArgs s{{q.wp ? p.pp : nullptr, q.wn ? p.pn : nullptr, p.pg}, {q.dwp, q.dwn, q.dgate},
                        {(int)o.spans, (int)o.spans, (int)o.per_group}, (int)q.d};
    norm_sum_kernel<T><<<dim3((unsigned)((q.d + 63) / 64), (unsigned)(p.pg ? q.gate_rows : 1), p.pg ? 3 : 2), 1024, 0, st>>>(s);
    VH_LAUNCH_CHECK();
  }
  return VH_OK;
}

#define VH_INST(T)                                                     \
  template int run_residual_norm<T>(const ResidualNormCall&, hipStream_t); \
  template int run_residual_norm_backward<T>(const ResidualNormGradCall&, float*, hipStream_t);
VH_INST(float)
VH_INST(bf16)
#undef VH_INST

}  // namespace vh
