// Distillation from the largest logits of a teacher, with the hard-label loss beside it: loss and gradient in one pass over the student's
// logits.  Per row, with q = softmax(z / T) and P_j the teacher's probability of class j:
//   P from K (logit, class) pairs: softmax(t / T) over the pairs, or - given the teacher's log-sum-exp over ALL classes at temperature T -
//     exp(t / T - lse) for the pairs and the mass that is left spread evenly over the classes no pair names
//   loss = w_s T^2 sum_j P_j (log P_j - log q_j) + w_h CE(z, (1 - a) onehot(label) + a / C)
//   dz_j = w_s T (S q_j - P_j) + w_h (softmax(z)_j - y_j),   S = sum_j P_j  (1, or 0 where no pair is usable)
//
// Bound by HBM: z is read once and dz written once.  The row stays in registers between the pass that finds the maximum and the sums and the pass
// that writes the gradient (C 16-byte pieces a thread; what does not fit is read a second time), so there is one block reduction and no re-read.
// A thread keeps the sums relative to its own maximum and the block joins (maximum, sum) pairs: one barrier instead of two.
// Measured, with gradient: [2048 x 131072] 255 us (1075 MB, 4.2 TB/s; with the sum of the logits 276; the loss alone 139; a copy of the bytes takes 216),
// [1024 x 21843] 40 us with that sum (135 MB, 3.4 TB/s), [128 x 1000] 8 us: a launch, and the 64-bit logarithms and exponentials of the pairs one after the
// other.  What is left above the copy: a row's loads do not overlap the stores of the row before it in the same registers, and the exponentials (10 %).
// Exponentials are v_exp_f32 on (z - max) * (log2 e / T), per-thread sums fp32; everything that exists once a row - the pairs, the
// normalisers, the sum of the logits, the loss - is in 64 bits: a divergence near zero is the difference of numbers a hundred times its size.
// The gradient is written for every class as if no pair named it, then the at most K + 1 classes with a pair or the label are written again.
#include <type_traits>

#include "common.h"
#include "savit.h"

namespace {

constexpr int DS_MAX_K = 512;
constexpr double LN2 = 0.69314718055994530942;

struct DistillParams {
  const void* z;
  const float* top;     // [R, K] teacher logits
  const int* at;        // [R, K] their classes; outside [0, C): no pair
  const float* lse;     // [R] or nullptr
  const int* labels;    // [R] or nullptr; outside [0, C): no hard term for the row
  const float* weight;  // [R] or nullptr
  float* loss_rows;     // [R] or nullptr
  void* dz;             // or nullptr
  long ldz, lddz;
  int R, C, K, slots;
  float soft, hard, smooth, T, c_soft, c_hard, grad_scale;  // c_soft = log2 e / T, c_hard = log2 e
  double inv_T;
};

template <typename T>
struct Piece;  // 16 bytes of a row
template <>
struct Piece<float> {
  static constexpr int E = 4;
  typedef f32x4 vec __attribute__((aligned(4)));
  float v[4];
  __device__ __forceinline__ void clear() { v[0] = v[1] = v[2] = v[3] = -INFINITY; }
  __device__ __forceinline__ void load(const float* p) {
    const vec r = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  }
  __device__ __forceinline__ void load_part(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : -INFINITY;
  }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
};
template <>
struct Piece<bf16_t> {
  static constexpr int E = 8;
  typedef u32x4 vec __attribute__((aligned(2)));
  uint32_t v[4];
  __device__ __forceinline__ void clear() { v[0] = v[1] = v[2] = v[3] = 0xff80ff80u; }
  __device__ __forceinline__ void load(const bf16_t* p) {
    const vec r = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  }
  __device__ __forceinline__ void load_part(const bf16_t* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < n ? p[2 * i] : 0xff80u, hi = 2 * i + 1 < n ? p[2 * i + 1] : 0xff80u;
      v[i] = lo | (hi << 16);
    }
  }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float((i & 1) ? (v[i >> 1] & 0xffff0000u) : (v[i >> 1] << 16)); }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f32_to_bf16(v); }
// n <= E results to consecutive columns
template <int E>
__device__ __forceinline__ void put_piece(float* p, const float (&v)[E], int n) {
  typedef f32x4 vec __attribute__((aligned(4)));
  if (n == E) {
#pragma unroll
    for (int i = 0; i < E; i += 4) __builtin_nontemporal_store(vec{v[i], v[i + 1], v[i + 2], v[i + 3]}, reinterpret_cast<vec*>(p + i));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) p[i] = v[i];
  }
}
template <int E>
__device__ __forceinline__ void put_piece(bf16_t* p, const float (&v)[E], int n) {
  if (n == E) {
    if constexpr (E == 8) {
      typedef u32x4 vec __attribute__((aligned(2)));
      __builtin_nontemporal_store(vec{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])}, reinterpret_cast<vec*>(p));
    } else {
      typedef u32x2 vec __attribute__((aligned(2)));
      __builtin_nontemporal_store(vec{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}, reinterpret_cast<vec*>(p));
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) p[i] = f32_to_bf16(v[i]);
  }
}

// what a thread (a wave, the row) has seen: maximum, sums of exponentials relative to it at temperatures T and 1.
// The maximum starts at the lowest finite value: -inf then counts nothing, and a row of lowest values is uniform.
struct Seen {
  float m, s, h;
};
constexpr float LOW = -1e20f;  // logits at or below it are masked classes: their sum is one of its own, others would vanish beside it

__device__ __forceinline__ unsigned hash_of(int j) { return (unsigned)j * 2654435761u >> 16; }
// the wave reductions in 64 bits: the same exchanges as wave_sum's, on both halves (a shuffle through LDS takes five times as long)
struct Halves {
  unsigned lo, hi;
};
template <int CTRL>
__device__ __forceinline__ double dpp_mov_d(double v) {
  const Halves a = __builtin_bit_cast(Halves, v);
  return __builtin_bit_cast(double, Halves{(unsigned)__builtin_amdgcn_update_dpp(0, (int)a.lo, CTRL, 0xf, 0xf, false),
                                           (unsigned)__builtin_amdgcn_update_dpp(0, (int)a.hi, CTRL, 0xf, 0xf, false)});
}
__device__ __forceinline__ double half_row_d(double v, double& other) {  // value and partner 16 lanes away, in either order
  const Halves a = __builtin_bit_cast(Halves, v);
  const auto l = __builtin_amdgcn_permlane16_swap(a.lo, a.lo, false, false), h = __builtin_amdgcn_permlane16_swap(a.hi, a.hi, false, false);
  const unsigned l0 = l[0], l1 = l[1], h0 = h[0], h1 = h[1];
  other = __builtin_bit_cast(double, Halves{l1, h1});
  return __builtin_bit_cast(double, Halves{l0, h0});
}
__device__ __forceinline__ double half_wave_d(double v, double& other) {  // and 32 lanes away
  const Halves a = __builtin_bit_cast(Halves, v);
  const auto l = __builtin_amdgcn_permlane32_swap(a.lo, a.lo, false, false), h = __builtin_amdgcn_permlane32_swap(a.hi, a.hi, false, false);
  const unsigned l0 = l[0], l1 = l[1], h0 = h[0], h1 = h[1];
  other = __builtin_bit_cast(double, Halves{l1, h1});
  return __builtin_bit_cast(double, Halves{l0, h0});
}
template <typename F>
__device__ __forceinline__ double wave_join_d(double v, F f) {
  v = f(v, dpp_mov_d<0xB1>(v));   // quad_perm [1,0,3,2]
  v = f(v, dpp_mov_d<0x4E>(v));   // quad_perm [2,3,0,1]
  v = f(v, dpp_mov_d<0x141>(v));  // row_half_mirror
  v = f(v, dpp_mov_d<0x140>(v));  // row_mirror
  double b;
  v = half_row_d(v, b);
  v = f(v, b);
  v = half_wave_d(v, b);
  return f(v, b);
}
__device__ __forceinline__ double wave_sum_d(double v) {
  return wave_join_d(v, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double wave_max_d(double v) {
  return wave_join_d(v, [](double a, double b) { return fmax(a, b); });
}
__device__ __forceinline__ double lane_d(double v, int lane) {
  const Halves a = __builtin_bit_cast(Halves, v);
  return __builtin_bit_cast(double, Halves{(unsigned)__builtin_amdgcn_readlane((int)a.lo, lane), (unsigned)__builtin_amdgcn_readlane((int)a.hi, lane)});
}

// exp2((z - m) c) as exp2(fma(z, c, -mb)), mb = m c rounded: one instruction less an element (the exponentials are a third of the kernel's
// time at 131 072 classes).  The sums are then relative to mb, not m c: residue() puts them right.  Where m c is beyond 1e5 (a row masked with the type's
// lowest value) the plain form is taken.
__device__ __forceinline__ bool in_range(float mb) { return fabsf(mb) < 1e5f; }
__device__ __forceinline__ float residue(float m, float c) { return in_range(m * c) ? __builtin_amdgcn_exp2f(-__builtin_fmaf(m, c, -(m * c))) : 1.f; }
__device__ __forceinline__ float rescale(float from, float to, float c) {
#pragma clang fp contract(off)  // both products rounded
  if (in_range(from * c) && in_range(to * c)) return __builtin_amdgcn_exp2f(from * c - to * c);
  return __builtin_amdgcn_exp2f((from - to) * c) * residue(from, c) / residue(to, c);  // (one of them in range: a sum relative to its rounded product)
}
// SUM: and the sums of the exponents, a piece each
template <int G, bool SUM, typename T>
__device__ __forceinline__ float sum_exps(const Piece<T>* q, float m, float c, float (&x)[G]) {
  const float mb = m * c;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  auto sums = [&](auto exponent) {
#pragma unroll
    for (int k = 0; k < G; ++k) {
      x[k] = 0.f;
#pragma unroll
      for (int e = 0; e < Piece<T>::E; ++e) {
        const float v = exponent(q[k].get(e));
        s[e & 3] += __builtin_amdgcn_exp2f(v);
        if constexpr (SUM) x[k] += v;
      }
    }
  };
  if (in_range(mb)) sums([&](float z) { return __builtin_fmaf(z, c, -mb); });
  else sums([&](float z) { return (z - m) * c; });
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// over the W lanes of a group (W = 1, 4, 8, 16)
template <int W>
__device__ __forceinline__ float waves_sum(float v) {
  if constexpr (W >= 4) {
    v += dpp_mov<0xB1>(v);  // quad_perm [1,0,3,2]
    v += dpp_mov<0x4E>(v);  // quad_perm [2,3,0,1]
  }
  if constexpr (W >= 8) v += dpp_mov<0x141>(v);   // row_half_mirror
  if constexpr (W >= 16) v += dpp_mov<0x140>(v);  // row_mirror
  return v;
}
template <int W>
__device__ __forceinline__ float waves_max(float v) {
  if constexpr (W >= 4) {
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
  }
  if constexpr (W >= 8) v = fmaxf(v, dpp_mov<0x141>(v));
  if constexpr (W >= 16) v = fmaxf(v, dpp_mov<0x140>(v));
  return v;
}

// W waves a row (4 / W rows a block where W < 4), C pieces of the row kept by a thread, OCC waves a SIMD.  SUM: the sum of the logits is needed (mass of the
// teacher beside its pairs, label smoothing); a kernel of its own, as its registers cost the others 3 % at 131 072 classes.
template <typename TI, typename TO, int W, int C, int OCC, bool SUM>
__global__ __launch_bounds__(W < 4 ? 256 : 64 * W, OCC) void distill_kernel(const DistillParams p) {
  constexpr int TH = 64 * W, RPB = W < 4 ? 4 / W : 1, E = Piece<TI>::E, GROUP = C % 4 == 0 ? 4 : 2;
  static_assert(C % GROUP == 0, "whole groups");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ Seen part[RPB][W];
  __shared__ double tpart[RPB][W][2], lpart[RPB][W][2], xpart[RPB][W];
  __shared__ double mpart[RPB][W][2];
  __shared__ int distinct[RPB], repeated[RPB], masked[RPB];
  const int sub = RPB > 1 ? threadIdx.x / TH : 0;  // row of the block
  const int tid = RPB > 1 ? threadIdx.x - sub * TH : threadIdx.x;
  const int wave = tid >> 6;
  const bool first_lane = (tid & 63) == 0;
  const int row = blockIdx.x * RPB + sub;
  const int K = p.K;
  // LDS of a row: K pairs {logit / T and then its exponential, z at the class, class, what the gradient takes off there}, and a hash table of their classes
  double* tt = reinterpret_cast<double*>(smem) + (size_t)sub * K;
  float* zt = reinterpret_cast<float*>(smem + (size_t)RPB * K * 8) + (size_t)sub * K;
  int* at = reinterpret_cast<int*>(smem + (size_t)RPB * K * 12) + (size_t)sub * K;
  float* off = reinterpret_cast<float*>(smem + (size_t)RPB * K * 16) + (size_t)sub * K;
  int* table = reinterpret_cast<int*>(smem + (size_t)RPB * K * 20) + (size_t)sub * p.slots;
  const unsigned mask = p.slots - 1;

  const float weight = row < p.R ? (p.weight ? p.weight[row] : 1.0f) : 0.0f;
  const bool live = weight != 0.0f;  // rows of weight 0 are not read
  const TI* z = reinterpret_cast<const TI*>(p.z) + (size_t)row * p.ldz;
  const int pieces = (p.C + E - 1) / E, full = p.C / E;  // the last piece may be a partial one
  const int label = live && p.labels ? p.labels[row] : -1;
  const bool has_label = p.hard != 0.0f && (unsigned)label < (unsigned)p.C;
  const float zl = tid == TH - 64 && has_label ? to_float(z[label]) : 0.f;  // read before anything is written in z's place
  const bool two = p.hard != 0.0f && p.c_hard != p.c_soft;  // a second sum of exponentials
  auto fetch = [&](Piece<TI>& q, int i) {
    if (i < full) q.load(z + (size_t)i * E);
    else q.load_part(z + (size_t)i * E, p.C - i * E);
  };

  // Requests in this order: the pairs, the row, the logits at the pairs' classes (memory answers in order: pairs asked for behind the row would
  // only come with it, and the logits at their classes one more round trip later)
  const bool paired = live && tid < K;
  const int j0 = paired ? p.at[(size_t)row * K + tid] : -1;
  const float t0 = paired ? p.top[(size_t)row * K + tid] : 0.f;
  Piece<TI> r[C];
  if (live) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      r[c].clear();
      if (tid + c * TH < pieces) fetch(r[c], tid + c * TH);
    }
  }
  for (int i = tid; i < p.slots; i += TH) table[i] = -1;
  if (tid == 0) distinct[sub] = repeated[sub] = masked[sub] = 0;
  __syncthreads();

  double tm = -1.7976931348623157e308;
  float z0 = 0.f;
  if (live && 64 * wave < K) {
    int mine = 0;
    auto pair = [&](int k, int j, float t) {
      const bool ok = (unsigned)j < (unsigned)p.C;
      const double td = ok ? (double)t * p.inv_T : -__builtin_inf();
      at[k] = ok ? j : -1;
      tt[k] = td;
      tm = fmax(tm, td);
      if (ok) {  // twice as many slots as pairs: an empty one is always found
        unsigned s = hash_of(j) & mask;
        int was;
        while ((was = atomicCAS(&table[s], -1, j)) != -1 && was != j) s = (s + 1) & mask;
        if (was == -1) ++mine;
        else repeated[sub] = 1;
      }
      return ok ? to_float(z[j]) : 0.f;
    };
    if (tid < K) z0 = pair(tid, j0, t0);
    for (int k = tid + TH; k < K; k += TH) zt[k] = pair(k, p.at[(size_t)row * K + k], p.top[(size_t)row * K + k]);
    if (mine) atomicAdd(&distinct[sub], mine);
  }
  Seen me{-3.402823466e38f, 0.f, 0.f};
  double xsum = 0.0;  // of the logits, times log2 e / T
  if (live) {
    // G pieces at a time: one comparison with the running maximum, then independent exponentials (a piece at a time its short dependent
    // chains left a third of the time idle); pieces beyond the row are -inf and add nothing
    auto see = [&](const Piece<TI>* q, int i0, auto g) {
      constexpr int G = decltype(g)::value;
      float m = me.m;
#pragma unroll
      for (int k = 0; k < G; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, q[k].get(e));
      if (m != me.m) {
        me.s *= rescale(me.m, m, p.c_soft);
        if (two) me.h *= rescale(me.m, m, p.c_hard);
        me.m = m;
      }
      float x[G], none[G];
      me.s += sum_exps<G, SUM>(q, m, p.c_soft, x);
      if (two) me.h += sum_exps<G, false>(q, m, p.c_hard, none);
      if constexpr (SUM) {  // the logits' sum, in units of the exponents: what they have in common is not in it, and goes in 64 bits a group
        const float mb = m * p.c_soft;
        const bool near = in_range(mb);
        int count = 0;
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const int i = i0 + k * TH;
          count += i < full ? E : i < pieces ? p.C - full * E : 0;
          if (i >= full) {  // (columns beyond the row were -inf)
            x[k] = 0.f;
            if (i < pieces) {
#pragma unroll
              for (int e = 0; e < E; ++e)
                if (e < p.C - full * E) x[k] += near ? __builtin_fmaf(q[k].get(e), p.c_soft, -mb) : (q[k].get(e) - m) * p.c_soft;
            }
          }
        }
        float d = x[0];
#pragma unroll
        for (int k = 1; k < G; ++k) d += x[k];
        if (d > 0.5f * LOW * p.c_soft && (count == 0 || fabsf(m) < -0.1f * LOW)) xsum += (double)d + (double)count * (near ? (double)mb : (double)m * p.c_soft);
        else masked[sub] = 1;  // a masked class, perhaps: the row is summed again
      }
    };
#pragma unroll
    for (int c = 0; c < C; c += GROUP)
      if (c * TH < pieces) see(r + c, tid + c * TH, std::integral_constant<int, GROUP>{});
    for (int i = tid + C * TH; i < pieces; i += TH) {
      Piece<TI> q;
      fetch(q, i);
      see(&q, i, std::integral_constant<int, 1>{});
    }
  }
  if (tid < K) zt[tid] = z0;
  {
    me.s *= residue(me.m, p.c_soft);
    if (two) me.h *= residue(me.m, p.c_hard);
    const float M = wave_max(me.m);
    const Seen w{M, wave_sum(me.s * __builtin_amdgcn_exp2f((me.m - M) * p.c_soft)),
                 two ? wave_sum(me.h * __builtin_amdgcn_exp2f((me.m - M) * p.c_hard)) : 0.f};
    if constexpr (SUM) xsum = wave_sum_d(xsum);
    double ts = 0.0;
    if (64 * wave < K) {
      tm = p.lse ? (live ? (double)p.lse[row] : 0.0) : wave_max_d(tm);  // what this wave's sum is relative to
      if (live)
        for (int k = tid; k < K; k += TH) ts += tt[k] = exp(tt[k] - tm);  // from here on relative to the wave's
      ts = wave_sum_d(ts);
    }
    if (first_lane) {
      part[sub][wave] = w;
      if constexpr (SUM) xpart[sub][wave] = xsum;
      tpart[sub][wave][0] = tm;
      tpart[sub][wave][1] = ts;
    }
  }
  __syncthreads();

  auto is_named = [&](int j) {
    unsigned s = hash_of(j) & mask;
    while (table[s] != -1 && table[s] != j) s = (s + 1) & mask;
    return table[s] != -1;
  };
  if constexpr (SUM) {
    if (masked[sub]) {  // in 64 bits; masked classes apart, and those apart that no pair names (a named one of probability 0 takes no part)
      double all = 0.0, others = 0.0;
      xsum = 0.0;
#pragma unroll 1
      for (int i = tid; i < pieces; i += TH) {  // a thread its own pieces: nobody else writes a gradient in their place
#pragma unroll 1
        for (int j = i * E; j < (i + 1) * E && j < p.C; ++j) {
          const float v = to_float(z[j]);
          if (v <= LOW) {
            all += (double)v;
            if (!is_named(j)) others += (double)v;
          } else {
            xsum += (double)v * p.c_soft;
          }
        }
      }
      xsum = wave_sum_d(xsum);
      all = wave_sum_d(all);
      others = wave_sum_d(others);
      if (first_lane) {
        xpart[sub][wave] = xsum;
        mpart[sub][wave][0] = all;
        mpart[sub][wave][1] = others;
      }
    }
  }

  // mass of the pairs with what is left over for the classes that no pair names
  auto masses = [&](double& mass, double& left) {
    left = mass = 0.0;
    for (int w = 0; w < W && 64 * w < K; ++w) mass += tpart[sub][w][1];
    if (p.lse) {
      if (p.C > distinct[sub]) left = mass < 1.0 ? 1.0 - mass : (mass == mass ? 0.0 : mass);
      mass += left;
    } else if (mass > 0.0) {
      mass = 1.0;  // (NaN goes on)
    }
  };
  const double gs = (double)p.grad_scale * weight;
  const double hard = has_label ? p.hard : 0.0;
  float M, a_soft, a_hard = 0.f, base;
  {  // the waves' partials, one a lane: every group of W lanes joins them
    const Seen s = part[sub][tid & (W - 1)];
    M = waves_max<W>(s.m);
    const float S = waves_sum<W>(s.s * __builtin_amdgcn_exp2f((s.m - M) * p.c_soft));
    if (hard != 0.0) a_hard = (float)(gs * hard) / (two ? waves_sum<W>(s.h * __builtin_amdgcn_exp2f((s.m - M) * p.c_hard)) : S);
    double mass, left;
    masses(mass, left);
    a_soft = (float)(gs * p.soft * p.T * mass) / S;
    base = (float)(gs * p.soft * p.T * left) / (float)(left != 0.0 ? p.C - distinct[sub] : 1) + (float)(gs * hard * p.smooth) / (float)p.C;
  }
  // the gradient but for the target.  FAST: relative to M c rounded, as the sums were before residue() put them right: the same factor
  const bool fast = in_range(M * p.c_soft) && in_range(M * p.c_hard);
  const float Ms = M * p.c_soft, Mh = M * p.c_hard;
  if (fast) {
    a_soft *= residue(M, p.c_soft);
    a_hard *= residue(M, p.c_hard);
  }
  const float a_both = a_soft + a_hard;
  auto gradient = [&](float zj, auto is_fast) {
    constexpr bool FAST = decltype(is_fast)::value;
    const float es = __builtin_amdgcn_exp2f(FAST ? __builtin_fmaf(zj, p.c_soft, -Ms) : (zj - M) * p.c_soft);
    if (!two) return a_both * es;
    return a_soft * es + a_hard * __builtin_amdgcn_exp2f(FAST ? __builtin_fmaf(zj, p.c_hard, -Mh) : (zj - M) * p.c_hard);
  };
  auto gradient_any = [&](float zj) { return fast ? gradient(zj, std::true_type{}) : gradient(zj, std::false_type{}); };
  TO* dz = reinterpret_cast<TO*>(p.dz) + (size_t)row * p.lddz;
  if (p.dz && row < p.R) {
    auto give_all = [&](auto is_fast) {
      auto give = [&](const Piece<TI>& q, int i) {
        float d[E];
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = gradient(q.get(e), is_fast) - base;
        put_piece<E>(dz + (size_t)i * E, d, i < full ? E : p.C - i * E);
      };
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (tid + c * TH < pieces) give(r[c], tid + c * TH);
      for (int i = tid + C * TH; i < pieces; i += TH) {
        Piece<TI> q;
        fetch(q, i);
        give(q, i);
      }
    };
    if (live) {
      if (fast) give_all(std::true_type{});
      else give_all(std::false_type{});
    } else {
      const float d[E] = {};
      for (int i = tid; i < pieces; i += TH) put_piece<E>(dz + (size_t)i * E, d, i < full ? E : p.C - i * E);
    }
  }

  // the named classes' share of the loss, and what the gradient takes off there (while the stores above drain)
  auto join = [&](float c, bool h) {  // a sum of exponentials, in 64 bits (only after the gradient, whose registers it would take)
    double s = 0.0;
#pragma unroll 1
    for (int w = 0; w < W; ++w) s += (double)((h ? part[sub][w].h : part[sub][w].s) * __builtin_amdgcn_exp2f((part[sub][w].m - M) * c));
    return s;
  };
  asm volatile("" ::: "memory");
  double log_s = 0.0, log_h = 0.0;  // of the row's sums
  if (live && (64 * wave < K || wave == W - 1)) {
    const bool odd = two && (tid & 1);  // two logarithms for one, on even and odd lanes
    const double x = log(join(odd ? p.c_hard : p.c_soft, odd));
    log_s = lane_d(x, 0);
    log_h = two ? lane_d(x, 1) : log_s;
  }
  if (live && 64 * wave < K) {
    double ref = tpart[sub][0][0], inv = 1.0;  // P = tt inv, and exp(its wave's reference - ref) where that is another
    auto apart = [&](int w) { return tpart[sub][w][0] == ref ? 1.0 : exp(tpart[sub][w][0] - ref); };
    if (!p.lse) {
      double sum = 0.0;
      for (int w = 1; w < W && 64 * w < K; ++w) ref = fmax(ref, tpart[sub][w][0]);
      for (int w = 0; w < W && 64 * w < K; ++w) sum += tpart[sub][w][1] == 0.0 ? 0.0 : tpart[sub][w][1] * apart(w);
      inv = sum == 0.0 ? 0.0 : 1.0 / sum;
    }
    const double mine = apart(wave) * inv;
    double kl = 0.0, named = 0.0;  // (named: the sum of their logits)
    for (int k = tid; k < K; k += TH) {
      const int j = at[k];
      if (j < 0) continue;
      double P = tt[k] * mine;
      bool first = true;
      if (repeated[sub]) {  // a class named more than once has the sum, and counts once
        P = 0.0;
        for (int i = 0; i < K; ++i)
          if (at[i] == j) {
            if (i < k) first = false;
            P += tt[i] * (apart((i % TH) >> 6) * inv);
          }
      }
      off[k] = (float)(gs * (p.soft * p.T * P + hard * ((j == label ? 1.0 - p.smooth : 0.0) + (double)p.smooth / p.C)));
      if (first) {
        const double lq = (double)(zt[k] - M) * ((double)p.c_soft * LN2) - log_s;
        if (!(zt[k] <= LOW)) named += (double)zt[k];
        if (P != 0.0) kl += P * (log(P) - lq);
      }
    }
    kl = wave_sum_d(kl);
    if (p.lse) named = wave_sum_d(named);  // (asked for where mass is left over)
    if (first_lane) {
      lpart[sub][wave][0] = kl;
      lpart[sub][wave][1] = named;
    }
  }
  __syncthreads();  // the named classes are written after everybody's pieces

  if (!live) {
    if (tid == 0 && row < p.R && p.loss_rows) p.loss_rows[row] = 0.f;
    return;
  }
  if (p.dz) {
    for (int k = tid; k < K; k += TH)
      if (at[k] >= 0) put(dz + at[k], gradient_any(zt[k]) - off[k]);
  }
  if (tid != TH - 64) return;  // the row's scalars: a thread of the wave with the fewest pairs
  double mass, left;
  masses(mass, left);
  const double share = left != 0.0 ? left / (p.C - distinct[sub]) : 0.0;
  if (p.dz && has_label) {  // the label's class, unless a pair names it
    if (!is_named(label)) put(dz + label, gradient_any(zl) - (float)(gs * (p.soft * p.T * share + hard * (1.0 - p.smooth + (double)p.smooth / p.C))));
  }
  if (p.loss_rows == nullptr) return;
  double kl = 0.0, named = 0.0, loss = 0.0;
  for (int w = 0; w < W && 64 * w < K; ++w) {
    kl += lpart[sub][w][0];
    named += lpart[sub][w][1];
  }
  double Z = 0.0, masked_all = 0.0, masked_others = 0.0;
  if constexpr (SUM)
    for (int w = 0; w < W; ++w) {
      Z += xpart[sub][w];
      if (masked[sub]) {
        masked_all += mpart[sub][w][0];
        masked_others += mpart[sub][w][1];
      }
    }
  Z /= (double)p.c_soft;
  if (left != 0.0) {
    const double others = p.C - distinct[sub];
    kl += left * log(share) - share * ((Z - named + masked_others - others * M) * ((double)p.c_soft * LN2) - others * log_s);
  }
  if (p.soft != 0.0f) loss = (double)p.soft * p.T * p.T * kl;
  if (hard != 0.0) {
    double ce = log_h - (1.0 - p.smooth) * ((double)zl - M);
    if (p.smooth != 0.0f) ce -= p.smooth * ((Z + masked_all) / p.C - M);
    loss += hard * ce;
  }
  p.loss_rows[row] = (float)(loss * weight);
}

// out[c] += sum over rows of g[:, c]: 64 columns a block, 16 row strips, fixed order
template <typename T>
__global__ __launch_bounds__(1024) void distill_colsum_kernel(const T* __restrict__ g, long ld, int R, int C, float* __restrict__ out) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, strip = threadIdx.x >> 6, col = blockIdx.x * 64 + c;
  float s = 0.f;
  if (col < C) {
#pragma unroll 8
    for (int r = strip; r < R; r += 16) s += to_float(g[(size_t)r * ld + col]);
  }
  red[strip][c] = s;
  __syncthreads();
  if (strip == 0 && col < C) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][c];
    out[col] += s;
  }
}

template <typename TI, typename TO, int W, int C, int OCC>
int launch_distill(const DistillParams& p, hipStream_t st) {
  constexpr int RPB = W < 4 ? 4 / W : 1;
  auto kfn = p.lse != nullptr || p.smooth != 0.0f ? distill_kernel<TI, TO, W, C, OCC, true> : distill_kernel<TI, TO, W, C, OCC, false>;
  hipLaunchKernelGGL(kfn, dim3((unsigned)((p.R + RPB - 1) / RPB)), dim3(W < 4 ? 256 : 64 * W), (size_t)RPB * (p.K * 20 + p.slots * 4), st, p);
  SAVIT_LAUNCH_RET();
}
// A row's threads, and the pieces a thread keeps, grow with the row: a wave (no idle wave where rows are short), four, eight, sixteen; eight waves and
// more share a CU with another row's, so that one row loads while another computes or stores.  Two pieces a thread against four: [128 x 1000] fp32 7.1
// against 7.8 us, [8192 x 4000] bf16 60 / 64; eight waves of four against eight of twelve: [8192 x 8000] fp32 133 / 137, [64 x 8000] 8.5 / 8.9.
template <typename TI, typename TO>
int choose_distill(const DistillParams& p, hipStream_t st) {
  const int pieces = (p.C + Piece<TI>::E - 1) / Piece<TI>::E;
  if (pieces <= 64 * 2) return launch_distill<TI, TO, 1, 2, 4>(p, st);
  if (pieces <= 256 * 2) return launch_distill<TI, TO, 4, 2, 5>(p, st);
  if (pieces <= 256 * 4) return launch_distill<TI, TO, 4, 4, 5>(p, st);
  if (pieces <= 512 * 4) return launch_distill<TI, TO, 8, 4, 4>(p, st);
  if (pieces <= 512 * 12) return launch_distill<TI, TO, 8, 12, 4>(p, st);
  return launch_distill<TI, TO, 16, 16, 4>(p, st);
}

}  // namespace

extern "C" int savit_distill_xent(const void* logits, long ld_logits, int logits_bf16, const float* teacher_logits, const int* teacher_index, int K,
                                  const float* teacher_lse, const int* labels, const float* row_weight, float temperature, float distill_weight,
                                  float hard_weight, float label_smoothing, float grad_scale, float* loss_rows, void* dlogits, long ld_dlogits,
                                  int dlogits_bf16, float* dbias, int R, int C, void* stream) {
  SAVIT_CHECK_ARG(logits && R >= 0 && C > 0 && ld_logits >= C && K >= 0 && K <= DS_MAX_K && (K == 0 || (teacher_logits && teacher_index)));
  SAVIT_CHECK_ARG(temperature >= 1e-30f && temperature <= 1e30f && (hard_weight == 0.f || labels) && label_smoothing >= 0.f && label_smoothing <= 1.f);
  SAVIT_CHECK_ARG((dlogits || loss_rows) && (!dlogits || ld_dlogits >= C) && (!dbias || dlogits));
  SAVIT_CHECK_ARG(((uintptr_t)logits % (logits_bf16 ? 2 : 4)) == 0 && ((uintptr_t)dlogits % (dlogits_bf16 ? 2 : 4)) == 0);
  const long zs = logits_bf16 ? 2 : 4, ds = dlogits_bf16 ? 2 : 4;
  SAVIT_CHECK_ARG(dlogits == logits ? logits_bf16 == dlogits_bf16 && ld_logits == ld_dlogits
                                    : !savit_rows_overlap(dlogits, ld_dlogits * ds, C * ds, logits, ld_logits * zs, C * zs, R));
  if (R == 0) return SAVIT_OK;
  DistillParams p{};
  p.z = logits; p.top = teacher_logits; p.at = teacher_index; p.lse = teacher_lse; p.labels = labels; p.weight = row_weight;
  p.loss_rows = loss_rows; p.dz = dlogits; p.ldz = ld_logits; p.lddz = ld_dlogits; p.R = R; p.C = C; p.K = K;
  p.soft = distill_weight; p.hard = hard_weight; p.smooth = hard_weight != 0.f ? label_smoothing : 0.f; p.T = temperature;
  p.c_soft = (float)(1.4426950408889634 / (double)temperature);
  p.c_hard = 1.44269504088896340736f;
  p.inv_T = 1.0 / (double)temperature;
  p.grad_scale = grad_scale;
  for (p.slots = 16; p.slots < 2 * K; p.slots *= 2) {}
  const hipStream_t st = (hipStream_t)stream;
  int rc;
  if (logits_bf16) rc = dlogits && !dlogits_bf16 ? choose_distill<bf16_t, float>(p, st) : choose_distill<bf16_t, bf16_t>(p, st);
  else rc = dlogits && dlogits_bf16 ? choose_distill<float, bf16_t>(p, st) : choose_distill<float, float>(p, st);
  if (rc != SAVIT_OK || !dbias) return rc;
  const dim3 grid((unsigned)((C + 63) / 64));
  if (dlogits_bf16) hipLaunchKernelGGL(distill_colsum_kernel<bf16_t>, grid, dim3(1024), 0, st, (const bf16_t*)dlogits, ld_dlogits, R, C, dbias);
  else hipLaunchKernelGGL(distill_colsum_kernel<float>, grid, dim3(1024), 0, st, (const float*)dlogits, ld_dlogits, R, C, dbias);
  SAVIT_LAUNCH_RET();
}
