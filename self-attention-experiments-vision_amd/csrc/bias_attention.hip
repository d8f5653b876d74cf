// Softmax attention with an additive per-head bias, forward and backward, with the bias gradient summed over the batch.
//   S[b,h,i,j] = q_i . k_j + bias[h,i,j] ;  P = softmax_j(S) ;  O = P V                (queries arrive scaled, as in attention.hip)
//   dP = dO V^T ;  delta_i = sum_j P_ij dP_ij ;  dS = P (dP - delta) ;  dQ = dS K ;  dK = dS^T Q ;  dV = P^T dO ;  dbias[h] = sum_b dS
// The batch may be padded: keys and queries at or beyond lens[b] take no part, their rows of O and of the gradients are zero, their
// log-sum-exp -inf.  So are those of a query whose bias leaves no key (-inf, or the lowest value of float or bfloat16: scaled by log2 e it is -inf).
//
// Tiles: a wave owns 32 queries (forward, dQ) or 32 keys (dK, dV); the other side streams through LDS in segments of 64 rows shared by the
// W waves of a workgroup, fetched into registers under the arithmetic of the segment before and written to the other of two LDS buffers: one barrier a
// segment.  Scores are computed transposed (query on the lane, keys in registers) where the softmax runs along keys: its statistics are
// in-register reductions plus one half-wave exchange, and the score tile is the next product's operand without an LDS round trip.  The bias tile
// is fetched one tile ahead and is the INITIAL value of the score accumulators: adding it costs nothing.  W = 1, 2 or 4 by the sequence
// length, so that short sequences (windows) leave no wave idle.
//
// delta is summed from the fp32 probabilities, in a loop of its own over the keys, not taken as rowsum(dO . O): O is rounded to bf16, and the table
// gradient that dS feeds is an fp32 parameter gradient (2^-9 of O in delta is 1e-4 of the gradient; this way it is 1e-6).
// The bias gradient is a kernel of its own: a workgroup keeps one [queries x 64 keys] tile of one head in registers and walks over the
// images, so the sum over the batch is in a fixed order and touches memory once; long batches are cut into parts that a last launch adds.  It
// recomputes two products; a sum by atomics would move N^2 values per image and head through memory and repeat in no fixed order.
#include "attn_tiles.h"
#include "common.h"
#include "savit.h"

namespace {

constexpr float LOG2E_F = 1.4426950408889634f, LN2_F = 0.6931471805599453f;
constexpr float LOWEST = -3.402823466e38f;

struct BiasAttnParams {
  const bf16_t* qkv;
  const float* bias;   // [H, N, ldb]
  const int* lens;     // [B] or nullptr
  bf16_t* o;
  float* lse;          // [B, H, N]
  const bf16_t* d_o;
  bf16_t* dqkv;
  float* stat;         // backward: [B, H, 2, Np]: -lse log2 e (-inf where the query takes no part), delta
  float* dbias;        // [H, N, ldb], or the slab [parts][H, N, ldb]
  int B, N, H, ld, d, ldb, Np;
  int blocks;          // query (key) blocks of W * 32 rows
  int key_blocks, parts;
  float dq_scale;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* p, size_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (uint32_t)bytes, 0x00020000);
}
constexpr uint32_t OUTSIDE = 0xfffffff0u;  // beyond every descriptor's range: loads return zero

__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) { return __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0); }
__device__ __forceinline__ f32x4 load4f(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) { return __builtin_bit_cast(f32x4, load16(r, voff, soff)); }

__device__ __forceinline__ int length_of(const BiasAttnParams& p, int b) {
  if (p.lens == nullptr) return p.N;
  const int l = __builtin_amdgcn_readfirstlane(p.lens[b]);
  return l < 0 ? 0 : l > p.N ? p.N : l;
}

// two images (64 columns a row, SEG rows) of a segment: registers on their way from memory to LDS
template <int W, int KS>
struct Segment {
  static constexpr int SEG = W == 1 ? 32 : 64, LOADS = SEG * 8 / (64 * W), IMG = SEG * ROWB;
  u32x4 a[LOADS], b[LOADS];
  // rows row0 .. row0 + SEG - 1 of two column ranges of the image behind ra / rb; rows >= len and columns >= 16 KS are zero
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t ra, uint32_t lda2, uint32_t col_a2, __amdgpu_buffer_rsrc_t rb, uint32_t ldb2, uint32_t col_b2, int row0,
                                        int len) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int i = threadIdx.x + k * 64 * W, t = row0 + (i >> 3), c = i & 7;
      const bool in = t < len && c < 2 * KS;
      a[k] = load16(ra, in ? (uint32_t)t * lda2 + col_a2 + 16 * c : OUTSIDE, 0);
      b[k] = load16(rb, in ? (uint32_t)t * ldb2 + col_b2 + 16 * c : OUTSIDE, 0);
    }
  }
  __device__ __forceinline__ void put(char* img) const {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int i = threadIdx.x + k * 64 * W;
      const int off = img_off(i >> 3, i & 7);
      *reinterpret_cast<u32x4*>(img + off) = a[k];
      *reinterpret_cast<u32x4*>(img + IMG + off) = b[k];
    }
  }
};

struct Lane {
  int ql, half, trow, tcol;
  __device__ __forceinline__ Lane() {
    const int lane = threadIdx.x & 63, g = lane >> 4, t = lane & 15;
    ql = lane & 31;
    half = lane >> 5;
    trow = 4 * (g >> 1) + (t >> 2);
    tcol = 16 * (g & 1) + 4 * (t & 3);
  }
  // key (or query) that register r of a 32 x 32 tile holds
  __device__ __forceinline__ int reg(int r) const { return (r & 3) + 8 * (r >> 2) + 4 * half; }
};

// bias of a transposed tile: query on the lane (row offset in voff), keys k0 .. k0 + 31 in registers
__device__ __forceinline__ void load_bias_t(f32x16& s, __amdgpu_buffer_rsrc_t r, uint32_t voff, int k0, int N) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 v = load4f(r, voff, (uint32_t)(k0 + 8 * g) * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * g + i] = v[i];
  }
}

template <int KS>
__device__ __forceinline__ void load_frags(bf16x8 (&f)[KS], const bf16_t* base, size_t row, int ld, int col, int half, bool ok) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) f[ks] = load_row_frag_global(base, row, ld, col + 16 * ks + 8 * half, ok);
}

// S^T (or dP^T) tile: rows of the image against the lane's fragments
template <int KS>
__device__ __forceinline__ void tile_product(f32x16& s, const char* img, int row, const bf16x8 (&f)[KS], int half) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_row_frag(img, row, 2 * ks + half), f[ks], s, 0, 0, 0);
}
// out^T[e][lane] += sum over the tile's 32 rows of image[row][e] * a[row][lane]
template <int KS>
__device__ __forceinline__ void tile_accumulate(f32x16 (&out)[2], const char* img, int row0, const f32x16& a, const Lane& L) {
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
    const bf16x8 af = acc_to_frag(a, s2);
#pragma unroll
    for (int eb = 0; eb < (KS > 2 ? 2 : 1); ++eb)
      out[eb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_tr_frag(img, row0 + 16 * s2 + L.trow, 32 * eb + L.tcol), af, out[eb], 0, 0, 0);
  }
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// workgroup -> (head, image, block): all blocks and images of a head in a row, and consecutive numbers on one XCD, so that its L2 holds the
// head's bias for every image
__device__ __forceinline__ void item_of(const BiasAttnParams& p, int& h, int& b, int& blk) {
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  blk = t % p.blocks;
  const int r = t / p.blocks;
  b = r % p.B;
  h = r / p.B;
}

template <int W, int KS>
__global__ __launch_bounds__(64 * W) void bias_attn_fwd_kernel(const BiasAttnParams p) {
  typedef Segment<W, KS> Seg;
  __shared__ __attribute__((aligned(16))) char smem[4 * Seg::IMG];
  constexpr int hd = 16 * KS;
  const Lane L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int q = (blk * W + wave) * 32 + L.ql;
  const bool ok = q < len;
  const bf16_t* img = p.qkv + (size_t)b * p.N * p.ld;
  const auto rs = rsrc_of(img, (size_t)p.N * p.ld * 2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t boff = q < p.N ? (uint32_t)(q * p.ldb + 4 * L.half) * 4 : OUTSIDE;
  const uint32_t ck = (uint32_t)(p.d + h * hd) * 2, cv = ck + (uint32_t)p.d * 2;
  const int nseg = blk * W * 32 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;  // a block beyond the sequence only clears its rows
  Seg sg;
  f32x16 oacc[2] = {zero16(), zero16()};
  float m = LOWEST, l = 0.f;  // running reference (log2 units) and sum
  if (nseg > 0) {
    bf16x8 qf[KS];
    sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, 0, len);
    load_frags<KS>(qf, img, q, p.ld, h * hd, L.half, ok);
    f32x16 next;
    load_bias_t(next, rb, boff, 0, p.N);
    sg.put(smem);
    __syncthreads();
    for (int s = 0; s < nseg; ++s) {
      const bool more = s + 1 < nseg;
      if (more) sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, (s + 1) * Seg::SEG, len);
      const char* imgK = smem + (s & 1) * 2 * Seg::IMG;
      const char* imgV = imgK + Seg::IMG;
#pragma unroll
      for (int t = 0; t < Seg::SEG / 32; ++t) {
        const int k0 = s * Seg::SEG + 32 * t;
        if (k0 >= len) break;
        f32x16 sc = next;
        load_bias_t(next, rb, boff, k0 + 32, p.N);
        tile_product<KS>(sc, imgK, 32 * t + L.ql, qf, L.half);
        if (k0 + 32 > len) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (k0 + L.reg(r) >= len) sc[r] = -INFINITY;
        }
        float top = sc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, sc[r]);
        top = half_max(top) * LOG2E_F;
        // the reference follows the maximum only when it is more than 2^8 behind (P then stays below 2^8, exact in range for fp32 sums and bf16
        // operands alike): most tiles after the first skip the rescaling of the accumulators
        if (__any(top > m + 8.f)) {
          const float mn = fmaxf(m, top);
          const float alpha = __builtin_amdgcn_exp2f(m - mn);
          l *= alpha;
#pragma unroll
          for (int eb = 0; eb < 2; ++eb)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[eb][r] *= alpha;
          m = mn;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], LOG2E_F, -m));
          l += sc[r];
        }
        tile_accumulate<KS>(oacc, imgV, 32 * t, sc, L);
      }
      if (more) {
        sg.put(smem + ((s + 1) & 1) * 2 * Seg::IMG);
        __syncthreads();
      }
    }
  }
  l = half_sum(l);
  if (q < p.N) {
    const bool some = ok && l != 0.f;
    if (!some) oacc[0] = oacc[1] = zero16();
    store_row_tile(p.o + ((size_t)b * p.N + q) * p.d + h * hd, oacc, L.half, hd, some ? 1.0f / l : 0.f);
    if (L.half == 0) p.lse[((size_t)b * p.H + h) * p.N + q] = some ? (m + __log2f(l)) * LN2_F : -INFINITY;
  }
}

// dQ, and the statistics the other two kernels read.  Two loops over the keys: delta, then dQ.
template <int W, int KS>
__global__ __launch_bounds__(64 * W) void bias_attn_dq_kernel(const BiasAttnParams p) {
  typedef Segment<W, KS> Seg;
  __shared__ __attribute__((aligned(16))) char smem[4 * Seg::IMG];
  constexpr int hd = 16 * KS;
  const Lane L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int q = (blk * W + wave) * 32 + L.ql;
  const bool ok = q < len;
  const bf16_t* img = p.qkv + (size_t)b * p.N * p.ld;
  const auto rs = rsrc_of(img, (size_t)p.N * p.ld * 2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t boff = q < p.N ? (uint32_t)(q * p.ldb + 4 * L.half) * 4 : OUTSIDE;
  const uint32_t ck = (uint32_t)(p.d + h * hd) * 2, cv = ck + (uint32_t)p.d * 2;
  const int nseg = blk * W * 32 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;
  float nl = -INFINITY, delta = 0.f;
  if (ok) {
    const float v = p.lse[((size_t)b * p.H + h) * p.N + q];
    nl = v == -INFINITY ? -INFINITY : -LOG2E_F * v;
  }
  Seg sg;
  f32x16 dq[2] = {zero16(), zero16()};
  if (nseg > 0) {
    bf16x8 qf[KS], df[KS];
    sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, 0, len);
    load_frags<KS>(qf, img, q, p.ld, h * hd, L.half, ok);
    load_frags<KS>(df, p.d_o, (size_t)b * p.N + q, p.d, h * hd, L.half, ok);
    f32x16 next;
    load_bias_t(next, rb, boff, 0, p.N);
    sg.put(smem);
    __syncthreads();
    for (int s2 = 0; s2 < 2 * nseg; ++s2) {
      const bool second = s2 >= nseg, more = s2 + 1 < 2 * nseg;
      const int s = second ? s2 - nseg : s2, sn = s + 1 < nseg ? s + 1 : 0;
      if (more) sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, sn * Seg::SEG, len);
      if (s2 == nseg) delta = half_sum(delta);
      const char* imgK = smem + (s2 & 1) * 2 * Seg::IMG;
      const char* imgV = imgK + Seg::IMG;
#pragma unroll
      for (int t = 0; t < Seg::SEG / 32; ++t) {
        const int k0 = s * Seg::SEG + 32 * t;
        if (k0 >= len) break;
        f32x16 sc = next;
        load_bias_t(next, rb, boff, k0 + 32 < len ? k0 + 32 : 0, p.N);
        f32x16 dp = zero16();
        tile_product<KS>(sc, imgK, 32 * t + L.ql, qf, L.half);
        tile_product<KS>(dp, imgV, 32 * t + L.ql, df, L.half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], LOG2E_F, nl));
          if (k0 + 32 > len && k0 + L.reg(r) >= len) pr = 0.f;
          sc[r] = pr;
        }
        if (!second) {
#pragma unroll
          for (int r = 0; r < 16; ++r) delta += sc[r] * dp[r];
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[r] *= dp[r] - delta;
          tile_accumulate<KS>(dq, imgK, 32 * t, sc, L);
        }
      }
      if (more) {
        sg.put(smem + ((s2 + 1) & 1) * 2 * Seg::IMG);
        __syncthreads();
      }
    }
  }
  if (q < p.N) {
    if (!ok) dq[0] = dq[1] = zero16();
    store_row_tile(p.dqkv + ((size_t)b * p.N + q) * p.ld + h * hd, dq, L.half, hd, p.dq_scale);
  }
  if (L.half == 0 && q < p.Np) {
    float* st = p.stat + ((size_t)b * p.H + h) * 2 * p.Np + q;
    st[0] = nl;
    st[p.Np] = delta;
  }
}

// dK and dV: key on the lane, queries in registers
template <int W, int KS>
__global__ __launch_bounds__(64 * W) void bias_attn_dkv_kernel(const BiasAttnParams p) {
  typedef Segment<W, KS> Seg;
  __shared__ __attribute__((aligned(16))) char smem[4 * Seg::IMG];
  constexpr int hd = 16 * KS;
  const Lane L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int key = (blk * W + wave) * 32 + L.ql;
  const bool ok = key < len;
  const bf16_t* img = p.qkv + (size_t)b * p.N * p.ld;
  const bf16_t* imd = p.d_o + (size_t)b * p.N * p.d;
  const auto rs = rsrc_of(img, (size_t)p.N * p.ld * 2);
  const auto rd = rsrc_of(imd, (size_t)p.N * p.d * 2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const auto rt = rsrc_of(p.stat + ((size_t)b * p.H + h) * 2 * p.Np, (size_t)p.Np * 8);
  const uint32_t cq = (uint32_t)(h * hd) * 2;
  const uint32_t boff = ok ? (uint32_t)(4 * L.half * p.ldb + key) * 4 : OUTSIDE;
  const int nseg = blk * W * 32 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;
  Seg sg;
  f32x16 dk[2] = {zero16(), zero16()}, dv[2] = {zero16(), zero16()};
  if (nseg > 0) {
    bf16x8 kf[KS], vf[KS];
    sg.fetch(rs, (uint32_t)p.ld * 2, cq, rd, (uint32_t)p.d * 2, cq, 0, len);
    load_frags<KS>(kf, img, key, p.ld, p.d + h * hd, L.half, ok);
    load_frags<KS>(vf, img, key, p.ld, 2 * p.d + h * hd, L.half, ok);
    f32x16 next;
    auto load_bias = [&](int q0) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        next[r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rb, boff, (uint32_t)((q0 + (r & 3) + 8 * (r >> 2)) * p.ldb) * 4, 0));
    };
    load_bias(0);
    sg.put(smem);
    __syncthreads();
    for (int s = 0; s < nseg; ++s) {
      const bool more = s + 1 < nseg;
      if (more) sg.fetch(rs, (uint32_t)p.ld * 2, cq, rd, (uint32_t)p.d * 2, cq, (s + 1) * Seg::SEG, len);
      const char* imgQ = smem + (s & 1) * 2 * Seg::IMG;
      const char* imgD = imgQ + Seg::IMG;
#pragma unroll
      for (int t = 0; t < Seg::SEG / 32; ++t) {
        const int q0 = s * Seg::SEG + 32 * t;
        if (q0 >= len) break;
        f32x4 nl[4], dl[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          nl[g] = load4f(rt, (uint32_t)(4 * L.half) * 4, (uint32_t)(q0 + 8 * g) * 4);
          dl[g] = load4f(rt, (uint32_t)(4 * L.half) * 4, (uint32_t)(p.Np + q0 + 8 * g) * 4);
        }
        f32x16 sc = next;
        load_bias(q0 + 32);
        f32x16 dp = zero16();
        tile_product<KS>(sc, imgQ, 32 * t + L.ql, kf, L.half);
        tile_product<KS>(dp, imgD, 32 * t + L.ql, vf, L.half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], LOG2E_F, nl[r >> 2][r & 3]));
          dp[r] = sc[r] * (dp[r] - dl[r >> 2][r & 3]);
        }
        tile_accumulate<KS>(dv, imgD, 32 * t, sc, L);
        tile_accumulate<KS>(dk, imgQ, 32 * t, dp, L);
      }
      if (more) {
        sg.put(smem + ((s + 1) & 1) * 2 * Seg::IMG);
        __syncthreads();
      }
    }
  }
  if (key < p.N) {
    if (!ok) dk[0] = dk[1] = dv[0] = dv[1] = zero16();
    bf16_t* row = p.dqkv + ((size_t)b * p.N + key) * p.ld + p.d + h * hd;
    store_row_tile(row, dk, L.half, hd, 1.0f);
    store_row_tile(row + p.d, dv, L.half, hd, 1.0f);
  }
}

// dbias of a tile of 32 W queries x SEG keys of one head, summed over the images of a part
template <int W, int KS>
__global__ __launch_bounds__(64 * W) void bias_attn_db_kernel(const BiasAttnParams p) {
  typedef Segment<W, KS> Seg;
  constexpr int T = Seg::SEG / 32;
  __shared__ __attribute__((aligned(16))) char smem[4 * Seg::IMG];
  constexpr int hd = 16 * KS;
  const Lane L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int t0 = xcd_remap(blockIdx.x, gridDim.x);
  const int kb = t0 % p.key_blocks;
  t0 /= p.key_blocks;
  const int blk = t0 % p.blocks;
  t0 /= p.blocks;
  const int part = t0 % p.parts, h = t0 / p.parts;
  const int b0 = (int)((long)p.B * part / p.parts), b1 = (int)((long)p.B * (part + 1) / p.parts);
  const int q = (blk * W + wave) * 32 + L.ql, k0 = kb * Seg::SEG;
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t ck = (uint32_t)(p.d + h * hd) * 2, cv = ck + (uint32_t)p.d * 2;
  f32x16 bias[T], acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    load_bias_t(bias[t], rb, q < p.N ? (uint32_t)(q * p.ldb + 4 * L.half) * 4 : OUTSIDE, k0 + 32 * t, p.N);
    acc[t] = zero16();
  }
  Seg sg;
  auto fetch = [&](int b) {
    const auto rs = rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)p.N * p.ld * 2);
    sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, k0, length_of(p, b));
  };
  if (b0 < b1) {
    fetch(b0);
    sg.put(smem);
    __syncthreads();
  }
  for (int b = b0; b < b1; ++b) {
    const bool more = b + 1 < b1;
    const int len = length_of(p, b);
    bf16x8 qf[KS], df[KS];
    load_frags<KS>(qf, p.qkv, (size_t)b * p.N + q, p.ld, h * hd, L.half, q < len);
    load_frags<KS>(df, p.d_o, (size_t)b * p.N + q, p.d, h * hd, L.half, q < len);
    const float* st = p.stat + ((size_t)b * p.H + h) * 2 * p.Np + q;
    const float nl = q < len ? st[0] : -INFINITY, delta = q < len ? st[p.Np] : 0.f;
    if (more) fetch(b + 1);
    const char* imgK = smem + ((b - b0) & 1) * 2 * Seg::IMG;
    const char* imgV = imgK + Seg::IMG;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      f32x16 sc = bias[t], dp = zero16();
      tile_product<KS>(sc, imgK, 32 * t + L.ql, qf, L.half);
      tile_product<KS>(dp, imgV, 32 * t + L.ql, df, L.half);
      const bool edge = k0 + 32 * t + 32 > len;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float ds = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], LOG2E_F, nl)) * (dp[r] - delta);
        acc[t][r] += edge && k0 + 32 * t + L.reg(r) >= len ? 0.f : ds;
      }
    }
    if (more) {
      sg.put(smem + ((b - b0 + 1) & 1) * 2 * Seg::IMG);
      __syncthreads();
    }
  }
  if (q < p.N) {
    float* out = p.dbias + (((size_t)part * p.H + h) * p.N + q) * p.ldb + k0 + 4 * L.half;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (k0 + 32 * t + 8 * g + 4 * L.half < p.N)
          *reinterpret_cast<float4*>(out + 32 * t + 8 * g) = make_float4(acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]);
  }
}

// out = sum of the parts, in order: 64 16-byte columns a block, four strips of parts
__global__ __launch_bounds__(256) void bias_attn_parts_kernel(const float* __restrict__ slab, float* __restrict__ out, long n4, int parts) {
  __shared__ f32x4 red[4][64];
  const int c = threadIdx.x & 63, strip = threadIdx.x >> 6;
  const long i = (long)blockIdx.x * 64 + c;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < n4) {
#pragma unroll 4
    for (int k = strip; k < parts; k += 4) s += reinterpret_cast<const f32x4*>(slab)[(size_t)k * n4 + i];
  }
  red[strip][c] = s;
  __syncthreads();
  if (strip == 0 && i < n4) reinterpret_cast<f32x4*>(out)[i] = s + red[1][c] + red[2][c] + red[3][c];
}

int waves_of(int N) { return N <= 32 ? 1 : N <= 64 ? 2 : 4; }
int padded(int N) { return (N + 63) / 64 * 64; }

// parts of the batch in the dbias kernel: about four workgroups a CU, no more than there are images
int parts_of(int B, int N, int H) {
  const int W = waves_of(N);
  const long tiles = (long)H * ((N + 32 * W - 1) / (32 * W)) * ((N + (W == 1 ? 31 : 63)) / (W == 1 ? 32 : 64));
  const long want = 1024 * (4 / W) / tiles;
  return (int)(want < 1 ? 1 : want > B ? (B > 0 ? B : 1) : want);
}

bool size_ok(int B, int N, int H, int hd, int ld, int ldb) {
  if (!(B >= 0 && N > 0 && N <= 32768 && H > 0 && (hd == 16 || hd == 32 || hd == 48 || hd == 64))) return false;
  if (!(ld >= 3L * H * hd && ld % 8 == 0 && ldb >= N && ldb % 4 == 0)) return false;
  // 32-bit offsets inside one image's rows and one head's bias
  if ((long)(N + 64) * ld * 2 >= 0xfffffff0L || (long)(N + 64) * ldb * 4 >= 0xfffffff0L) return false;
  return (long)B * H * ((N + 31) / 32) <= 0x7fffffffL;
}
bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

#define BIAS_ATTN_KS(KERNEL, WV, GRID)                                                                                                              \
  switch (head_dim / 16) {                                                                                                                          \
    case 1: hipLaunchKernelGGL((KERNEL<WV, 1>), dim3((unsigned)(GRID)), dim3(64 * WV), 0, st, p); break;                                              \
    case 2: hipLaunchKernelGGL((KERNEL<WV, 2>), dim3((unsigned)(GRID)), dim3(64 * WV), 0, st, p); break;                                              \
    case 3: hipLaunchKernelGGL((KERNEL<WV, 3>), dim3((unsigned)(GRID)), dim3(64 * WV), 0, st, p); break;                                              \
    default: hipLaunchKernelGGL((KERNEL<WV, 4>), dim3((unsigned)(GRID)), dim3(64 * WV), 0, st, p); break;                                             \
  }
#define BIAS_ATTN_LAUNCH(KERNEL, GRID)                                                                                                              \
  do {                                                                                                                                              \
    if (W == 1) { BIAS_ATTN_KS(KERNEL, 1, GRID) } else if (W == 2) { BIAS_ATTN_KS(KERNEL, 2, GRID) } else { BIAS_ATTN_KS(KERNEL, 4, GRID) }           \
    const hipError_t e_ = hipGetLastError();                                                                                                        \
    if (e_ != hipSuccess) return (int)e_;                                                                                                           \
  } while (0)

}  // namespace

extern "C" int savit_bias_attention_fwd(const void* qkv, const float* bias, const int* lens, void* o, float* lse, int B, int N, int H, int head_dim, int ld_qkv,
                                        int ld_bias, void* stream) {
  SAVIT_CHECK_ARG(qkv && bias && o && lse && size_ok(B, N, H, head_dim, ld_qkv, ld_bias) && aligned16(qkv) && aligned16(bias) && aligned16(o));
  if (B == 0) return SAVIT_OK;
  BiasAttnParams p{};
  p.qkv = (const bf16_t*)qkv; p.bias = bias; p.lens = lens; p.o = (bf16_t*)o; p.lse = lse;
  p.B = B; p.N = N; p.H = H; p.ld = ld_qkv; p.d = H * head_dim; p.ldb = ld_bias;
  const int W = waves_of(N);
  const hipStream_t st = (hipStream_t)stream;
  p.blocks = (N + 32 * W - 1) / (32 * W);
  BIAS_ATTN_LAUNCH(bias_attn_fwd_kernel, (long)B * H * p.blocks);
  return SAVIT_OK;
}

extern "C" long savit_bias_attention_bwd_workspace_bytes(int B, int N, int H, int ld_bias, int want_dbias) {
  if (!(B >= 0 && N > 0 && N <= 32768 && H > 0 && ld_bias >= N)) return 0;
  const int parts = parts_of(B, N, H);
  return (long)B * H * 2 * padded(N) * 4 + (want_dbias && parts > 1 ? (long)parts * H * N * ld_bias * 4 : 0);
}

extern "C" int savit_bias_attention_bwd(const void* qkv, const float* bias, const int* lens, const void* d_o, const float* lse, void* dqkv, float* dbias, int B,
                                        int N, int H, int head_dim, int ld_qkv, int ld_bias, float dq_scale, void* workspace, long workspace_bytes,
                                        void* stream) {
  SAVIT_CHECK_ARG(qkv && bias && d_o && lse && dqkv && size_ok(B, N, H, head_dim, ld_qkv, ld_bias) && dqkv != qkv);
  SAVIT_CHECK_ARG(aligned16(qkv) && aligned16(bias) && aligned16(d_o) && aligned16(dqkv) && aligned16(dbias));
  const hipStream_t st = (hipStream_t)stream;
  if (B == 0) return dbias ? (int)SAVIT_EINVAL : SAVIT_OK;  // no image: there is no gradient to write
  SAVIT_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= savit_bias_attention_bwd_workspace_bytes(B, N, H, ld_bias, dbias != nullptr));
  BiasAttnParams p{};
  p.qkv = (const bf16_t*)qkv; p.bias = bias; p.lens = lens; p.d_o = (const bf16_t*)d_o; p.lse = const_cast<float*>(lse); p.dqkv = (bf16_t*)dqkv;
  p.B = B; p.N = N; p.H = H; p.ld = ld_qkv; p.d = H * head_dim; p.ldb = ld_bias; p.dq_scale = dq_scale;
  p.Np = padded(N);
  p.stat = (float*)workspace;
  const int W = waves_of(N);
  p.blocks = (N + 32 * W - 1) / (32 * W);
  BIAS_ATTN_LAUNCH(bias_attn_dq_kernel, (long)B * H * p.blocks);
  BIAS_ATTN_LAUNCH(bias_attn_dkv_kernel, (long)B * H * p.blocks);
  if (dbias) {
    p.parts = parts_of(B, N, H);
    const int seg = W == 1 ? 32 : 64;
    p.key_blocks = (N + seg - 1) / seg;
    p.dbias = p.parts == 1 ? dbias : p.stat + (size_t)B * H * 2 * p.Np;
    const long grid = (long)p.parts * H * p.blocks * p.key_blocks;
    SAVIT_CHECK_ARG(grid <= 0x7fffffffL);
    BIAS_ATTN_LAUNCH(bias_attn_db_kernel, grid);
    if (p.parts > 1) {
      const long n4 = (long)H * N * ld_bias / 4;
      hipLaunchKernelGGL(bias_attn_parts_kernel, dim3((unsigned)((n4 + 63) / 64)), dim3(256), 0, st, p.dbias, dbias, n4, p.parts);
      SAVIT_LAUNCH_RET();
    }
  }
  return SAVIT_OK;
}
