// Softmax attention with an additive per-head bias, forward and backward, with the bias gradient summed over the batch.
//   S[b,h,i,j] = q_i . k_j + bias[h,i,j] ;  P = softmax_j(S) ;  O = P V                (queries arrive scaled, as in attention.hip)
//   dP = dO V^T ;  delta_i = sum_j P_ij dP_ij ;  dS = P (dP - delta) ;  dQ = dS K ;  dK = dS^T Q ;  dV = P^T dO ;  dbias[h] = sum_b dS
// The batch may be padded: keys and queries at or beyond lens[b] take no part, their rows of O and of the gradients are zero, their
// log-sum-exp -inf.  So are those of a query whose bias leaves no key: scores below -2^127 are masked (-inf, the lowest values of float and bfloat16).  Any other
// mask is a number: among -1e9s alone the weights are uniform, as in a plain softmax.
//
// Tiles: a wave owns 16 or 32 queries (forward, dQ) or 16 keys (dK, dV); the other side streams through LDS in segments of 64 rows shared by the
// W waves of a workgroup, fetched into registers under the arithmetic of the segment before and written to the other of two LDS buffers: one barrier a
// segment.  Scores are computed transposed (query on the lane, keys in registers) where the softmax runs along keys: its statistics are
// in-register reductions plus an exchange between the lanes of a query, and the score tile is the next product's operand without an LDS round trip.
// The bias tile is fetched one tile ahead and is the INITIAL value of the score accumulators: adding it costs nothing.  W = 1, 2 or 4 by the sequence
// length, so that short sequences leave no wave idle.
// P and dS enter the matrix instructions as two bf16 numbers, the second what the first one's rounding took off (2^-16 of them is lost), in a product of its
// own: O and the gradients are rounded once, when stored, and are as near to 64 bits as an fp32 form's (0.0017 of their norm; with one number 0.0024).  It
// costs a tenth: [128 x 12 x 197] forward and backward 250 -> 273 us, [2048 x 4 x 49] 98 -> 107, [16 x 16 x 577] forward 66 -> 76.  Scores, statistics,
// delta, sums and dbias are fp32.
//
// What bounds it: at [128 x 12 x 197], heads of 64, the bytes take 31 us forward (59 measured) and 55 backward (107 dQ and dbias, 104 dK and dV), the
// products 20 and 50 (the low parts counted): with 2 to 3 waves a SIMD it is the chain LDS read - product - exponential - product of a tile, not one of the pipes, that the time
// goes into.  One segment or long rows come nearer: [2048 x 4 x 49], heads of 32, 26 us forward (bytes 21), 33 dK and dV (31 from memory; some of it is
// still in the caches), 37 dQ and dbias.
//
// delta is summed from the fp32 probabilities, in a loop of its own over the keys, not taken as rowsum(dO . O): O is rounded to bf16, and the table
// gradient that dS feeds is an fp32 parameter gradient (2^-9 of O in delta is 1e-4 of the gradient; this way it is 1e-6).
// Up to 224 tokens dQ and the bias gradient are one kernel with the keys resident (below).  Beyond, the bias gradient is a kernel of its own: a workgroup keeps one [queries x 64 keys] tile of one head in registers and walks over the
// images, so the sum over the batch is in a fixed order and touches memory once; long batches are cut into parts that a last launch adds.  It
// recomputes two products; a sum by atomics would move N^2 values per image and head through memory and repeat in no fixed order.
#include <type_traits>

#include "attn_tiles.h"
#include "common.h"
#include "savit.h"

namespace {

constexpr float LOG2E_F = 1.4426950408889634f, LN2_F = 0.6931471805599453f;
// A row's exponentials are exp2(s log2 e - r), r = reference(m) of a score m of the row.  One multiply-add an element: its product is exact, so r has to be m log2 e
// exactly where that is far from zero - rounded to 32 bits it is off by 440 at a mask of -1e10.  It is a pair there, and the exponentials are
// exp2((s - m) log2 e), an instruction more; b alone up to |m| = 2^20, where what b was rounded by (2^-4 at the most) is common to a row's sum and products.
constexpr float FAR = 1048576.f;
// Scores below it are masked: -inf, float's and bfloat16's lowest values; a row of nothing else is empty.  (A power of two: its own reference is exact.)
constexpr float MASKED = -1.7014118346046923e38f;
struct Reference {
  float b, lo;  // b + lo
};
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= FAR && m != MASKED; }
__device__ __forceinline__ Reference reference(float m) {
#pragma clang fp contract(off)  // b is the ROUNDED product, wherever it goes
  const float b = m * LOG2E_F;
  return {b, fabsf(m) < FAR ? 0.f : __builtin_fmaf(m, LOG2E_F, -b)};
}

struct BiasAttnParams {
  const bf16_t* qkv;
  const float* bias;   // [H, N, ldb]
  const int* lens;     // [B] or nullptr
  bf16_t* o;
  float* lse;          // [B, H, N]
  const bf16_t* d_o;
  bf16_t* dqkv;
  float* stat;         // backward: [B, H, 3, Np]: P = exp2((s - first) log2 e - second); the first is inf where the query takes no part; delta
  float* dbias;        // [H, N, lddb], or the slab [parts][H, N, lddb]
  int B, N, H, ld, d, ldb, lddb, Np;
  int hd;
  int blocks;          // query (key) blocks of a sequence
  int key_blocks, parts;
  int image_major;     // workgroups: all heads of an image in a row, or all images of a head
  float dq_scale;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* p, size_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (uint32_t)bytes, 0x00020000);
}
constexpr uint32_t OUTSIDE = 0xfffffff0u;  // beyond every descriptor's range (below 0xfff00000): loads return zero
constexpr uint32_t BEYOND = 0xfff00000u;   // the same for an offset that something below 1 MB is still added to

// (the scalar offset of these loads takes no part in the range check: it is always 0 here)
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off) { return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0); }
__device__ __forceinline__ f32x4 load4f(__amdgpu_buffer_rsrc_t r, uint32_t off) { return __builtin_bit_cast(f32x4, load16(r, off)); }

__device__ __forceinline__ void store16(__amdgpu_buffer_rsrc_t r, uint32_t off, u32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, 0); }
// off, or beyond every range.  Opaque: the compiler makes two loads in two branches of a plain choice.  (What is in flight is counted: behind a
// branch with a load or store in it, the count is not known and every wait is for everything - the segment just asked for included.  The kernels here
// therefore fetch unconditionally, out of range where there is nothing to fetch.)
__device__ __forceinline__ uint32_t only(bool in, uint32_t off) {
  uint32_t m = in ? 0u : OUTSIDE;
  asm("" : "+v"(m));
  return off | m;
}

__device__ __forceinline__ int length_of(const BiasAttnParams& p, int b) {
  if (p.lens == nullptr) return p.N;
  const int l = __builtin_amdgcn_readfirstlane(p.lens[b]);
  return l < 0 ? 0 : l > p.N ? p.N : l;
}

// Byte offset of 16-byte chunk c of an image's row (ROWB bytes).  The XOR by row bits 1..3 serves both shapes without bank conflicts: row fragments of
// 16 rows x 4 chunks (a pass of ds_read_b128 takes rows 0-3 and 12-15 of one chunk with rows 4-11 of its neighbour) or 32 rows x 2, and transposed reads
// of 16 rows x 2 chunks or 4 rows x 4.  (attention.hip's order of the bits is made for its 32-row tiles; 16 rows of it conflict: 38 % of dK / dV's LDS cycles.)
__device__ __forceinline__ int swizzle(int row) { return (row >> 1 & 1) << 2 | ((row >> 2 ^ row >> 3) & 1) << 1 | (row >> 3 & 1); }
__device__ __forceinline__ int at_chunk(int row, int c) { return row * ROWB + ((c ^ swizzle(row)) << 4); }
__device__ __forceinline__ bf16x8 row_frag(const char* img, int row, int c) { return *reinterpret_cast<const bf16x8*>(img + at_chunk(row, c)); }
__device__ __forceinline__ bf16x4 read_tr(const char* img, int row, int col) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(img + at_chunk(row, col >> 3) + ((col & 7) << 1)));
}

// two images (64 columns a row, SEG rows) of a segment: registers on their way from memory to LDS
template <int W, int KS>
struct Segment {
  static constexpr int SEG = W == 1 ? 32 : 64, LOADS = SEG * 8 / (64 * W), IMG = SEG * ROWB;
  u32x4 a[LOADS], b[LOADS];
  // rows row0 .. row0 + SEG - 1 of two column ranges of the image behind ra / rb; rows >= len and 16-byte chunks >= `chunks` of a row are zero
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t ra, uint32_t lda2, uint32_t col_a2, __amdgpu_buffer_rsrc_t rb, uint32_t ldb2, uint32_t col_b2, int row0,
                                        int len, int chunks = 2 * KS) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int i = threadIdx.x + k * 64 * W, t = row0 + (i >> 3), c = i & 7;
      const bool in = t < len && c < chunks;
      a[k] = load16(ra, in ? (uint32_t)t * lda2 + col_a2 + 16 * c : OUTSIDE);
      b[k] = load16(rb, in ? (uint32_t)t * ldb2 + col_b2 + 16 * c : OUTSIDE);
    }
  }
  __device__ __forceinline__ void put(char* img) const {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int i = threadIdx.x + k * 64 * W;
      const int off = at_chunk(i >> 3, i & 7);
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

// bias of a transposed tile: query on the lane (voff: its row; BEYOND: none), keys k0 .. k0 + 31 in registers
__device__ __forceinline__ void load_bias_t(f32x16& s, __amdgpu_buffer_rsrc_t r, uint32_t voff, int k0) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 v = load4f(r, voff + (uint32_t)(k0 + 8 * g) * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * g + i] = v[i];
  }
}

// S^T (or dP^T) tile: rows of the image against the lane's fragments
template <int KS>
__device__ __forceinline__ void tile_product(f32x16& s, const char* img, int row, const bf16x8 (&f)[KS], int half) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag(img, row, 2 * ks + half), f[ks], s, 0, 0, 0);
}
// what the rounding of (a, b) to the bf16 pair u took off, as another pair: the operand of a second product
__device__ __forceinline__ uint32_t low_parts(uint32_t u, float a, float b) {
  return pack_bf16x2(a - __builtin_bit_cast(float, u << 16), b - __builtin_bit_cast(float, u & 0xffff0000u));
}
// out^T[e][lane] += sum over the tile's 32 rows of image[row][e] * a[row][lane], a as two bf16 (heads of 48 and 64)
__device__ __forceinline__ void tile_accumulate(f32x16 (&out)[2], const char* img, int row0, const f32x16& a, const Lane& L) {
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
    union { uint32_t u[4]; bf16x8 v; } hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = a[8 * s2 + 2 * j], y = a[8 * s2 + 2 * j + 1];
      hi.u[j] = pack_bf16x2(x, y);
      lo.u[j] = low_parts(hi.u[j], x, y);
    }
    bf16x8 vf[2];
#pragma unroll
    for (int eb = 0; eb < 2; ++eb) {
      const int row = row0 + 16 * s2 + L.trow, col = 32 * eb + L.tcol;
      vf[eb] = __builtin_shufflevector(read_tr(img, row, col), read_tr(img, row + 8, col), 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int eb = 0; eb < 2; ++eb) out[eb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[eb], hi.v, out[eb], 0, 0, 0);
#pragma unroll
    for (int eb = 0; eb < 2; ++eb) out[eb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[eb], lo.v, out[eb], 0, 0, 0);
  }
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// keys k0 + .. of a transposed tile that lie at or beyond len get v
__device__ __forceinline__ void mask_keys(f32x16& s, int k0, int len, const Lane& L, float v) {
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (k0 + L.reg(r) >= len) s[r] = v;
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// rows row0 .. row0 + 3 and row0 + 16 .. + 19 (row0 = 4 (lane / 16)) of columns col0 .. + 15: A operand whose k order is that of two stacked 16 x 16
// accumulators
__device__ __forceinline__ bf16x8 lds_tr_pair(const char* img, int row, int col) {
  const bf16x4 lo = read_tr(img, row, col), hi = read_tr(img + 16 * ROWB, row, col);  // (16 rows on: the same swizzle)
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// sum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quarters_sum(float v) {
  float a = v, b = v;
  permlane16_swap(a, b);
  return half_sum(a + b);
}

__device__ __forceinline__ float quarters_max(float v) {
  float a = v, b = v;
  permlane16_swap(a, b);
  return half_max(fmaxf(a, b));
}
// Columns of the 2 KS2 accumulators of a lane's row (16 eb + 4 (lane / 16) ..), scaled, rounded and stored 16 bytes at a time: lanes 16 apart trade pieces of
// two accumulators first.  Columns >= hd are skipped.
template <int KS2, typename F>
__device__ __forceinline__ void pieces_of_row16(const f32x4 (&o)[2 * KS2], int g, float sc, F store) {
#pragma unroll
  for (int eb = 0; eb < 2 * KS2; eb += 2) {
    uint32_t a0 = pack_bf16x2(o[eb][0] * sc, o[eb][1] * sc), a1 = pack_bf16x2(o[eb][2] * sc, o[eb][3] * sc);
    uint32_t b0 = pack_bf16x2(o[eb + 1][0] * sc, o[eb + 1][1] * sc), b1 = pack_bf16x2(o[eb + 1][2] * sc, o[eb + 1][3] * sc);
    const auto r0 = __builtin_amdgcn_permlane16_swap(a0, b0, false, false), r1 = __builtin_amdgcn_permlane16_swap(a1, b1, false, false);
    store((g & 1) ? 16 * (eb + 1) + 4 * (g - 1) : 16 * eb + 4 * g, u32x4{(uint32_t)r0[0], (uint32_t)r1[0], (uint32_t)r0[1], (uint32_t)r1[1]});
  }
}
template <int KS2>
__device__ __forceinline__ void store_row16(bf16_t* row, const f32x4 (&o)[2 * KS2], int g, int hd, float sc) {
  pieces_of_row16<KS2>(o, g, sc, [&](int col, u32x4 v) {
    if (col < hd) *reinterpret_cast<u32x4*>(row + col) = v;
  });
}

// workgroup -> (head, image, block), consecutive numbers on one XCD.  All images of a head in a row: the L2 holds the head's bias for every image.
// All heads of an image in a row: the L2 holds every head's bias, and the heads' pieces of a row, which lie next to each other in memory, are read
// together (many_heads)
__device__ __forceinline__ void item_of(const BiasAttnParams& p, int& h, int& b, int& blk) {
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  blk = t % p.blocks;
  const int r = t / p.blocks;
  b = p.image_major ? r / p.H : r % p.B;
  h = p.image_major ? r % p.H : r / p.B;
}

// forward: the reference's score follows the maximum once it is 2^8 behind; returns what the sums so far are multiplied by
constexpr float BEHIND = 5.5f;
__device__ __forceinline__ float follow(float& m, float top) {
#pragma clang fp contract(off)
  const Reference from = reference(m);
  m = fmaxf(m, top);
  const Reference to = reference(m);
  return __builtin_amdgcn_exp2f((from.b - to.b) + (from.lo - to.lo));
}
// m + log l: the sum was relative to reference(m), which is m log2 e but for b's rounding
__device__ __forceinline__ float log_sum(float m, float l) {
#pragma clang fp contract(off)
  const Reference rf = reference(m);
  return __builtin_fmaf(__log2f(l) - (__builtin_fmaf(m, LOG2E_F, -rf.b) - rf.lo), LN2_F, m);
}

// backward: the exponentials are taken relative to a row's log-sum-exp.  That is one 32-bit number: far from zero it holds the row's maximum and little of the
// sum's logarithm.  The dQ kernels, which see all of a row, therefore sum the exponentials again: P is the forward's whatever the scores have in common (taken
// from the log-sum-exp alone it was off by 1e-3 at a common bias of 1e4, by a factor of 230 in a row of nothing but -1e8).
struct RowReference {
  float less, b;  // exponentials: exp2((s - less) log2 e - b); s - less where some row of the wave is far
  float shift;    // b + less log2 e - m log2 e
  bool far;
  __device__ __forceinline__ RowReference(float m) {
#pragma clang fp contract(off)
    far = fabsf(m) >= FAR && m != INFINITY;  // (inf, a row that takes no part: its exponentials are 0)
    less = far ? m : 0.f;
    b = far ? 0.f : m * LOG2E_F;
    shift = far ? 0.f : -__builtin_fmaf(m, LOG2E_F, -b);
  }
  // log2 of the sum relative to m log2 e, of one relative to this
  __device__ __forceinline__ float rest(float sum) const { return sum == 0.f ? 0.f : __log2f(sum) + shift; }
};
// a row's log-sum-exp as a reference: inf where it takes no part
__device__ __forceinline__ float or_none(float lse) { return lse == -INFINITY ? INFINITY : lse; }

template <int KS>
__global__ __launch_bounds__(256, 3) void bias_attn_fwd_kernel(const BiasAttnParams p) {
  constexpr int W = 4;
  typedef Segment<W, KS> Seg;
  __shared__ __attribute__((aligned(16))) char smem[4 * Seg::IMG];
  constexpr int hd = 16 * KS;
  const Lane L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int q = (blk * W + wave) * 32 + L.ql;
  const bool ok = q < len, live = (blk * W + wave) * 32 < len;  // live: some query of the wave is
  const auto rs = rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)p.N * p.ld * 2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t boff = q < p.N ? (uint32_t)(q * p.ldb + 4 * L.half) * 4 : BEYOND;
  const uint32_t ck = (uint32_t)(p.d + h * hd) * 2, cv = ck + (uint32_t)p.d * 2;
  const int nseg = blk * W * 32 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;  // a block beyond the sequence only clears its rows
  Seg sg;
  f32x16 oacc[2] = {zero16(), zero16()};
  float m = MASKED, l = 0.f;  // score that the reference is made of, and the running sum relative to it
  bool far = false;           // some query of the wave has one far from zero
  if (nseg > 0) {
    bf16x8 qf[KS];
    sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, 0, len);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(ok, (uint32_t)q * p.ld * 2 + (h * hd + 16 * ks + 8 * L.half) * 2)));
    f32x16 next;
    load_bias_t(next, rb, boff, 0);
    sg.put(smem);
    __syncthreads();
    auto segment = [&](int s, auto more) {
      const char* imgK = smem + (s & 1) * 2 * Seg::IMG;
      const char* imgV = imgK + Seg::IMG;
#pragma unroll
      for (int t = 0; t < Seg::SEG / 32; ++t) {
        const int k0 = s * Seg::SEG + 32 * t;
        f32x16 sc = next;
        if (more || t == 0) load_bias_t(next, rb, boff, k0 + 32);
        if (more && t == 0) sg.fetch(rs, (uint32_t)p.ld * 2, ck, rs, (uint32_t)p.ld * 2, cv, (s + 1) * Seg::SEG, len);  // (behind the bias: loads arrive in order)
        if (!live || (!more && k0 >= len)) continue;
        tile_product<KS>(sc, imgK, 32 * t + L.ql, qf, L.half);
        if (!more && k0 + 32 > len) mask_keys(sc, k0, len, L, -INFINITY);
        float top = sc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, sc[r]);
        top = half_max(top);
        // the reference follows the maximum only when it is more than 2^8 behind (P then stays below 2^8, exact in range for fp32 sums and bf16
        // operands alike): most tiles after the first skip the rescaling of the accumulators
        if (__any(top > m + BEHIND)) {
          const float alpha = follow(m, top);
          l *= alpha;
#pragma unroll
          for (int eb = 0; eb < 2; ++eb)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[eb][r] *= alpha;
          far = __any(is_far(m));
        }
        float ref = m * LOG2E_F;
        if (far) {
          const float less = is_far(m) ? m : 0.f;
          if (is_far(m)) ref = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[r] -= less;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], LOG2E_F, -ref));
          l += sc[r];
        }
        tile_accumulate(oacc, imgV, 32 * t, sc, L);
      }
      if constexpr (more) {
        sg.put(smem + ((s + 1) & 1) * 2 * Seg::IMG);
        __syncthreads();
      }
    };
    for (int s = 0; s + 1 < nseg; ++s) segment(s, std::true_type{});
    segment(nseg - 1, std::false_type{});
  }
  l = half_sum(l);
  if (q < p.N) {
    const bool some = ok && l != 0.f;
    if (!some) oacc[0] = oacc[1] = zero16();
    store_row_tile(p.o + ((size_t)b * p.N + q) * p.d + h * hd, oacc, L.half, hd, some ? 1.0f / l : 0.f);
    if (L.half == 0) p.lse[((size_t)b * p.H + h) * p.N + q] = some ? log_sum(m, l) : -INFINITY;
  }
}

// The same with 16 queries a wave (ONE: and no more keys than a segment; else the last segment asks for one that is out of range): twice the waves of half the registers, for narrow heads, short sequences and grids that leave SIMDs empty.  What
// it reads from LDS serves half as many queries.
template <int W, int KS2, bool ONE>
__global__ __launch_bounds__(64 * W, W == 4 ? 4 : 3) void bias_attn_fwd16_kernel(const BiasAttnParams p) {
  typedef Segment<W, 2 * KS2> Seg;
  constexpr int T = Seg::SEG / 16;
  __shared__ __attribute__((aligned(16))) char smem[(ONE ? 2 : 4) * Seg::IMG];
  const int lane = threadIdx.x & 63, ql = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int q = (blk * W + wave) * 16 + ql;
  const uint32_t ld2 = (uint32_t)p.ld * 2, d2 = (uint32_t)p.d * 2, hcol = (uint32_t)(h * p.hd) * 2;
  const auto rs = rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)len * ld2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t boff = q < p.N ? (uint32_t)(q * p.ldb + 4 * g) * 4 : BEYOND;
  const int nseg = blk * W * 16 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;
  Seg sg;
  f32x4 o[2 * KS2];
#pragma unroll
  for (int eb = 0; eb < 2 * KS2; ++eb) o[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = MASKED, l = 0.f;  // as above
  bool far = false;
  if (nseg > 0) {
    bf16x8 qf[KS2];
    sg.fetch(rs, ld2, d2 + hcol, rs, ld2, 2 * d2 + hcol, 0, len, p.hd / 8);
#pragma unroll
    for (int ks = 0; ks < KS2; ++ks) {
      const int c = 32 * ks + 8 * g;
      qf[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(c < p.hd, (uint32_t)q * ld2 + hcol + 2 * c)));
    }
    f32x4 sc[T];
#pragma unroll
    for (int t = 0; t < T; ++t) sc[t] = load4f(rb, boff + 64 * t);
    sg.put(smem);
    __syncthreads();
    for (int s = 0; s < (ONE ? 1 : nseg); ++s) {
      const int k0 = s * Seg::SEG;
      if constexpr (!ONE) {
        sg.fetch(rs, ld2, d2 + hcol, rs, ld2, 2 * d2 + hcol, k0 + Seg::SEG, len, p.hd / 8);
        __builtin_amdgcn_sched_barrier(0);  // (else the loads sink to their use)
      }
      const char* imgK = smem + (s & 1) * 2 * Seg::IMG;
      const char* imgV = imgK + Seg::IMG;
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int ks = 0; ks < KS2; ++ks) sc[t] = mfma16(row_frag(imgK, 16 * t + ql, 4 * ks + g), qf[ks], sc[t]);
      if (k0 + Seg::SEG > len) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (k0 + 16 * t + 4 * g + r >= len) sc[t][r] = -INFINITY;
      }
      float top = sc[0][0];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, sc[t][r]);
      top = quarters_max(top);
      if (__any(top > m + BEHIND)) {
        const float alpha = follow(m, top);
        l *= alpha;
#pragma unroll
        for (int eb = 0; eb < 2 * KS2; ++eb) o[eb] *= alpha;
        far = __any(is_far(m));
      }
      float ref = m * LOG2E_F;
      if (far) {
        const float less = is_far(m) ? m : 0.f;
        if (is_far(m)) ref = 0.f;
#pragma unroll
        for (int t = 0; t < T; ++t) sc[t] -= less;
      }
#pragma unroll
      for (int t = 0; t < T; t += 2) {
        union { uint32_t u[4]; bf16x8 v; } pf, pl;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x4& x = sc[t + k];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], LOG2E_F, -ref));
            l += x[r];
          }
          pf.u[2 * k] = pack_bf16x2(x[0], x[1]);
          pf.u[2 * k + 1] = pack_bf16x2(x[2], x[3]);
          pl.u[2 * k] = low_parts(pf.u[2 * k], x[0], x[1]);
          pl.u[2 * k + 1] = low_parts(pf.u[2 * k + 1], x[2], x[3]);
          if constexpr (!ONE) x = load4f(rb, boff + (uint32_t)(k0 + Seg::SEG + 16 * (t + k)) * 4);
        }
#pragma unroll
        for (int eb = 0; eb < 2 * KS2; ++eb) {
          const bf16x8 vf = lds_tr_pair(imgV, 16 * t + 4 * g + (ql >> 2), 16 * eb + 4 * (ql & 3));
          o[eb] = mfma16(vf, pf.v, o[eb]);
          o[eb] = mfma16(vf, pl.v, o[eb]);
        }
      }
      if (!ONE && s + 1 < nseg) {
        sg.put(smem + ((s + 1) & 1) * 2 * Seg::IMG);
        __syncthreads();
      }
    }
  }
  l = quarters_sum(l);
  if (q < p.N) {
    const bool some = q < len && l != 0.f;
    if (!some) {
#pragma unroll
      for (int eb = 0; eb < 2 * KS2; ++eb) o[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    store_row16<KS2>(p.o + ((size_t)b * p.N + q) * p.d + h * p.hd, o, g, p.hd, some ? 1.0f / l : 0.f);
    if (g == 0) p.lse[((size_t)b * p.H + h) * p.N + q] = some ? log_sum(m, l) : -INFINITY;
  }
}

// dQ, and the statistics the other two kernels read.  Two loops over the keys: delta, then dQ.  16 queries a wave.
template <int KS2>
__global__ __launch_bounds__(256, 3) void bias_attn_dq_kernel(const BiasAttnParams p) {
  constexpr int W = 4;
  typedef Segment<W, 2 * KS2> Seg;
  constexpr int T = Seg::SEG / 16;
  __shared__ __attribute__((aligned(16))) char smem[4 * Seg::IMG];
  const int lane = threadIdx.x & 63, ql = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int q = (blk * W + wave) * 16 + ql;
  const uint32_t ld2 = (uint32_t)p.ld * 2, d2 = (uint32_t)p.d * 2, hcol = (uint32_t)(h * p.hd) * 2;
  const auto rs = rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)len * ld2);
  const auto ro = rsrc_of(p.d_o + (size_t)b * p.N * p.d, (size_t)len * d2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t boff = q < p.N ? (uint32_t)(q * p.ldb + 4 * g) * 4 : BEYOND;
  const int nseg = blk * W * 16 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;
  const float m = or_none(q < len ? p.lse[((size_t)b * p.H + h) * p.N + q] : -INFINITY);
  const RowReference rf(m);
  const bool far = __any(rf.far);
  float delta = 0.f, sum = 0.f, inv = 0.f;
  Seg sg;
  f32x4 dq[2 * KS2];
#pragma unroll
  for (int eb = 0; eb < 2 * KS2; ++eb) dq[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (nseg > 0) {
    bf16x8 qf[KS2], df[KS2];
    sg.fetch(rs, ld2, d2 + hcol, rs, ld2, 2 * d2 + hcol, 0, len, p.hd / 8);
#pragma unroll
    for (int ks = 0; ks < KS2; ++ks) {
      const int c = 32 * ks + 8 * g;
      qf[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(c < p.hd, (uint32_t)q * ld2 + hcol + 2 * c)));
      df[ks] = __builtin_bit_cast(bf16x8, load16(ro, only(c < p.hd, (uint32_t)q * d2 + hcol + 2 * c)));
    }
    f32x4 sc[T];
#pragma unroll
    for (int t = 0; t < T; ++t) sc[t] = load4f(rb, boff + 64 * t);
    sg.put(smem);
    __syncthreads();
    int buf = 0;
    auto pass = [&](auto second) {
      for (int k0 = 0; k0 < len; k0 += Seg::SEG) {
        const bool last = k0 + Seg::SEG >= len, more = !last || !second;
        const int kn = last && !second ? 0 : k0 + Seg::SEG;
        sg.fetch(rs, ld2, d2 + hcol, rs, ld2, 2 * d2 + hcol, kn, len, p.hd / 8);
        __builtin_amdgcn_sched_barrier(0);  // (else the loads sink to their use)
        const char* imgK = smem + buf * 2 * Seg::IMG;
        const char* imgV = imgK + Seg::IMG;
        f32x4 dp[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
          dp[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS2; ++ks) {
            sc[t] = mfma16(row_frag(imgK, 16 * t + ql, 4 * ks + g), qf[ks], sc[t]);
            dp[t] = mfma16(row_frag(imgV, 16 * t + ql, 4 * ks + g), df[ks], dp[t]);
          }
        }
        if (far) {
#pragma unroll
          for (int t = 0; t < T; ++t) sc[t] -= rf.less;
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], LOG2E_F, -rf.b));
        if (last) {
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (k0 + 16 * t + 4 * g + r >= len) sc[t][r] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < T; t += 2) {
          union { uint32_t u[4]; bf16x8 v; } pf, pl;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            f32x4& x = sc[t + k];
            if constexpr (second) {
              x = x * (dp[t + k] - delta);
              pf.u[2 * k] = pack_bf16x2(x[0], x[1]);
              pf.u[2 * k + 1] = pack_bf16x2(x[2], x[3]);
              pl.u[2 * k] = low_parts(pf.u[2 * k], x[0], x[1]);
              pl.u[2 * k + 1] = low_parts(pf.u[2 * k + 1], x[2], x[3]);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                sum += x[r];
                delta += x[r] * dp[t + k][r];
              }
            }
            x = load4f(rb, boff + (uint32_t)(kn + 16 * (t + k)) * 4);
          }
          if constexpr (second) {
#pragma unroll
            for (int eb = 0; eb < 2 * KS2; ++eb) {
              const bf16x8 kf = lds_tr_pair(imgK, 16 * t + 4 * g + (ql >> 2), 16 * eb + 4 * (ql & 3));
              dq[eb] = mfma16(kf, pf.v, dq[eb]);
              dq[eb] = mfma16(kf, pl.v, dq[eb]);
            }
          }
        }
        if (more) {
          buf ^= 1;
          sg.put(smem + buf * 2 * Seg::IMG);
          __syncthreads();
        }
      }
    };
    pass(std::false_type{});
    sum = quarters_sum(sum);
    inv = sum == 0.f ? 0.f : 1.f / sum;
    delta = quarters_sum(delta) * inv;
    pass(std::true_type{});
  }
  float rest = rf.rest(sum);
  if (q >= len) {  // whatever the bias holds in such a row
    delta = rest = inv = 0.f;
#pragma unroll
    for (int eb = 0; eb < 2 * KS2; ++eb) dq[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (q < p.N) store_row16<KS2>(p.dqkv + ((size_t)b * p.N + q) * p.ld + h * p.hd, dq, g, p.hd, p.dq_scale * inv);
  if (g == 0 && q < p.Np) {
    float* st = p.stat + ((size_t)b * p.H + h) * 3 * p.Np + q;
    st[0] = m;
    st[p.Np] = rest;
    st[2 * p.Np] = delta;
  }
}

// dK and dV: a wave owns 16 keys (on the lane; queries in registers), Q and dO stream.  16 and not 32 keys a wave: 64 accumulators fewer leave room for four waves
// a SIMD instead of two, which is worth more than the LDS reads that 32 keys would share
template <int W, int KS2, bool ONE>
__global__ __launch_bounds__(64 * W, W == 2 ? 2 : 3) void bias_attn_dkv_kernel(const BiasAttnParams p) {
  typedef Segment<W, 2 * KS2> Seg;
  constexpr int T = Seg::SEG / 16;
  __shared__ __attribute__((aligned(16))) char smem[(ONE ? 2 : 4) * Seg::IMG];
  constexpr int SL = (3 * Seg::SEG + 64 * W - 1) / (64 * W);
  __shared__ __attribute__((aligned(16))) float stats[ONE ? 1 : 2][64 * W * SL];  // of the two buffers: SEG of each of the three statistics (and what the other threads write)
  const int lane = threadIdx.x & 63, ql = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, b, blk;
  item_of(p, h, b, blk);
  const int len = length_of(p, b);
  const int key = (blk * W + wave) * 16 + ql;
  const bool ok = key < len, live = (blk * W + wave) * 16 < len;  // live: some key of the wave is
  const uint32_t ld2 = (uint32_t)p.ld * 2, d2 = (uint32_t)p.d * 2, hcol = (uint32_t)(h * p.hd) * 2;
  const auto rs = rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)len * ld2);
  const auto rd = rsrc_of(p.d_o + (size_t)b * p.N * p.d, (size_t)len * d2);
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const auto rt = rsrc_of(p.stat + ((size_t)b * p.H + h) * 3 * p.Np, (size_t)p.Np * 12);
  const uint32_t boff = (uint32_t)(4 * g * p.ldb + key) * 4, brow = (uint32_t)p.ldb * 4;
  const int nseg = blk * W * 16 < len ? (len + Seg::SEG - 1) / Seg::SEG : 0;
  Seg sg;
  float st[SL];
  auto fetch = [&](int q0) {
    sg.fetch(rs, ld2, hcol, rd, d2, hcol, q0, len, p.hd / 8);
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      const uint32_t i = threadIdx.x + k * 64 * W, row = q0 + i % Seg::SEG + i / Seg::SEG * p.Np;
      st[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rt, i < 3 * Seg::SEG ? row * 4 : OUTSIDE, 0, 0));
    }
  };
  auto put = [&](int buf) {
    sg.put(smem + buf * 2 * Seg::IMG);
#pragma unroll
    for (int k = 0; k < SL; ++k) stats[buf][threadIdx.x + k * 64 * W] = st[k];
  };
  f32x4 dk[2 * KS2], dv[2 * KS2];
#pragma unroll
  for (int eb = 0; eb < 2 * KS2; ++eb) dk[eb] = dv[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (nseg > 0) {
    bf16x8 kf[KS2], vf[KS2];
    fetch(0);
#pragma unroll
    for (int ks = 0; ks < KS2; ++ks) {
      const int c = 32 * ks + 8 * g;
      kf[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(c < p.hd, (uint32_t)key * ld2 + d2 + hcol + 2 * c)));
      vf[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(c < p.hd, (uint32_t)key * ld2 + 2 * d2 + hcol + 2 * c)));
    }
    f32x4 sc[T];
    auto load_bias = [&](int t, int q0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[t][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rb, boff + (uint32_t)(q0 + r) * brow, 0, 0));
    };
#pragma unroll
    for (int t = 0; t < T; ++t) load_bias(t, 16 * t);
    put(0);
    __syncthreads();
    for (int s = 0; s < (ONE ? 1 : nseg); ++s) {
      const int q0 = s * Seg::SEG;
      if constexpr (!ONE) fetch(q0 + Seg::SEG);
      const char* imgQ = smem + (s & 1) * 2 * Seg::IMG;
      const char* imgD = imgQ + Seg::IMG;
#pragma unroll
      for (int t = 0; t < T; t += 2) {
        if (live && q0 + 16 * t < len) {  // (uniform; the second tile of a pair may lie beyond: its queries take no part)
          union { uint32_t u[4]; bf16x8 v; } pf, df, pl, sl;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            f32x4 dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS2; ++ks) {
              sc[t + k] = mfma16(row_frag(imgQ, 16 * (t + k) + ql, 4 * ks + g), kf[ks], sc[t + k]);
              dp = mfma16(row_frag(imgD, 16 * (t + k) + ql, 4 * ks + g), vf[ks], dp);
            }
            const f32x4 m = *reinterpret_cast<const f32x4*>(&stats[s & 1][16 * (t + k) + 4 * g]);
            const f32x4 rest = *reinterpret_cast<const f32x4*>(&stats[s & 1][Seg::SEG + 16 * (t + k) + 4 * g]);
            const f32x4 dl = *reinterpret_cast<const f32x4*>(&stats[s & 1][2 * Seg::SEG + 16 * (t + k) + 4 * g]);
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              pr[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t + k][r] - m[r], LOG2E_F, -rest[r]));
              dp[r] = pr[r] * (dp[r] - dl[r]);
            }
            if (q0 + 16 * (t + k) + 16 > len) {  // whatever the bias holds there
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (q0 + 16 * (t + k) + 4 * g + r >= len) pr[r] = dp[r] = 0.f;
            }
            pf.u[2 * k] = pack_bf16x2(pr[0], pr[1]);
            pf.u[2 * k + 1] = pack_bf16x2(pr[2], pr[3]);
            df.u[2 * k] = pack_bf16x2(dp[0], dp[1]);
            df.u[2 * k + 1] = pack_bf16x2(dp[2], dp[3]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              pl.u[2 * k + i] = low_parts(pf.u[2 * k + i], pr[2 * i], pr[2 * i + 1]);
              sl.u[2 * k + i] = low_parts(df.u[2 * k + i], dp[2 * i], dp[2 * i + 1]);
            }
          }
#pragma unroll
          for (int eb = 0; eb < 2 * KS2; ++eb) {
            const bf16x8 gf = lds_tr_pair(imgD, 16 * t + 4 * g + (ql >> 2), 16 * eb + 4 * (ql & 3));
            const bf16x8 qf = lds_tr_pair(imgQ, 16 * t + 4 * g + (ql >> 2), 16 * eb + 4 * (ql & 3));
            dv[eb] = mfma16(gf, pf.v, dv[eb]);
            dk[eb] = mfma16(qf, df.v, dk[eb]);
            dv[eb] = mfma16(gf, pl.v, dv[eb]);
            dk[eb] = mfma16(qf, sl.v, dk[eb]);
          }
        }
        if constexpr (!ONE) {
          load_bias(t, q0 + Seg::SEG + 16 * t);
          load_bias(t + 1, q0 + Seg::SEG + 16 * (t + 1));
        }
      }
      if (!ONE && s + 1 < nseg) {
        put((s + 1) & 1);
        __syncthreads();
      }
    }
  }
  if (key < p.N) {
    if (!ok) {
#pragma unroll
      for (int eb = 0; eb < 2 * KS2; ++eb) dk[eb] = dv[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bf16_t* row = p.dqkv + ((size_t)b * p.N + key) * p.ld + p.d + h * p.hd;
    store_row16<KS2>(row, dk, g, p.hd, 1.0f);
    store_row16<KS2>(row + p.d, dv, g, p.hd, 1.0f);
  }
}

// columns col .. col + 3 of a bias gradient's row; what lies behind column N is the caller's
__device__ __forceinline__ void store_columns(float* row, int col, int N, f32x4 v) {
  if (col + 4 <= N) {
    *reinterpret_cast<f32x4*>(row + col) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (col + i < N) row[col + i] = v[i];
  }
}

// dbias of a tile of 32 W queries x SEG keys of one head, summed over the images of a part
template <int KS>
__global__ __launch_bounds__(256, 2) void bias_attn_db_kernel(const BiasAttnParams p) {
  constexpr int W = 4;
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
    load_bias_t(bias[t], rb, q < p.N ? (uint32_t)(q * p.ldb + 4 * L.half) * 4 : BEYOND, k0 + 32 * t);
    acc[t] = zero16();
  }
  Seg sg;
  bf16x8 qn[KS], dn[KS];
  float mn, restn, deltan;
  auto fetch = [&](int b, bool any) {  // an image's operands, one image ahead (any: or nothing, out of range)
    const int len = any ? length_of(p, b) : 0;
    const uint32_t ld2 = (uint32_t)p.ld * 2, d2 = (uint32_t)p.d * 2, col = (uint32_t)(h * hd + 8 * L.half) * 2;
    const auto rs = rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)len * ld2), rd = rsrc_of(p.d_o + (size_t)b * p.N * p.d, (size_t)len * d2);
    const auto rt = rsrc_of(p.stat + ((size_t)b * p.H + h) * 3 * p.Np, (size_t)p.Np * 12);
    sg.fetch(rs, ld2, ck, rs, ld2, cv, k0, len);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qn[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(q < len, (uint32_t)q * ld2 + col + 32 * ks)));
      dn[ks] = __builtin_bit_cast(bf16x8, load16(rd, only(q < len, (uint32_t)q * d2 + col + 32 * ks)));
    }
    mn = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rt, only(q < p.Np, (uint32_t)q * 4), 0, 0));
    restn = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rt, only(q < p.Np, (uint32_t)(q + p.Np) * 4), 0, 0));
    deltan = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rt, only(q < p.Np, (uint32_t)(q + 2 * p.Np) * 4), 0, 0));
  };
  if (b0 < b1) {
    fetch(b0, true);
    sg.put(smem);
    __syncthreads();
  }
  for (int b = b0; b < b1; ++b) {
    const bool more = b + 1 < b1;
    const int len = length_of(p, b);
    bf16x8 qf[KS], df[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = qn[ks];
      df[ks] = dn[ks];
    }
    const float m = mn, rest = restn, delta = deltan;
    fetch(more ? b + 1 : b, more);
    __builtin_amdgcn_sched_barrier(0);  // (else the loads sink to their use)
    const char* imgK = smem + ((b - b0) & 1) * 2 * Seg::IMG;
    const char* imgV = imgK + Seg::IMG;
    f32x16 sc[T], dp[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      sc[t] = bias[t];
      dp[t] = zero16();
      tile_product<KS>(sc[t], imgK, 32 * t + L.ql, qf, L.half);
      tile_product<KS>(dp[t], imgV, 32 * t + L.ql, df, L.half);
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r] - m, LOG2E_F, -rest)) * (dp[t][r] - delta);
      if (k0 + 32 * t + 32 > len) mask_keys(sc[t], k0 + 32 * t, len, L, 0.f);
      if (q < len) {  // (whatever the bias holds in other rows)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] += sc[t][r];
      }
    }
    if (more) {
      sg.put(smem + ((b - b0 + 1) & 1) * 2 * Seg::IMG);
      __syncthreads();
    }
  }
  if (q < p.N) {
    float* out = p.dbias + (((size_t)part * p.H + h) * p.N + q) * p.lddb;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store_columns(out, k0 + 32 * t + 8 * g + 4 * L.half, p.N, f32x4{acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]});
  }
}

// ------------------------------------------------------------------------------------------ dQ and dbias, short sequences (N <= 16 KT, KT <= 14)
// A workgroup holds all keys of an (image, head) in LDS; a wave owns 16 queries (v_mfma_f32_16x16x32), so that P and dP of ALL keys (8 KT registers)
// stay in registers between delta and dS - no score is computed twice - and the wave's dS, added up over the images, too (4 KT): the
// bias gradient costs 4 additions a tile instead of a kernel that computes dS again.  32 queries a wave would need 512 registers for this.
// Persistent over the images of one head, with two K / V image pairs: the next image's rows are fetched into registers (in groups where they are many) while this one is
// computed, and put into the other pair half an image later; the only barrier is the one between images.  The score tiles are independent
// accumulators: every LDS and MFMA latency is covered by the other tiles of the same wave.

template <int KT, int KS2, bool DB>
__global__ __launch_bounds__(512, 2) void bias_attn_dq_resident_kernel(const BiasAttnParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int KE = KT + KT % 2, IMG = KE * 16 * ROWB, PIECES = KE * 16 * 8 * 2, RES_GROUPS = KT <= 6 ? 1 : KT <= 8 ? 2 : 4;
  constexpr bool AHEAD = KT <= 8;  // the next image's bias ahead too: longer rows leave no registers for them (14 tiles: 93 spills, twice the time)
  const int lane = threadIdx.x & 63, ql = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = xcd_remap(blockIdx.x, gridDim.x);
  int part, h, blk;
  if (p.image_major) {
    blk = t0 % p.blocks;
    h = t0 / p.blocks % p.H;
    part = t0 / p.blocks / p.H;
  } else {
    part = t0 % p.parts;
    blk = t0 / p.parts % p.blocks;
    h = t0 / p.parts / p.blocks;
  }
  const int b0 = (int)((long)p.B * part / p.parts), b1 = (int)((long)p.B * (part + 1) / p.parts);
  const int q = (blk * (int)(blockDim.x >> 6) + wave) * 16 + ql;
  const auto rb = rsrc_of(p.bias + (size_t)h * p.N * p.ldb, (size_t)p.N * p.ldb * 4);
  const uint32_t boff = q < p.N ? (uint32_t)(q * p.ldb + 4 * g) * 4 : BEYOND;
  const uint32_t ld2 = (uint32_t)p.ld * 2, d2 = (uint32_t)p.d * 2, hcol = (uint32_t)(h * p.hd) * 2;

  // the next image's K and V rows: PIECES 16-byte pieces in RES_GROUPS groups ; rows at and beyond its length are out of the descriptor's range (zero),
  // columns at and beyond hd repeat others (they meet zeros of the query fragments, or output rows that are not stored)
  constexpr int LEAST = 64 * (KE <= 8 ? KE - 1 : KE / 2), MAXL = (PIECES / RES_GROUPS + LEAST - 1) / LEAST;  // threads, pieces a thread and group
  u32x4 st[RES_GROUPS][MAXL];  // (the first image's all at once; then a group at a time)
  const int chunks = p.hd / 8;
  auto thread = [] {  // opaque: the offsets below are computed where they are used, 16 of them held over the loop are 16 registers too many
    int i = threadIdx.x;
    if constexpr (RES_GROUPS == 4) asm volatile("" : "+v"(i));
    return i;
  };
  auto fetch = [&](__amdgpu_buffer_rsrc_t rs, int grp) {
    const int i0 = thread();
#pragma unroll
    for (int k = 0; k < MAXL; ++k) {
      const int u = grp * (PIECES / RES_GROUPS) + i0 + k * blockDim.x;
      const int t = (u >> 4), c = (u & 7) < chunks ? (u & 7) : 0;
      const bool in = i0 + k * (int)blockDim.x < PIECES / RES_GROUPS;
      st[grp][k] = load16(rs, in ? (uint32_t)t * ld2 + ((u & 8) ? 2 * d2 : d2) + hcol + 16 * c : OUTSIDE);
    }
  };
  auto put = [&](int grp, int buf) {
    const int i0 = thread();
#pragma unroll
    for (int k = 0; k < MAXL; ++k) {
      const int u = grp * (PIECES / RES_GROUPS) + i0 + k * blockDim.x;
      if (i0 + k * (int)blockDim.x < PIECES / RES_GROUPS)
        *reinterpret_cast<u32x4*>(smem + buf * 2 * IMG + ((u & 8) ? IMG : 0) + at_chunk(u >> 4, u & 7)) = st[grp][k];
    }
  };
  auto image = [&](int b, int len) { return rsrc_of(p.qkv + (size_t)b * p.N * p.ld, (size_t)len * ld2); };
  bf16x8 qf[KS2], df[KS2];
  float lse;
  auto load_queries = [&](int b, int len) {
    const auto rs = image(b, len), rd = rsrc_of(p.d_o + (size_t)b * p.N * p.d, (size_t)len * d2), rl = rsrc_of(p.lse + ((size_t)b * p.H + h) * p.N, (size_t)len * 4);
#pragma unroll
    for (int ks = 0; ks < KS2; ++ks) {
      const int c = 32 * ks + 8 * g;
      qf[ks] = __builtin_bit_cast(bf16x8, load16(rs, only(c < p.hd, (uint32_t)q * ld2 + hcol + 2 * c)));
      df[ks] = __builtin_bit_cast(bf16x8, load16(rd, only(c < p.hd, (uint32_t)q * d2 + hcol + 2 * c)));
    }
    lse = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rl, (uint32_t)q * 4, 0, 0));
  };

  f32x4 acc[DB ? KT : 1];
  if constexpr (DB) {
#pragma unroll
    for (int t = 0; t < KT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int len = length_of(p, b0);
  {
    const auto rs = image(b0, len);
#pragma unroll
    for (int i = 0; i < RES_GROUPS; ++i) fetch(rs, i);
#pragma unroll
    for (int i = 0; i < RES_GROUPS; ++i) put(i, 0);
  }
  load_queries(b0, len);
  f32x4 sc[KT], dp[KT];
  if constexpr (AHEAD) {
#pragma unroll
    for (int t = 0; t < KT; ++t) sc[t] = load4f(rb, boff + 64 * t);
  }
  for (int b = b0; b < b1; ++b) {
    const int buf = (b - b0) & 1, bn = b + 1 < b1 ? b + 1 : b, lenn = b + 1 < b1 ? length_of(p, bn) : 0;  // (behind the last one nothing is in range)
    const auto rn = image(bn, lenn);
    const char* imgK = smem + buf * 2 * IMG;
    const char* imgV = imgK + IMG;
    if constexpr (!AHEAD) {
#pragma unroll
      for (int t = 0; t < KT; ++t) sc[t] = load4f(rb, boff + 64 * t);
    }
    __syncthreads();  // this image's rows are there, and everybody is done with the other pair
    fetch(rn, 0);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      dp[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS2; ++ks) {
        sc[t] = mfma16(row_frag(imgK, 16 * t + ql, 4 * ks + g), qf[ks], sc[t]);
        dp[t] = mfma16(row_frag(imgV, 16 * t + ql, 4 * ks + g), df[ks], dp[t]);
      }
    }
    const float m = or_none(q < len ? lse : -INFINITY);
    const RowReference rf(m);
    if (__any(rf.far)) {
#pragma unroll
      for (int t = 0; t < KT; ++t) sc[t] -= rf.less;
    }
    float d[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], LOG2E_F, -rf.b));
      if (16 * t + 16 > len) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * t + 4 * g + r >= len) sc[t][r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] += sc[t][r];
        d[r] += sc[t][r] * dp[t][r];
      }
    }
    const float sum = quarters_sum((e[0] + e[1]) + (e[2] + e[3]));
    float inv = sum == 0.f ? 0.f : 1.f / sum, rest = rf.rest(sum);
    float delta = quarters_sum((d[0] + d[1]) + (d[2] + d[3])) * inv;
    if (q >= len) {  // whatever the bias holds in such a row
      delta = inv = rest = 0.f;
#pragma unroll
      for (int t = 0; t < KT; ++t) sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (RES_GROUPS >= 2) {
      put(0, buf ^ 1);
      fetch(rn, 1);
    }
    f32x4 dq[2 * KS2];
#pragma unroll
    for (int eb = 0; eb < 2 * KS2; ++eb) dq[eb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KT; t += 2) {
      union { uint32_t u[4]; bf16x8 v; } f, fl;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (t + k == KT) {
          f.u[2] = f.u[3] = fl.u[2] = fl.u[3] = 0;
          break;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[t + k][r] *= dp[t + k][r] - delta;
          if constexpr (DB) acc[t + k][r] = __builtin_fmaf(sc[t + k][r], inv, acc[t + k][r]);
        }
        f.u[2 * k] = pack_bf16x2(sc[t + k][0], sc[t + k][1]);
        f.u[2 * k + 1] = pack_bf16x2(sc[t + k][2], sc[t + k][3]);
        fl.u[2 * k] = low_parts(f.u[2 * k], sc[t + k][0], sc[t + k][1]);
        fl.u[2 * k + 1] = low_parts(f.u[2 * k + 1], sc[t + k][2], sc[t + k][3]);
      }
#pragma unroll
      for (int eb = 0; eb < 2 * KS2; ++eb) {
        const bf16x8 kf = lds_tr_pair(imgK, 16 * t + 4 * g + (ql >> 2), 16 * eb + 4 * (ql & 3));
        dq[eb] = mfma16(kf, f.v, dq[eb]);
        dq[eb] = mfma16(kf, fl.v, dq[eb]);
      }
      if constexpr (RES_GROUPS == 4) {
        if (t == KE / 6 * 2) { put(1, buf ^ 1); fetch(rn, 2); }
        if (t == KE / 6 * 4) { put(2, buf ^ 1); fetch(rn, 3); }
      }
      if constexpr (AHEAD) {  // into registers that have just become free
#pragma unroll
        for (int k = 0; k < 2; ++k) sc[t + k] = load4f(rb, boff + 64 * (t + k));
      }
      if (AHEAD && t == KT / 4 * 2) load_queries(bn, lenn);
    }
    const auto ro = rsrc_of(p.dqkv + (size_t)b * p.N * p.ld, (size_t)p.N * ld2);
    pieces_of_row16<KS2>(dq, g, p.dq_scale * inv, [&](int col, u32x4 v) { store16(ro, only(q < p.N && col < p.hd, (uint32_t)q * ld2 + hcol + 2 * col), v); });
    {  // statistics of the queries, and of the padding up to Np (fewer than three times the rows here) that the dK / dV kernel's tiles read
      const int row = q + g * (int)(blockDim.x >> 6) * 16 * p.blocks;
      const auto rt = rsrc_of(p.stat + ((size_t)b * p.H + h) * 3 * p.Np, (size_t)p.Np * 12);
      auto put_stat = [&](int k, float v) {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rt, only(row < p.Np, (uint32_t)(row + k * p.Np) * 4), 0, 0);
      };
      put_stat(0, g == 0 ? m : INFINITY);
      put_stat(1, g == 0 ? rest : 0.f);
      put_stat(2, g == 0 ? delta : 0.f);
    }
    put(RES_GROUPS - 1, buf ^ 1);
    if constexpr (!AHEAD) load_queries(bn, lenn);
    len = lenn;
  }
  if constexpr (DB) {
    if (q < p.N) {
      float* out = p.dbias + (((size_t)part * p.H + h) * p.N + q) * p.lddb;
#pragma unroll
      for (int t = 0; t < KT; ++t) store_columns(out, 16 * t + 4 * g, p.N, acc[t]);
    }
  }
}

// out = sum of the parts (rows of quads 16-byte columns; out's are ld elements apart): 16 columns a block, 16 strips of parts, fixed order
__global__ __launch_bounds__(256) void bias_attn_parts_kernel(const float* __restrict__ slab, float* __restrict__ out, long n4, int parts, int N, int quads, int ld) {
  __shared__ f32x4 red[16][16];
  const int c = threadIdx.x & 15, strip = threadIdx.x >> 4;
  const long i = (long)blockIdx.x * 16 + c;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < n4) {
#pragma unroll 4
    for (int k = strip; k < parts; k += 16) s += reinterpret_cast<const f32x4*>(slab)[(size_t)k * n4 + i];
  }
  red[strip][c] = s;
  __syncthreads();
  if (strip == 0 && i < n4) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][c];
    const long row = i / quads;
    store_columns(out + (size_t)row * ld, (int)(i - row * quads) * 4, N, s);
  }
}

int padded(int N) { return (N + 63) / 64 * 64; }
int quads_of(int N) { return (N + 3) / 4; }  // of a row of the slab

// Up to 224 tokens the keys of an (image, head) are resident and the bias gradient is part of the dQ kernel: the backward takes 213 us against 302 of the
// streaming kernels at [128 x 12 x 197], 71 / 120 at [2048 x 4 x 49], 87 / 125 at [64 x 8 x 224], 27 / 31 at [2 x 12 x 197]; without a bias gradient 188 /
// 221, 66 / 80, 74 / 88, 20 / 19.  (Beyond, the registers of a wave do not hold a row's P, dP and dS sum.)
constexpr int RESIDENT_N = 224;
bool resident(int N) { return N <= RESIDENT_N; }
constexpr int CUS = 256;  // not the device's or a budget's: the parts set the order of the bias gradient's sum

int clamp_parts(long want, int B) { return (int)(want < 1 ? 1 : want > B ? (B > 0 ? B : 1) : want); }
// waves of the resident kernel: one a 16 queries, two workgroups a sequence beyond eight
int resident_waves(int N) {
  const int nq = (N + 15) / 16;
  return nq > 8 ? (nq + 1) / 2 : nq;
}
int resident_blocks(int N) { return (N + 15) / 16 > 8 ? 2 : 1; }
// parts of the batch, a workgroup each: the persistent kernel's fill the chip once with 8 waves a CU (160 KB of LDS a CU; 12 and 16 waves, more than fit at once,
// take 215 and 216 us against 208 at [1024 x 12 x 49], heads of 64) ...
int resident_parts(int B, int N, int H) {
  const int kt = (N + 31) / 32 * 2, W = resident_waves(N);
  int per_cu = 8 / W;
  if (per_cu > 160 / (8 * kt)) per_cu = 160 / (8 * kt);
  return clamp_parts((long)CUS * (per_cu < 1 ? 1 : per_cu) / ((long)H * resident_blocks(N)), B);
}
// ... the dbias kernel's are about four workgroups a CU
int db_parts(int B, int N, int H) {
  const long tiles = (long)H * ((N + 127) / 128) * ((N + 63) / 64);
  return clamp_parts(4L * CUS / tiles, B);
}
int dbias_parts(int B, int N, int H) { return resident(N) ? resident_parts(B, N, H) : db_parts(B, N, H); }

// All heads of an image in a row where their biases fit an XCD's L2 (4 MB) beside the rows: half of it where heads end inside a cache line of a row, a
// quarter where they are whole lines and less is won.  Against all images of a head in a row, forward and backward: [2048 x 4 x 49], heads of 32,
// 25 and 71 us against 27.5 and 82; [128 x 12 x 197], heads of 48 (1.9 MB), forward 55 / 58; heads of 64: [1024 x 8 x 128] forward 149 / 162, [1024 x 8 x 64]
// backward 184 / 192, but [128 x 12 x 197] (1.9 MB) forward 63.3 / 62.3 and [16 x 16 x 577] (21 MB) 80 / 59
bool many_heads(int N, int H, int hd, int ldb) { return (long)H * N * ldb * 4 <= (hd == 64 ? 1L << 20 : 2L << 20); }

bool size_ok(int B, int N, int H, int hd, int ld, int ldb) {
  if (!(B >= 0 && N > 0 && N <= 32768 && H > 0 && (hd == 16 || hd == 32 || hd == 48 || hd == 64))) return false;
  if (!(ld >= 3L * H * hd && ld % 8 == 0 && ldb >= N && ldb % 4 == 0)) return false;
  // 32-bit offsets inside one image's rows and one head's bias
  if ((long)(N + 128) * ld * 2 >= 0xfff00000L || (long)(N + 128) * ldb * 4 >= 0xfff00000L) return false;
  return (long)B * H * ((N + 31) / 32) <= 0x7fffffffL;
}
bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

#define BIAS_ATTN_LAUNCH(KERNEL, GRID)                                                              \
  do {                                                                                              \
    const dim3 g_((unsigned)(GRID)), t_(256);                                                       \
    switch (head_dim / 16) {                                                                        \
      case 1: hipLaunchKernelGGL((KERNEL<1>), g_, t_, 0, st, p); break;                             \
      case 2: hipLaunchKernelGGL((KERNEL<2>), g_, t_, 0, st, p); break;                             \
      case 3: hipLaunchKernelGGL((KERNEL<3>), g_, t_, 0, st, p); break;                             \
      default: hipLaunchKernelGGL((KERNEL<4>), g_, t_, 0, st, p); break;                            \
    }                                                                                               \
    const hipError_t e_ = hipGetLastError();                                                        \
    if (e_ != hipSuccess) return (int)e_;                                                           \
  } while (0)

template <int KT, int KS2, bool DB>
int launch_resident_k(const BiasAttnParams& p, hipStream_t st) {
  auto kfn = bias_attn_dq_resident_kernel<KT, KS2, DB>;
  SAVIT_LDS_ONCE(kfn);
  hipLaunchKernelGGL(kfn, dim3((unsigned)(p.parts * p.H * p.blocks)), dim3(64 * resident_waves(p.N)), (size_t)4 * (KT + KT % 2) * 16 * ROWB, st, p);
  SAVIT_LAUNCH_RET();
}
template <int KT>
int launch_resident_kt(const BiasAttnParams& p, bool db, hipStream_t st) {
  if (p.hd <= 32) return db ? launch_resident_k<KT, 1, true>(p, st) : launch_resident_k<KT, 1, false>(p, st);
  return db ? launch_resident_k<KT, 2, true>(p, st) : launch_resident_k<KT, 2, false>(p, st);
}
int launch_resident(const BiasAttnParams& p, bool db, hipStream_t st) {
  const int nq = (p.N + 15) / 16;  // rounded to an even number up to eight; beyond, a tile less is 12 registers less, where they are all in use (197 tokens: 110 us with 14, 107 with 13)
  switch (nq) {
    case 1: case 2: return launch_resident_kt<2>(p, db, st);
    case 3: case 4: return launch_resident_kt<4>(p, db, st);
    case 5: case 6: return launch_resident_kt<6>(p, db, st);
    case 7: case 8: return launch_resident_kt<8>(p, db, st);
    case 9: return launch_resident_kt<9>(p, db, st);
    case 10: return launch_resident_kt<10>(p, db, st);
    case 11: return launch_resident_kt<11>(p, db, st);
    case 12: return launch_resident_kt<12>(p, db, st);
    case 13: return launch_resident_kt<13>(p, db, st);
    default: return launch_resident_kt<14>(p, db, st);
  }
}

template <typename F>
int launch_waves(BiasAttnParams p, int W, int rows, F kfn, hipStream_t st) {  // rows: of a wave
  p.blocks = (p.N + rows * W - 1) / (rows * W);
  const long grid = (long)p.B * p.H * p.blocks;
  SAVIT_CHECK_ARG(grid <= 0x7fffffffL);
  hipLaunchKernelGGL(kfn, dim3((unsigned)grid), dim3(64 * W), 0, st, p);
  SAVIT_LAUNCH_RET();
}
// kernels with 16 rows a wave: as many waves as a short sequence has tiles, four at the most
template <typename A, typename B, typename C, typename D>
int launch_sixteen(const BiasAttnParams& p, A one_wave, B two, C segment, D many, hipStream_t st) {
  if (p.N <= 16) return launch_waves(p, 1, 16, one_wave, st);
  if (p.N <= 32) return launch_waves(p, 2, 16, two, st);
  return p.N <= 64 ? launch_waves(p, 4, 16, segment, st) : launch_waves(p, 4, 16, many, st);
}
#define BIAS_ATTN_SIXTEEN(K)                                                                        \
  (p.hd <= 32 ? launch_sixteen(p, K<1, 1, true>, K<2, 1, true>, K<4, 1, true>, K<4, 1, false>, st)  \
              : launch_sixteen(p, K<1, 2, true>, K<2, 2, true>, K<4, 2, true>, K<4, 2, false>, st))
int launch_fwd(BiasAttnParams p, hipStream_t st) {
  // 32 queries a wave where heads are wide, sequences long and the grid is two workgroups a CU or more, else 16 (heads of 64; 32 against 16 a wave:
  // [128 x 12 x 197] 63 against 75 us, [32 x 12 x 197] 20 / 23, [16 x 12 x 197] 14.0 / 13.4, [8 x 16 x 577] 38 / 37, [4 x 16 x 577] 27.5 / 24,
  // [8 x 8 x 1500] 90 / 98, [1 x 8 x 1500] 40 / 28; up to 64 tokens one segment is all there is and 16 are never slower)
  if (p.N > 64 && p.hd > 32 && (long)p.B * p.H * ((p.N + 127) / 128) >= 2L * CUS)
    return p.hd == 48 ? launch_waves(p, 4, 32, bias_attn_fwd_kernel<3>, st) : launch_waves(p, 4, 32, bias_attn_fwd_kernel<4>, st);
  return BIAS_ATTN_SIXTEEN(bias_attn_fwd16_kernel);
}
int launch_dkv(const BiasAttnParams& p, hipStream_t st) { return BIAS_ATTN_SIXTEEN(bias_attn_dkv_kernel); }

}  // namespace

extern "C" int savit_bias_attention_fwd(const void* qkv, const float* bias, const int* lens, void* o, float* lse, int B, int N, int H, int head_dim, int ld_qkv,
                                        int ld_bias, void* stream) {
  SAVIT_CHECK_ARG(qkv && bias && o && lse && size_ok(B, N, H, head_dim, ld_qkv, ld_bias) && o != qkv && aligned16(qkv) && aligned16(bias) && aligned16(o));
  if (B == 0) return SAVIT_OK;
  const long d = (long)H * head_dim, rows = (long)B * N;
  SAVIT_CHECK_ARG(!savit_rows_overlap(o, 2 * d, 2 * d, qkv, 2L * ld_qkv, 6 * d, rows));
  BiasAttnParams p{};
  p.qkv = (const bf16_t*)qkv; p.bias = bias; p.lens = lens; p.o = (bf16_t*)o; p.lse = lse;
  p.B = B; p.N = N; p.H = H; p.ld = ld_qkv; p.d = H * head_dim; p.hd = head_dim; p.ldb = ld_bias;
  p.image_major = many_heads(N, H, head_dim, ld_bias);
  return launch_fwd(p, (hipStream_t)stream);
}

extern "C" long savit_bias_attention_bwd_workspace_bytes(int B, int N, int H, int ld_bias, int want_dbias) {
  if (!(B >= 0 && N > 0 && N <= 32768 && H > 0 && ld_bias >= N)) return 0;
  const int parts = dbias_parts(B, N, H);
  return (long)B * H * 3 * padded(N) * 4 + (want_dbias && parts > 1 ? (long)parts * H * N * quads_of(N) * 16 : 0);
}

extern "C" int savit_bias_attention_bwd(const void* qkv, const float* bias, const int* lens, const void* d_o, const float* lse, void* dqkv, float* dbias, int B,
                                        int N, int H, int head_dim, int ld_qkv, int ld_bias, float dq_scale, void* workspace, long workspace_bytes,
                                        void* stream) {
  SAVIT_CHECK_ARG(qkv && bias && d_o && lse && dqkv && size_ok(B, N, H, head_dim, ld_qkv, ld_bias) && dqkv != qkv && dqkv != d_o && dbias != bias);
  SAVIT_CHECK_ARG(aligned16(qkv) && aligned16(bias) && aligned16(d_o) && aligned16(dqkv) && aligned16(dbias));
  const hipStream_t st = (hipStream_t)stream;
  if (B == 0) return dbias ? (int)SAVIT_EINVAL : SAVIT_OK;  // no image: there is no gradient to write
  const long d = (long)H * head_dim, rows = (long)B * N;  // later kernels read what the first ones would have overwritten
  SAVIT_CHECK_ARG(!savit_rows_overlap(dqkv, 2L * ld_qkv, 6 * d, qkv, 2L * ld_qkv, 6 * d, rows) && !savit_rows_overlap(dqkv, 2L * ld_qkv, 6 * d, d_o, 2 * d, 2 * d, rows));
  SAVIT_CHECK_ARG(!savit_rows_overlap(dbias, 4L * ld_bias, 4L * N, bias, 4L * ld_bias, 4L * N, (long)H * N));
  SAVIT_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= savit_bias_attention_bwd_workspace_bytes(B, N, H, ld_bias, dbias != nullptr));
  BiasAttnParams p{};
  p.qkv = (const bf16_t*)qkv; p.bias = bias; p.lens = lens; p.d_o = (const bf16_t*)d_o; p.lse = const_cast<float*>(lse); p.dqkv = (bf16_t*)dqkv;
  p.B = B; p.N = N; p.H = H; p.ld = ld_qkv; p.d = H * head_dim; p.hd = head_dim; p.ldb = ld_bias; p.dq_scale = dq_scale;
  p.image_major = many_heads(N, H, head_dim, ld_bias);
  p.Np = padded(N);
  p.stat = (float*)workspace;
  const int parts = dbias_parts(B, N, H);
  float* slab = parts == 1 ? dbias : p.stat + (size_t)B * H * 3 * p.Np;
  p.parts = parts;
  p.dbias = slab;
  p.lddb = parts == 1 ? ld_bias : 4 * quads_of(N);
  if (resident(N)) {
    p.blocks = resident_blocks(N);
    const int rr = launch_resident(p, dbias != nullptr, st);
    if (rr != SAVIT_OK) return rr;
  } else {
    const int rq = head_dim <= 32 ? launch_waves(p, 4, 16, bias_attn_dq_kernel<1>, st) : launch_waves(p, 4, 16, bias_attn_dq_kernel<2>, st);
    if (rq != SAVIT_OK) return rq;
  }
  const int rc = launch_dkv(p, st);
  if (rc != SAVIT_OK) return rc;
  if (dbias) {
    if (!resident(N)) {
      p.blocks = (N + 127) / 128;
      p.key_blocks = (N + 63) / 64;
      const long grid = (long)p.parts * H * p.blocks * p.key_blocks;
      SAVIT_CHECK_ARG(grid <= 0x7fffffffL);
      BIAS_ATTN_LAUNCH(bias_attn_db_kernel, grid);
    }
    if (p.parts > 1) {
      const long n4 = (long)H * N * quads_of(N);
      hipLaunchKernelGGL(bias_attn_parts_kernel, dim3((unsigned)((n4 + 15) / 16)), dim3(256), 0, st, slab, dbias, n4, p.parts, N, quads_of(N), ld_bias);
      SAVIT_LAUNCH_RET();
    }
  }
  return SAVIT_OK;
}
