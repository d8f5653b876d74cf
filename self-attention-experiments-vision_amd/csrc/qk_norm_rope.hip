// Per-head normalisation of queries and keys with the position rotation in the same pass, forward and backward.
//
// A row of the packed buffer holds H query heads, Hk key heads and Hk value heads of hd columns.  Per (row, head) of the first two:
//   n = (x - c mean x) / sqrt(mean (x - c mean x)^2 + eps)     c = 1: LayerNorm statistics, 0: root mean square
//   y = s R(p) (w . n)                                          s = q_scale for queries, 1 for keys
// R(p) turns hd / 2 pairs by the angles whose cosine | sine are row p of the table; a pair is (e, e + hd/2), or (2e, 2e+1) when interleaved.
//   backward, with g = s R(p)^T dy and h = g . w:   dw += sum g . n ;   dx = r (h - c mean h - n mean(h . n)),   r = 1 / sqrt(..)
//
// Bound by HBM: forward reads and writes a row once, backward reads the cotangent row and the saved queries and keys and writes a row;
// statistics are recomputed from x, which is cheaper than to store and load them.  All arithmetic is in fp32, one rounding at the store.
// Measured, bf16: [128 x 197 rows, 3 x 12 heads of 64] forward 48 us (232 MB: 4.8 TB/s, a large copy reaches 5.0), backward 71 us (310 MB, 4.4 TB/s) and
// 5 us for the weights' sums; [16384 rows, 3 x 8 heads of 48] 19 us (75 MB, 4.0 TB/s); 4 rows: one launch.
//
// Layout: G = 1..16 lanes per head, each with 8 columns of the head's lower half and the 8 columns hd/2 above them, so that both
// kinds of pairs lie in one lane and a reduction takes log2 G lane exchanges.  A group of G lanes owns a fixed chunk of HS heads (backward: one) and walks over rows:
// its weights stay in registers (in backward its weight gradients too), the table row is fetched once for HS heads, and neighbouring
// groups read neighbouring chunks of the same row.
#include "common.h"
#include "savit.h"

namespace {

struct QknParams {
  const void* x;       // raw rows (forward input, saved for backward)
  const void* g;       // backward: cotangent rows
  void* y;             // forward: output rows; backward: gradient rows
  const float *wq, *wk;  // query, key weights [hd]
  const float* table;  // [T, hd] cosines | sines; nullptr: no rotation
  const int* pos;      // [rows] or nullptr: row % N
  float* slab;         // backward: [gridDim.x][2 * hd] partial weight gradients
  float *dwq, *dwk;    // backward, one block: added to directly
  long ldx, ldg, ldy;
  int rows, N, H, Hk, hd, T;
  int nq, nk, nv;      // chunks of HS heads in each section (nv = 0: values stay where they are)
  float eps, q_scale;
  int center, inter;
};

template <typename T>
struct Vec8;  // 8 consecutive elements
template <>
struct Vec8<bf16_t> {
  uint4 r;
  __device__ __forceinline__ void load(const bf16_t* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(bf16_t* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    r = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
};

// sum over the G lanes of a group (every lane gets it)
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v += dpp_mov<0xB1>(v);   // quad_perm [1,0,3,2]
  if constexpr (G >= 4) v += dpp_mov<0x4E>(v);   // quad_perm [2,3,0,1]
  if constexpr (G >= 8) v += dpp_mov<0x141>(v);  // row_half_mirror: the other quad (quads are uniform by now)
  if constexpr (G >= 16) v += dpp_mov<0x140>(v); // row_mirror: the other half row
  return v;
}

// cosines and sines of this lane's 8 pairs at row p of the table; a position outside the table poisons the row instead of reading there
__device__ __forceinline__ void load_angles(const QknParams& p, int row, int l, float (&cs)[8], float (&sn)[8]) {
  const int at = p.pos ? p.pos[row] : (int)((uint32_t)row % (uint32_t)p.N);
  if ((uint32_t)at >= (uint32_t)p.T) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = sn[i] = __builtin_nanf("");
    return;
  }
  const float* t = p.table + (size_t)at * p.hd;
  // (e, e + hd/2): pairs 8l .. 8l+7.  (2e, 2e+1): pairs 4l .. 4l+3 of the lower half and hd/4 + 4l .. of the upper one
  const int e0 = p.inter ? 4 * l : 8 * l, e1 = p.inter ? p.hd / 4 + 4 * l : 8 * l + 4;
  const float4 c0 = *reinterpret_cast<const float4*>(t + e0), c1 = *reinterpret_cast<const float4*>(t + e1);
  const float4 s0 = *reinterpret_cast<const float4*>(t + p.hd / 2 + e0), s1 = *reinterpret_cast<const float4*>(t + p.hd / 2 + e1);
  cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
  sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
}

// turns this lane's pairs by the angles (SIGN = 1) or back (SIGN = -1): a = lower columns, b = upper columns
template <int SIGN>
__device__ __forceinline__ void rotate(float (&a)[8], float (&b)[8], const float (&cs)[8], const float (&sn)[8], bool inter) {
  if (inter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float s0 = SIGN * sn[i], s1 = SIGN * sn[4 + i];
      const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
      a[2 * i] = a0 * cs[i] - a1 * s0;
      a[2 * i + 1] = a0 * s0 + a1 * cs[i];
      b[2 * i] = b0 * cs[4 + i] - b1 * s1;
      b[2 * i + 1] = b0 * s1 + b1 * cs[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = SIGN * sn[i], x = a[i], z = b[i];
      a[i] = x * cs[i] - z * s;
      b[i] = x * s + z * cs[i];
    }
  }
}

// the group's chunk of heads: section (0 queries, 1 keys, 2 values), first column, heads
template <int HS>
__device__ __forceinline__ void chunk_of(const QknParams& p, int c, int& sec, int& col0, int& heads) {
  int h0, n;
  if (c < p.nq) { sec = 0; h0 = c * HS; n = p.H; col0 = h0 * p.hd; }
  else if (c < p.nq + p.nk) { sec = 1; h0 = (c - p.nq) * HS; n = p.Hk; col0 = (p.H + h0) * p.hd; }
  else { sec = 2; h0 = (c - p.nq - p.nk) * HS; n = p.Hk; col0 = (p.H + p.Hk + h0) * p.hd; }
  heads = (n - h0) < HS ? n - h0 : HS;
}

template <typename T, int G, int HS>
__global__ __launch_bounds__(256) void qkn_fwd_kernel(const QknParams p) {
  const int l = threadIdx.x & (G - 1);
  const int groups = gridDim.x * (256 / G);
  const int chunks = p.nq + p.nk + p.nv;
  const int step = groups / chunks;
  const int grp = blockIdx.x * (256 / G) + threadIdx.x / G;
  if (grp >= step * chunks) return;
  int sec, col0, heads;
  chunk_of<HS>(p, grp % chunks, sec, col0, heads);
  const bool on = 16 * l < p.hd;  // hd / 16 lanes of the G have columns
  const int lo = col0 + 8 * l, hi = lo + p.hd / 2;
  const float inv = 1.0f / (float)p.hd;
  float wa[8], wb[8];
  if (sec < 2 && on) {
    const float sc = sec == 0 ? p.q_scale : 1.0f;
    const float* w = sec == 0 ? p.wq : p.wk;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wa[i] = w[8 * l + i] * sc;
      wb[i] = w[p.hd / 2 + 8 * l + i] * sc;
    }
  }
  for (int row = grp / chunks; row < p.rows; row += step) {
    const T* x = reinterpret_cast<const T*>(p.x) + (size_t)row * p.ldx;
    T* y = reinterpret_cast<T*>(p.y) + (size_t)row * p.ldy;
    Vec8<T> va[HS], vb[HS];
#pragma unroll
    for (int h = 0; h < HS; ++h)
      if (on && h < heads) {
        va[h].load(x + lo + h * p.hd);
        vb[h].load(x + hi + h * p.hd);
      }
    float cs[8], sn[8];
    if (sec < 2 && p.table && on) load_angles(p, row, l, cs, sn);
#pragma unroll
    for (int h = 0; h < HS; ++h) {
      if (h >= heads) break;
      if (sec < 2) {
        float a[8], b[8];
        if (on) {
          va[h].get(a);
          vb[h].get(b);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
        }
        if (p.center) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) s += a[i] + b[i];
          const float mean = group_sum<G>(s) * inv;
          if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              a[i] -= mean;
              b[i] -= mean;
            }
          }
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
        const float r = rsqrtf(group_sum<G>(ss) * inv + p.eps);
        if (on) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            a[i] = a[i] * r * wa[i];
            b[i] = b[i] * r * wb[i];
          }
          if (p.table) rotate<1>(a, b, cs, sn, p.inter);
          va[h].set(a);
          vb[h].set(b);
        }
      }
      if (on) {
        va[h].store(y + lo + h * p.hd);
        vb[h].store(y + hi + h * p.hd);
      }
    }
  }
}

constexpr int QKN_BWD_THREADS = 256;

template <typename T, int G>
__global__ __launch_bounds__(QKN_BWD_THREADS, sizeof(T) == 2 ? 4 : 3) void qkn_bwd_kernel(const QknParams p) {
  constexpr int GPB = QKN_BWD_THREADS / G;
  __shared__ float red[QKN_BWD_THREADS * 16];
  const int l = threadIdx.x & (G - 1);
  const int chunks = p.nq + p.nk + p.nv;
  const int step = (int)gridDim.x * GPB / chunks;
  const int grp = blockIdx.x * GPB + threadIdx.x / G;
  const bool on = 16 * l < p.hd;
  const float inv = 1.0f / (float)p.hd;
  float da[8], db[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.f;
  if (grp < step * chunks) {
    int sec, col0, heads;
    chunk_of<1>(p, grp % chunks, sec, col0, heads);
    const int lo = col0 + 8 * l, hi = lo + p.hd / 2;
    float wa[8], wb[8];
    const float sc = sec == 0 ? p.q_scale : 1.0f;
    if (sec < 2 && on) {
      const float* w = sec == 0 ? p.wq : p.wk;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        wa[i] = w[8 * l + i];
        wb[i] = w[p.hd / 2 + 8 * l + i];
      }
    }
    for (int row = grp / chunks; row < p.rows; row += step) {
      const T* x = reinterpret_cast<const T*>(p.x) + (size_t)row * p.ldx;
      const T* g = reinterpret_cast<const T*>(p.g) + (size_t)row * p.ldg;
      T* y = reinterpret_cast<T*>(p.y) + (size_t)row * p.ldy;
      Vec8<T> ga, gb, va, vb;
      if (on) {
        ga.load(g + lo);
        gb.load(g + hi);
        if (sec < 2) {
          va.load(x + lo);
          vb.load(x + hi);
        }
      }
      float cs[8], sn[8];
      if (sec < 2 && p.table && on) load_angles(p, row, l, cs, sn);
      if (sec < 2) {
        float a[8], b[8], u[8], v[8];
        if (on) {
          va.get(a);
          vb.get(b);
          ga.get(u);
          gb.get(v);
          if (p.table) rotate<-1>(u, v, cs, sn, p.inter);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) a[i] = b[i] = u[i] = v[i] = 0.f;
        }
        if (p.center) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) s += a[i] + b[i];
          const float mean = group_sum<G>(s) * inv;
          if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              a[i] -= mean;
              b[i] -= mean;
            }
          }
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
        const float r = rsqrtf(group_sum<G>(ss) * inv + p.eps);
        float hn = 0.f, hs = 0.f;
        if (on) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            a[i] *= r;
            b[i] *= r;
            u[i] *= sc;
            v[i] *= sc;
            da[i] += u[i] * a[i];
            db[i] += v[i] * b[i];
            u[i] *= wa[i];
            v[i] *= wb[i];
            hn += u[i] * a[i] + v[i] * b[i];
            hs += u[i] + v[i];
          }
        }
        hn = group_sum<G>(hn) * inv;
        hs = p.center ? group_sum<G>(hs) * inv : 0.f;
        if (on) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u[i] = r * (u[i] - hs - a[i] * hn);
            v[i] = r * (v[i] - hs - b[i] * hn);
          }
          ga.set(u);
          gb.set(v);
        }
      }
      if (on) {
        ga.store(y + lo);
        gb.store(y + hi);
      }
    }
  }
  // weight gradients of the block: groups in a fixed order, so that the sums repeat bit by bit
  float* mine = red + (threadIdx.x / G) * (16 * G);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mine[8 * l + i] = da[i];
    mine[8 * G + 8 * l + i] = db[i];
  }
  __syncthreads();
  const int cols = 2 * p.hd, parts = cols < QKN_BWD_THREADS ? QKN_BWD_THREADS / cols : 1;
  float s[2] = {0.f, 0.f};  // 512 columns at the most
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int item = threadIdx.x + k * QKN_BWD_THREADS;
    const int col = item % cols, part = item / cols;
    if (part < parts) {
      const int sec = col / p.hd, e = col - sec * p.hd;
      const int at = e < p.hd / 2 ? e : 8 * G + e - p.hd / 2;
      const int c_lo = sec == 0 ? 0 : p.nq, c_hi = sec == 0 ? p.nq : p.nq + p.nk;
      int c = (int)(((unsigned)blockIdx.x * GPB + part) % (unsigned)chunks);
      const int c_step = parts % chunks;
      for (int g = part; g < GPB; g += parts) {
        if (c >= c_lo && c < c_hi) s[k] += red[g * 16 * G + at];
        c += c_step;
        if (c >= chunks) c -= chunks;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if ((int)threadIdx.x + k * QKN_BWD_THREADS < cols * parts) red[threadIdx.x + k * QKN_BWD_THREADS] = s[k];
  __syncthreads();
  for (int col = threadIdx.x; col < cols; col += QKN_BWD_THREADS) {
    float sum = red[col];
    for (int k = 1; k < parts; ++k) sum += red[k * cols + col];
    if (gridDim.x == 1) {
      const int sec = col / p.hd;
      (sec == 0 ? p.dwq : p.dwk)[col - sec * p.hd] += sum;
    } else {
      p.slab[(size_t)blockIdx.x * cols + col] = sum;
    }
  }
}

// dw += column sums of the slab: 16 columns a block, 64 strips of rows, fixed order
__global__ __launch_bounds__(1024) void qkn_dw_kernel(const float* __restrict__ slab, int rows, int hd, float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float s = 0.f;
#pragma unroll 4
  for (int r = r0; r < rows; r += 64) s += slab[(size_t)r * (2 * hd) + col];
  red[r0][c] = s;
  __syncthreads();
  if (threadIdx.x < 64) {  // four partial sums a column
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[r0 + 4 * k][c];
    red[r0][c] = s;
  }
  __syncthreads();
  if (r0 == 0) {
    float* dw = col < hd ? dwq + col : dwk + col - hd;
    *dw += (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
  }
}

int lanes_of(int hd) {
  int g = 1;
  while (16 * g < hd) g *= 2;
  return g;
}

// heads a group takes at a time in forward: HS amortises the table row and keeps 2 HS 16-byte loads of a lane in flight; one where
// that leaves too few groups to fill the chip, and in backward (four times the operands a head: more waves beat wider chunks, 71 us against 81)
template <int HS>
int chunks_of(int H, int Hk, bool values, QknParams* p) {
  const int nq = (H + HS - 1) / HS, nk = (Hk + HS - 1) / HS;
  if (p) { p->nq = nq; p->nk = nk; p->nv = values ? nk : 0; }
  return nq + nk + (values ? nk : 0);
}
bool wide_chunks(long rows, int H, int Hk, int G) { return rows * (H + 2 * Hk) / 4 * G >= 256L * 1024; }

constexpr int QKN_BWD_BLOCKS = 1024;  // four per CU

bool geometry_ok(int rows, int N, int H, int Hk, int hd) {
  return rows >= 0 && rows <= (1 << 30) && N > 0 && H > 0 && Hk > 0 && H <= 4096 && Hk <= 4096 && hd >= 16 && hd <= 256 && hd % 16 == 0;
}
bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

template <typename T, int G, int HS>
int launch_fwd(QknParams& p, bool values, hipStream_t st) {
  const int chunks = chunks_of<HS>(p.H, p.Hk, values, &p);
  const long want = ((long)p.rows * chunks + 256 / G - 1) / (256 / G);
  const long least = (chunks + 256 / G - 1) / (256 / G);
  long blocks = want < 4096 ? want : 4096;
  if (blocks < least) blocks = least;
  hipLaunchKernelGGL((qkn_fwd_kernel<T, G, HS>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  SAVIT_LAUNCH_RET();
}
template <typename T, int G>
int launch_bwd(QknParams& p, bool values, long ws_bytes, hipStream_t st) {
  constexpr int GPB = QKN_BWD_THREADS / G;
  const int chunks = chunks_of<1>(p.H, p.Hk, values, &p);
  const long want = ((long)p.rows * chunks + GPB - 1) / GPB;
  const long least = (chunks + GPB - 1) / GPB;
  long blocks = want < QKN_BWD_BLOCKS ? want : QKN_BWD_BLOCKS;
  if (blocks < least) blocks = least;
  SAVIT_CHECK_ARG(blocks == 1 || (p.slab && ws_bytes >= blocks * 2 * p.hd * 4));
  hipLaunchKernelGGL((qkn_bwd_kernel<T, G>), dim3((unsigned)blocks), dim3(QKN_BWD_THREADS), 0, st, p);
  if (blocks > 1) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(qkn_dw_kernel, dim3((unsigned)(2 * p.hd / 16)), dim3(1024), 0, st, p.slab, (int)blocks, p.hd, p.dwq, p.dwk);
  }
  SAVIT_LAUNCH_RET();
}

}  // namespace

extern "C" int savit_qk_norm_rope_fwd(const void* qkv, long ld, const float* wq, const float* wk, const float* table, int table_rows, const int* positions,
                                      void* out, long ld_out, int rows, int N, int H, int Hk, int head_dim, int is_bf16, float eps, float q_scale,
                                      int center, int interleaved, void* stream) {
  SAVIT_CHECK_ARG(qkv && wq && wk && out && geometry_ok(rows, N, H, Hk, head_dim) && eps >= 0.f);
  const long cols = (long)(H + 2 * Hk) * head_dim;
  const int q16 = is_bf16 ? 8 : 4;
  SAVIT_CHECK_ARG(ld >= cols && ld_out >= cols && ld % q16 == 0 && ld_out % q16 == 0 && aligned16(qkv) && aligned16(out) && aligned16(table));
  SAVIT_CHECK_ARG(table == nullptr || table_rows >= (positions ? 1 : (rows < N ? rows : N)));
  const int esz = is_bf16 ? 2 : 4;
  SAVIT_CHECK_ARG(out == qkv ? ld == ld_out : !savit_rows_overlap(out, ld_out * esz, cols * esz, qkv, ld * esz, cols * esz, rows));
  if (rows == 0) return SAVIT_OK;
  QknParams p{};
  p.x = qkv; p.y = out; p.wq = wq; p.wk = wk; p.table = table; p.pos = positions;
  p.ldx = ld; p.ldy = ld_out; p.rows = rows; p.N = N; p.H = H; p.Hk = Hk; p.hd = head_dim; p.T = table_rows;
  p.eps = eps; p.q_scale = q_scale; p.center = center; p.inter = interleaved;
  const bool values = out != qkv;
  const int G = lanes_of(head_dim);
  const bool wide = wide_chunks(rows, H, Hk, G);
#define QKN_FWD(GV)                                                                                                                     \
  case GV:                                                                                                                              \
    return is_bf16 ? (wide ? launch_fwd<bf16_t, GV, 4>(p, values, (hipStream_t)stream) : launch_fwd<bf16_t, GV, 1>(p, values, (hipStream_t)stream)) \
                   : (wide ? launch_fwd<float, GV, 2>(p, values, (hipStream_t)stream) : launch_fwd<float, GV, 1>(p, values, (hipStream_t)stream));
  switch (G) {
    QKN_FWD(1)
    QKN_FWD(2)
    QKN_FWD(4)
    QKN_FWD(8)
    QKN_FWD(16)
  }
  return SAVIT_EINVAL;
}

extern "C" long savit_qk_norm_rope_bwd_workspace_bytes(int H, int Hk, int head_dim) {
  if (!geometry_ok(1, 1, H, Hk, head_dim)) return 0;
  const int G = lanes_of(head_dim), GPB = QKN_BWD_THREADS / G;
  const long least = ((long)H + 2 * Hk + GPB - 1) / GPB;
  return (least > QKN_BWD_BLOCKS ? least : QKN_BWD_BLOCKS) * 2 * head_dim * 4;
}

extern "C" int savit_qk_norm_rope_bwd(const void* dqkv, long ld_dqkv, const void* qkv, long ld, const float* wq, const float* wk, const float* table,
                                      int table_rows, const int* positions, void* out, long ld_out, float* dwq, float* dwk, int rows, int N, int H, int Hk,
                                      int head_dim, int is_bf16, float eps, float q_scale, int center, int interleaved, void* workspace,
                                      long workspace_bytes, void* stream) {
  SAVIT_CHECK_ARG(dqkv && qkv && wq && wk && out && dwq && dwk && geometry_ok(rows, N, H, Hk, head_dim) && eps >= 0.f && out != qkv);
  SAVIT_CHECK_ARG((uintptr_t)dwq >= (uintptr_t)(dwk + head_dim) || (uintptr_t)dwk >= (uintptr_t)(dwq + head_dim));  // each is added to by its own blocks
  const long cols = (long)(H + 2 * Hk) * head_dim;
  const int q16 = is_bf16 ? 8 : 4;
  SAVIT_CHECK_ARG(ld >= cols && ld_out >= cols && ld_dqkv >= cols && ld % q16 == 0 && ld_out % q16 == 0 && ld_dqkv % q16 == 0);
  SAVIT_CHECK_ARG(aligned16(qkv) && aligned16(out) && aligned16(dqkv) && aligned16(table) && ((uintptr_t)workspace % 4) == 0);
  SAVIT_CHECK_ARG(table == nullptr || table_rows >= (positions ? 1 : (rows < N ? rows : N)));
  const int esz = is_bf16 ? 2 : 4;
  SAVIT_CHECK_ARG(out == dqkv ? ld_dqkv == ld_out : !savit_rows_overlap(out, ld_out * esz, cols * esz, dqkv, ld_dqkv * esz, cols * esz, rows));
  SAVIT_CHECK_ARG(!savit_rows_overlap(out, ld_out * esz, cols * esz, qkv, ld * esz, (long)(H + Hk) * head_dim * esz, rows));  // (its values are not read)
  if (rows == 0) return SAVIT_OK;
  QknParams p{};
  p.x = qkv; p.g = dqkv; p.y = out; p.wq = wq; p.wk = wk; p.table = table; p.pos = positions;
  p.slab = (float*)workspace; p.dwq = dwq; p.dwk = dwk;
  p.ldx = ld; p.ldg = ld_dqkv; p.ldy = ld_out; p.rows = rows; p.N = N; p.H = H; p.Hk = Hk; p.hd = head_dim; p.T = table_rows;
  p.eps = eps; p.q_scale = q_scale; p.center = center; p.inter = interleaved;
  const bool values = out != dqkv;
  const int G = lanes_of(head_dim);
#define QKN_BWD(GV)                                                                                        \
  case GV:                                                                                                 \
    return is_bf16 ? launch_bwd<bf16_t, GV>(p, values, workspace_bytes, (hipStream_t)stream)             \
                   : launch_bwd<float, GV>(p, values, workspace_bytes, (hipStream_t)stream);
  switch (G) {
    QKN_BWD(1)
    QKN_BWD(2)
    QKN_BWD(4)
    QKN_BWD(8)
    QKN_BWD(16)
  }
  return SAVIT_EINVAL;
}
