// Learned relative position bias by buckets, and the gradient of its table.
//   bias[h, i, j] = table[index[i, j], h]                 dtable[b, h] += sum of dbias[h, i, j] over the positions of bucket b
// The bucket function is the caller's: index [N, N] holds it for queries i and keys j (grid offsets with extra buckets for a class token,
// distances on a logarithmic scale, ..), shared by all heads and images.
//
// Forward is bound by the writes of the [H, N, ld] bias (the table and the index stay in L2): a thread writes 4 columns of 4 heads as 16-byte pieces.
// Backward is a gather along a list of positions sorted by bucket, laid out once with the index: every table entry is one sum in a fixed order -
// an atomic per position would make the gradient depend on scheduling, and the few buckets that far positions share would serialise.
// A wave takes one bucket's list for 4 heads (the list is read once for them); where lists are long it takes a fixed number of entries instead,
// and a second launch adds the pieces of a bucket.
// Measured: [8 x 1500 x 1500] forward 15 us (72 MB, 4.8 TB/s), table gradient of 32 buckets 23 + 5 us (72 MB read through the list);
// [16 x 577 x 577] 9.6 us (21 MB; bound by the gathers from 2212 buckets), [12 x 197 x 197] 5 us and 9 us.
#include "common.h"
#include "savit.h"

namespace {

constexpr int RB_HEADS = 4;

// A thread takes four columns of four heads; G threads in a row take 4 G heads of the same columns, so that they read one bucket's heads from the same
// cache line and the 64 / G column groups of a wave still store 1 KB / G in a row.
// VEC: H % 4 == 0 and the table 16-byte aligned - a bucket's four heads are one load (four times fewer gathers)
template <bool VEC, int G>
__global__ __launch_bounds__(256) void relpos_bias_kernel(const float* __restrict__ table, const int* __restrict__ index, float* __restrict__ bias, int N,
                                                          int H, int nb, int ld) {
  const unsigned quads = ld / 4, t = blockIdx.x * (256 / G) + threadIdx.x / G;
  const int h0 = (blockIdx.y * G + threadIdx.x % G) * RB_HEADS;
  if (t >= N * quads || h0 >= H) return;
  const int i = (int)(t / quads), j0 = (int)(t - i * quads) * 4;
  const int* row = index + (size_t)i * N;
  int b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = j0 + k < N ? row[j0 + k] : -1;
  float v[4][RB_HEADS];  // [column][head]
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float none = j0 + k < N ? __builtin_nanf("") : 0.f;
    const bool in = (unsigned)b[k] < (unsigned)nb;
    if constexpr (VEC) {
      float4 w = make_float4(none, none, none, none);
      if (in) w = *reinterpret_cast<const float4*>(table + (size_t)b[k] * H + h0);
      v[k][0] = w.x; v[k][1] = w.y; v[k][2] = w.z; v[k][3] = w.w;
    } else {
#pragma unroll
      for (int h = 0; h < RB_HEADS; ++h) v[k][h] = in && h0 + h < H ? table[(size_t)b[k] * H + h0 + h] : none;
    }
  }
#pragma unroll
  for (int h = 0; h < RB_HEADS; ++h)
    if (h0 + h < H) *reinterpret_cast<float4*>(bias + ((size_t)(h0 + h) * N + i) * ld + j0) = make_float4(v[0][h], v[1][h], v[2][h], v[3][h]);
}

// sum of positions order[p0 .. p1) of RB_HEADS heads over a wave; every lane gets the sums
__device__ __forceinline__ void sum_list(const float* __restrict__ dbias, const int* __restrict__ order, unsigned p0, unsigned p1, int N, int ld, int h0, int nh,
                                         unsigned total, float (&out)[RB_HEADS]) {
  const int lane = threadIdx.x & 63;
  const float* base[RB_HEADS];
#pragma unroll
  for (int k = 0; k < RB_HEADS; ++k) base[k] = dbias + (size_t)(h0 + (k < nh ? k : 0)) * N * ld;
  float s[RB_HEADS] = {};
  constexpr int U = 4;  // entries a lane has under way: the list, then all heads' values (a lane without an entry reads position 0 and drops it)
  for (unsigned q = p0 + lane; q < p1; q += 64 * U) {
    unsigned e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = q + 64 * u < p1 ? (unsigned)order[q + 64 * u] : 0xffffffffu;
    float v[U][RB_HEADS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned x = e[u] < total ? e[u] : 0, i = x / (unsigned)N;
      const size_t at = (size_t)i * ld + (x - i * (unsigned)N);
#pragma unroll
      for (int k = 0; k < RB_HEADS; ++k) v[u][k] = base[k][at];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < RB_HEADS; ++k) s[k] += e[u] < total ? v[u][k] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < RB_HEADS; ++k) out[k] = wave_sum(s[k]);
}
// where bucket b's list begins; a bad list is cut, never followed outside
__device__ __forceinline__ unsigned list_at(const int* start, int b, unsigned total) {
  const unsigned v = (unsigned)start[b];
  return v < total ? v : total;
}

// short lists: a wave a bucket
__global__ __launch_bounds__(256) void relpos_grad_kernel(const float* __restrict__ dbias, const int* __restrict__ order, const int* __restrict__ start,
                                                          float* __restrict__ dtable, int N, int H, int nb, int ld) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= nb) return;
  const int h0 = blockIdx.y * RB_HEADS, nh = (H - h0) < RB_HEADS ? H - h0 : RB_HEADS;
  const unsigned total = (unsigned)N * (unsigned)N;
  float s[RB_HEADS];
  sum_list(dbias, order, list_at(start, b, total), list_at(start, b + 1, total), N, ld, h0, nh, total, s);
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < RB_HEADS; ++k)
      if (k < nh) dtable[(size_t)b * H + h0 + k] += s[k];
  }
}

// long lists: a wave RB_CHUNK entries, whatever buckets they belong to; the piece of bucket b in chunk c goes to slab row c + b (every new piece
// is a new chunk, a new bucket or both, so rows are not shared)
constexpr int RB_CHUNK = 256;  // four entries a lane, all under way at once: 23 us at 1500 tokens and 8 heads (longer chunks, a loop of such loads: 36)
__global__ __launch_bounds__(256) void relpos_grad_chunks_kernel(const float* __restrict__ dbias, const int* __restrict__ order, const int* __restrict__ start,
                                                                 float* __restrict__ slab, int N, int H, int nb, int ld, int chunks) {
  const int c = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= chunks) return;
  const int h0 = blockIdx.y * RB_HEADS, nh = (H - h0) < RB_HEADS ? H - h0 : RB_HEADS;
  const unsigned total = (unsigned)N * (unsigned)N;
  const unsigned c0 = (unsigned)c * RB_CHUNK, c1 = c0 + RB_CHUNK < total ? c0 + RB_CHUNK : total;
  constexpr int U = RB_CHUNK / 64;
  float v[U][RB_HEADS];  // all of the chunk, under way while its buckets are looked for (an entry outside reads position 0 and is dropped)
  bool in[U];
  {
    unsigned e[U];
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = c0 + lane + 64 * u < c1 ? (unsigned)order[c0 + lane + 64 * u] : 0xffffffffu;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      in[u] = e[u] < total;
      const unsigned x = in[u] ? e[u] : 0, r = x / (unsigned)N;
      const size_t at = (size_t)r * ld + (x - r * (unsigned)N);
#pragma unroll
      for (int k = 0; k < RB_HEADS; ++k) v[u][k] = dbias[(size_t)(h0 + (k < nh ? k : 0)) * N * ld + at];
    }
  }
  int lo = 0, hi = nb;  // first bucket whose list ends behind c0
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list_at(start, mid + 1, total) > c0) hi = mid;
    else lo = mid + 1;
  }
  for (int b = lo; b < nb; ++b) {
    const unsigned l0 = list_at(start, b, total), l1 = list_at(start, b + 1, total);
    if (l0 >= c1) break;
    const unsigned p0 = l0 > c0 ? l0 : c0, p1 = l1 < c1 ? l1 : c1;
    if (p0 >= p1) continue;
    float s[RB_HEADS] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned q = c0 + (threadIdx.x & 63) + 64 * u;
#pragma unroll
      for (int k = 0; k < RB_HEADS; ++k) s[k] += in[u] && q >= p0 && q < p1 ? v[u][k] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < RB_HEADS; ++k) {
      const float sum = wave_sum(s[k]);
      if ((threadIdx.x & 63) == 0 && k < nh) slab[((size_t)c + b) * H + h0 + k] = sum;
    }
  }
}

// dtable[b, h] += the bucket's pieces: a block an entry, threads and tree in a fixed order
__global__ __launch_bounds__(256) void relpos_pieces_kernel(const float* __restrict__ slab, const int* __restrict__ start, float* __restrict__ dtable, int N,
                                                            int H) {
  __shared__ float red[4];
  const int i = blockIdx.x, b = i / H, h = i - b * H;
  const unsigned total = (unsigned)N * (unsigned)N;
  const unsigned l0 = list_at(start, b, total), l1 = list_at(start, b + 1, total);
  float s = 0.f;
  if (l0 < l1) {
#pragma unroll 4
    for (unsigned c = l0 / RB_CHUNK + threadIdx.x; c <= (l1 - 1) / RB_CHUNK; c += 256) s += slab[((size_t)c + b) * H + h];
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) dtable[i] += (red[0] + red[1]) + (red[2] + red[3]);
}

bool size_ok(int N, int H, int nb, int ld) { return N > 0 && N <= 32768 && H > 0 && H <= 65536 && nb > 0 && (long)nb * H <= (1L << 30) && ld >= N && ld % 4 == 0; }

// lists of 512 positions and more on average are cut into chunks: one wave a bucket leaves the far buckets' lists to a few waves (1500 tokens,
// 32 buckets, 8 heads: 3500 us against the chunks' 22 + 5); below, chunks of many short pieces only serialise
bool long_lists(int N, int nb) { return (long)N * N >= 512L * nb; }
int chunks_of(int N) { return (int)(((long)N * N + RB_CHUNK - 1) / RB_CHUNK); }

}  // namespace

extern "C" int savit_relpos_bias_fwd(const float* table, const int* index, float* bias, int N, int H, int buckets, int ld_bias, void* stream) {
  SAVIT_CHECK_ARG(table && index && bias && size_ok(N, H, buckets, ld_bias) && ((uintptr_t)bias % 16) == 0);
  const int groups = (H + RB_HEADS - 1) / RB_HEADS, G = groups == 1 ? 1 : groups == 2 ? 2 : 4;
  const long blocks = ((long)N * (ld_bias / 4) + 256 / G - 1) / (256 / G);
  SAVIT_CHECK_ARG(blocks <= 0xffffffL);  // (32-bit thread numbers)
  const dim3 grid((unsigned)blocks, (unsigned)((groups + G - 1) / G));
  auto launch = [&](auto kfn) { hipLaunchKernelGGL(kfn, grid, dim3(256), 0, (hipStream_t)stream, table, index, bias, N, H, buckets, ld_bias); };
  if (H % RB_HEADS == 0 && ((uintptr_t)table % 16) == 0)
    G == 1 ? launch(relpos_bias_kernel<true, 1>) : G == 2 ? launch(relpos_bias_kernel<true, 2>) : launch(relpos_bias_kernel<true, 4>);
  else
    G == 1 ? launch(relpos_bias_kernel<false, 1>) : G == 2 ? launch(relpos_bias_kernel<false, 2>) : launch(relpos_bias_kernel<false, 4>);
  SAVIT_LAUNCH_RET();
}

extern "C" long savit_relpos_bias_bwd_workspace_bytes(int N, int H, int buckets) {
  if (!size_ok(N, H, buckets, (N + 3) / 4 * 4) || !long_lists(N, buckets)) return 0;
  return ((long)chunks_of(N) + buckets) * H * 4;
}

extern "C" int savit_relpos_bias_bwd(const float* dbias, const int* order, const int* start, float* dtable, int N, int H, int buckets, int ld_bias,
                                     void* workspace, long workspace_bytes, void* stream) {
  SAVIT_CHECK_ARG(dbias && order && start && dtable && size_ok(N, H, buckets, ld_bias));
  const hipStream_t st = (hipStream_t)stream;
  const unsigned hg = (unsigned)((H + RB_HEADS - 1) / RB_HEADS);
  if (!long_lists(N, buckets)) {
    hipLaunchKernelGGL(relpos_grad_kernel, dim3((unsigned)((buckets + 3) / 4), hg), dim3(256), 0, st, dbias, order, start, dtable, N, H, buckets, ld_bias);
    SAVIT_LAUNCH_RET();
  }
  SAVIT_CHECK_ARG(workspace && ((uintptr_t)workspace % 4) == 0 && workspace_bytes >= savit_relpos_bias_bwd_workspace_bytes(N, H, buckets));
  const int chunks = chunks_of(N);
  hipLaunchKernelGGL(relpos_grad_chunks_kernel, dim3((unsigned)((chunks + 3) / 4), hg), dim3(256), 0, st, dbias, order, start, (float*)workspace, N, H, buckets,
                     ld_bias, chunks);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(relpos_pieces_kernel, dim3((unsigned)(buckets * H)), dim3(256), 0, st, (const float*)workspace, start, dtable, N, H);
  SAVIT_LAUNCH_RET();
}
