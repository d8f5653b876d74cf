// Learned relative position bias by buckets, and the gradient of its table.
//   bias[h, i, j] = table[index[i, j], h]                 dtable[b, h] += sum of dbias[h, i, j] over the positions of bucket b
// The bucket function is the caller's: index [N, N] holds it for queries i and keys j (grid offsets with extra buckets for a class token,
// distances on a logarithmic scale, ..), shared by all heads and images.
//
// Forward is bound by the writes of the [H, N, ld] bias (the table and the index stay in L2): a thread writes 4 columns of 4 heads as 16-byte pieces.
// Backward is a gather along a list of positions sorted by bucket, laid out once with the index: every table entry is one sum in a fixed order -
// an atomic per position would make the gradient depend on scheduling, and the few buckets that far positions share would serialise.
// A wave takes one bucket's list for 4 heads (the list is read once for them); where lists are long (N^2 / buckets >= 512) each is cut
// into parts whose sums a second launch adds in order.
#include "common.h"
#include "savit.h"

namespace {

constexpr int RB_HEADS = 4;

__global__ __launch_bounds__(256) void relpos_bias_kernel(const float* __restrict__ table, const int* __restrict__ index, float* __restrict__ bias, int N,
                                                          int H, int nb, int ld) {
  const int quads = ld / 4;
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= (long)N * quads) return;
  const int i = (int)(t / quads), j0 = (int)(t - (long)i * quads) * 4;
  const int h0 = blockIdx.y * RB_HEADS;
  const int* row = index + (size_t)i * N;
  int b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = j0 + k < N ? row[j0 + k] : -1;
#pragma unroll
  for (int k4 = 0; k4 < RB_HEADS; ++k4) {
    const int h = h0 + k4;
    if (h < H) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = (unsigned)b[k] < (unsigned)nb ? table[(size_t)b[k] * H + h] : j0 + k < N ? __builtin_nanf("") : 0.f;
      *reinterpret_cast<float4*>(bias + ((size_t)h * N + i) * ld + j0) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

// out: dtable (parts == 1, added to) or the slab [parts][nb * H]
__global__ __launch_bounds__(256) void relpos_grad_kernel(const float* __restrict__ dbias, const int* __restrict__ order, const int* __restrict__ start,
                                                          float* __restrict__ out, int N, int H, int nb, int ld, int parts) {
  const int lane = threadIdx.x & 63;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long)nb * parts) return;
  const int b = (int)(item / parts), part = (int)(item - (long)b * parts);
  const int h0 = blockIdx.y * RB_HEADS, nh = (H - h0) < RB_HEADS ? H - h0 : RB_HEADS;
  const unsigned total = (unsigned)N * (unsigned)N;
  unsigned lo = (unsigned)start[b], hi = (unsigned)start[b + 1];
  if (lo > total) lo = total;  // a bad list is cut, never followed outside
  if (hi > total) hi = total;
  const unsigned len = hi > lo ? hi - lo : 0;
  const unsigned per = (len + parts - 1) / parts;
  const unsigned p0 = lo + (per * part < len ? per * part : len), p1 = lo + (per * (part + 1) < len ? per * (part + 1) : len);
  const float* base[RB_HEADS];
#pragma unroll
  for (int k = 0; k < RB_HEADS; ++k) base[k] = dbias + (size_t)(h0 + (k < nh ? k : 0)) * N * ld;
  float s[RB_HEADS] = {};
#pragma unroll 4
  for (unsigned q = p0 + lane; q < p1; q += 64) {
    const unsigned e = (unsigned)order[q];
    if (e >= total) continue;
    const unsigned i = e / (unsigned)N;
    const size_t at = (size_t)i * ld + (e - i * (unsigned)N);
#pragma unroll
    for (int k = 0; k < RB_HEADS; ++k) s[k] += base[k][at];
  }
#pragma unroll
  for (int k = 0; k < RB_HEADS; ++k) {
    const float v = wave_sum(s[k]);
    if (lane == 0 && k < nh) {
      float* to = out + ((size_t)part * nb + b) * H + h0 + k;
      *to = parts == 1 ? *to + v : v;
    }
  }
}

__global__ __launch_bounds__(256) void relpos_parts_kernel(const float* __restrict__ slab, float* __restrict__ dtable, int n, int parts) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < parts; ++k) s += slab[(size_t)k * n + i];
  dtable[i] += s;
}

bool size_ok(int N, int H, int nb, int ld) { return N > 0 && N <= 32768 && H > 0 && H <= 65536 && nb > 0 && (long)nb * H <= (1L << 30) && ld >= N && ld % 4 == 0; }

int parts_of(int N, int nb) {
  const long p = (long)N * N / ((long)nb * 512);
  return p < 1 ? 1 : p > 128 ? 128 : (int)p;
}

}  // namespace

extern "C" int savit_relpos_bias_fwd(const float* table, const int* index, float* bias, int N, int H, int buckets, int ld_bias, void* stream) {
  SAVIT_CHECK_ARG(table && index && bias && size_ok(N, H, buckets, ld_bias) && ((uintptr_t)bias % 16) == 0);
  const long blocks = ((long)N * (ld_bias / 4) + 255) / 256;
  SAVIT_CHECK_ARG(blocks <= 0x7fffffffL);
  hipLaunchKernelGGL(relpos_bias_kernel, dim3((unsigned)blocks, (unsigned)((H + RB_HEADS - 1) / RB_HEADS)), dim3(256), 0, (hipStream_t)stream, table, index,
                     bias, N, H, buckets, ld_bias);
  SAVIT_LAUNCH_RET();
}

extern "C" long savit_relpos_bias_bwd_workspace_bytes(int N, int H, int buckets) {
  if (!size_ok(N, H, buckets, (N + 3) / 4 * 4)) return 0;
  const int parts = parts_of(N, buckets);
  return parts == 1 ? 0 : (long)parts * buckets * H * 4;
}

extern "C" int savit_relpos_bias_bwd(const float* dbias, const int* order, const int* start, float* dtable, int N, int H, int buckets, int ld_bias,
                                     void* workspace, long workspace_bytes, void* stream) {
  SAVIT_CHECK_ARG(dbias && order && start && dtable && size_ok(N, H, buckets, ld_bias));
  const int parts = parts_of(N, buckets);
  SAVIT_CHECK_ARG(parts == 1 || (workspace && ((uintptr_t)workspace % 4) == 0 && workspace_bytes >= (long)parts * buckets * H * 4));
  const long waves = (long)buckets * parts;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(relpos_grad_kernel, dim3((unsigned)((waves + 3) / 4), (unsigned)((H + RB_HEADS - 1) / RB_HEADS)), dim3(256), 0, st, dbias, order, start,
                     parts == 1 ? dtable : (float*)workspace, N, H, buckets, ld_bias, parts);
  if (parts > 1) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(relpos_parts_kernel, dim3((unsigned)((buckets * H + 255) / 256)), dim3(256), 0, st, (const float*)workspace, dtable, buckets * H, parts);
  }
  SAVIT_LAUNCH_RET();
}
