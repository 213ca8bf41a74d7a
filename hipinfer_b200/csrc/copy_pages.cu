// Pages of a cache copied to other pages, in every layer and plane of a cache group at once.
#include "common.cuh"

constexpr int CP_PLANES = 8, CP_PAIRS = 960, CP_THREADS = 256, CP_AHEAD = 4;      // a launch's arguments are at most 32 KB

struct CopyPlane {
  char* base;              // [layer][page][bytes]
  long layer_stride, page_stride, bytes;
  int layers, width;       // bytes that are copied at a time: 16, 4 or 1
};
struct CopyArgs {          // by value: nothing of a call lives in memory that the next could change
  CopyPlane plane[CP_PLANES];
  int n_planes;
  int src[CP_PAIRS], dst[CP_PAIRS];
};

template <typename V> __device__ __forceinline__ void copy_page(const char* src, char* dst, long bytes) {
  const V* from = (const V*)src;
  V* to = (V*)dst;
  const long n = bytes / (long)sizeof(V);
  for (long j = threadIdx.x; j < n; j += CP_AHEAD * CP_THREADS) {
    V x[CP_AHEAD];
#pragma unroll
    for (int k = 0; k < CP_AHEAD; k++)
      if (j + k * CP_THREADS < n) x[k] = from[j + k * CP_THREADS];
#pragma unroll
    for (int k = 0; k < CP_AHEAD; k++)
      if (j + k * CP_THREADS < n) to[j + k * CP_THREADS] = x[k];
  }
}

// One block has a pair of pages in one layer, in all planes. A thread asks for four of its vectors before it writes the first. Each plane goes by as many bytes at a
// time as its pages and addresses are multiples of: the scales of two heads are 8 bytes
// a page, and with one width for all planes the codes went byte by byte beside them (500 pages of 32 layers of 2 heads of 128 in 8 bits 92 us, 59 now).
// Bound by bandwidth: 500 pages of 32 layers of 8 heads of 128 in 8 bits, 1.05 GB moved, 162 us, 99 % of a copy's rate; 8 pages of 16 layers of 8 heads
// of 64 in 16 bits, 3.6 us, a launch's latency.
__global__ void __launch_bounds__(CP_THREADS) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  hb_pdl_launch();
  hb_pdl_wait();
  const long src = a.src[blockIdx.x], dst = a.dst[blockIdx.x];
  for (int i = 0; i < a.n_planes; i++) {
    const CopyPlane& p = a.plane[i];
    if ((int)blockIdx.y >= p.layers) continue;
    char* layer = p.base + blockIdx.y * p.layer_stride;
    const char* from = layer + src * p.page_stride;
    char* to = layer + dst * p.page_stride;
    if (p.width == 16) copy_page<uint4>(from, to, p.bytes);
    else if (p.width == 4) copy_page<uint32_t>(from, to, p.bytes);
    else copy_page<uint8_t>(from, to, p.bytes);
  }
}

// planes: n_planes x (base, layers, layer stride, page stride, bytes of a page), 64-bit each; src, dst: host arrays of n_pairs pages. No page
// is both read and written (the caller has seen to it).
HB_EXPORT int hb_copy_pages(const long* planes, int n_planes, const int* src, const int* dst, int n_pairs, cudaStream_t st) {
  if (n_planes <= 0 || n_pairs <= 0) return 0;
  for (int at = 0; at < n_planes; at += CP_PLANES) {
    CopyArgs a;
    a.n_planes = n_planes - at < CP_PLANES ? n_planes - at : CP_PLANES;
    int layers = 0;
    for (int i = 0; i < a.n_planes; i++) {
      const long* p = planes + 5 * (at + i);
      const long odd = p[0] | p[2] | p[3] | p[4];
      a.plane[i] = {(char*)p[0], p[2], p[3], p[4], (int)p[1], odd & 3 ? 1 : odd & 15 ? 4 : 16};
      layers = a.plane[i].layers > layers ? a.plane[i].layers : layers;
    }
    if (layers > 65535) HB_FAIL("hb_copy_pages: %d layers", layers);
    for (int first = 0; first < n_pairs; first += CP_PAIRS) {
      const int m = n_pairs - first < CP_PAIRS ? n_pairs - first : CP_PAIRS;
      for (int i = 0; i < m; i++) {
        a.src[i] = src[first + i];
        a.dst[i] = dst[first + i];
      }
      hb_launch(copy_pages_kernel, dim3(m, layers), dim3(CP_THREADS), 0, st, a);
    }
  }
  HB_CHECK_LAUNCH("hb_copy_pages");
  return 0;
}
