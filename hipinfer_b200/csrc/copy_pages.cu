// Pages of a cache copied to other pages, in every layer and plane of a cache group at once.
#include "common.cuh"

constexpr int CP_PLANES = 8, CP_PAIRS = 240;      // a launch's arguments are at most 4 KB

struct CopyPlane {
  char* base;              // [layer][page][bytes]
  long layer_stride, page_stride, bytes;
  int layers;
};
struct CopyArgs {          // by value: nothing of a call lives in memory that the next could change
  CopyPlane plane[CP_PLANES];
  int src[CP_PAIRS], dst[CP_PAIRS];
};

// One block has a pair of pages in one layer of one plane.
template <typename V>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  hb_pdl_launch();
  hb_pdl_wait();
  const CopyPlane& p = a.plane[blockIdx.z];
  if ((int)blockIdx.y >= p.layers) return;
  char* layer = p.base + blockIdx.y * p.layer_stride;
  const V* from = (const V*)(layer + a.src[blockIdx.x] * p.page_stride);
  V* to = (V*)(layer + a.dst[blockIdx.x] * p.page_stride);
  for (long i = threadIdx.x; i < p.bytes / (long)sizeof(V); i += 256) to[i] = from[i];
}

// planes: n_planes x (base, layers, layer stride, page stride, bytes of a page), 64-bit each; src, dst: host arrays of n_pairs pages. No page
// is both read and written (the caller has seen to it).
HB_EXPORT int hb_copy_pages(const long* planes, int n_planes, const int* src, const int* dst, int n_pairs, cudaStream_t st) {
  if (n_planes <= 0 || n_pairs <= 0) return 0;
  for (int at = 0; at < n_planes; at += CP_PLANES) {
    CopyArgs a = {};
    const int n = n_planes - at < CP_PLANES ? n_planes - at : CP_PLANES;
    int layers = 0;
    bool wide = true;
    for (int i = 0; i < n; i++) {
      const long* p = planes + 5 * (at + i);
      a.plane[i] = {(char*)p[0], p[2], p[3], p[4], (int)p[1]};
      layers = a.plane[i].layers > layers ? a.plane[i].layers : layers;
      wide = wide && !((p[0] | p[2] | p[3] | p[4]) & 15);
    }
    if (layers > 65535) HB_FAIL("hb_copy_pages: %d layers", layers);
    for (int first = 0; first < n_pairs; first += CP_PAIRS) {
      const int m = n_pairs - first < CP_PAIRS ? n_pairs - first : CP_PAIRS;
      for (int i = 0; i < m; i++) {
        a.src[i] = src[first + i];
        a.dst[i] = dst[first + i];
      }
      if (wide) hb_launch(copy_pages_kernel<uint4>, dim3(m, layers, n), dim3(256), 0, st, a);
      else hb_launch(copy_pages_kernel<uint8_t>, dim3(m, layers, n), dim3(256), 0, st, a);
    }
  }
  HB_CHECK_LAUNCH("hb_copy_pages");
  return 0;
}
