// Attention over a paged cache in 8 bits, of any sizes: 32-bit arithmetic on the plain units.
#include "cache8.cuh"

constexpr int C8A_KEYS = 128;      // keys of a pass, one a thread

// One block has a row and a query head: s_j = scale * ks_j * (q . kc_j) of 128 keys, a thread a key; the running maximum m and sum l of
// the softmax; o = sum_j e^(s_j - m) vs_j vc_j, a thread a dimension. A key is seen if it is not behind the row's position, not at or before
// position - window, and its page is there; a row that sees none is 0.
template <typename CT, typename T>
__global__ void __launch_bounds__(C8A_KEYS) cache8_attention_any_kernel(const T* q, long ld_q, const uint8_t* kc, const uint8_t* vc, const float* ks,
                                                                        const float* vs, long n_pages, int Hkv, int page_size, int D, const int* bt,
                                                                        long ld_table, int table_rows, int table_width, const int* row_req,
                                                                        const int* pos, int G, int window, float scale, T* out) {
  __shared__ float q_sh[256], w_sh[C8A_KEYS], red[32];
  __shared__ long base_sh[C8A_KEYS];
  hb_pdl_launch();
  hb_pdl_wait();
  const int t = blockIdx.x, head = blockIdx.y, h = head / G, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = row_req ? row_req[t] : t, p = pos[t];
  const bool known = r >= 0 && r < table_rows;
  for (int d = tid; d < D; d += C8A_KEYS) q_sh[d] = hb_to_float(q[t * ld_q + (long)head * D + d]) * scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  const long last = known ? min((long)p, (long)table_width * page_size - 1) : -1;
  const int lo = window > 0 ? max(0, p - window + 1) : 0;
  for (long j0 = lo; j0 <= last; j0 += C8A_KEYS) {
    const long j = j0 + tid;
    float s = -INFINITY, value_scale = 0.f;
    long base = -1;
    if (j <= last) {
      const long page = bt[r * ld_table + j / page_size];
      const int place = (int)(j % page_size);
      if (page >= 0 && page < n_pages) {
        base = ((page * Hkv + h) * page_size + place) * D;
        const long block = (page * Hkv + h) * c8_blocks(page_size) + place / C8_BLOCK;
        float dot = 0.f;
        for (int d = 0; d < D; d++) dot = fmaf(q_sh[d], CT::value(kc[base + d]), dot);
        s = dot * ks[block];
        value_scale = vs[block];
      }
    }
    float mx = hb_warp_max(s);
    const bool nan = __syncthreads_or(s != s);       // (a maximum loses a NaN; the barrier also ends the pass before)
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    for (int i = 0; i < C8A_KEYS / 32; i++) mx = fmaxf(mx, red[i]);
    const float m_new = fmaxf(m, mx), base_m = m_new == -INFINITY ? 0.f : m_new;
    const float f = expf(m - base_m), w = base < 0 ? 0.f : nan ? NAN : expf(s - base_m);
    m = m_new;
    base_sh[tid] = base;
    w_sh[tid] = base < 0 ? 0.f : w * value_scale;
    l = l * f + hb_block_sum(w, red);
    __syncthreads();
    for (int c = 0; c < 2; c++) {
      const int d = tid + c * C8A_KEYS;
      if (d >= D) break;
      float a = o[c] * f;
      for (int i = 0; i < C8A_KEYS; i++)
        if (base_sh[i] >= 0) a = fmaf(w_sh[i], CT::value(vc[base_sh[i] + d]), a);
      o[c] = a;
    }
  }
  for (int c = 0; c < 2; c++) {
    const int d = tid + c * C8A_KEYS;
    if (d < D) out[((long)t * gridDim.y + head) * D + d] = hb_from_float<T>(l == 0.f ? 0.f : o[c] / l);
  }
}

// q [n_rows][ld_q] with Hkv * G heads of D, out [n_rows][Hkv * G * D]; bt [table_rows][ld_table]; row_req null: row t is request t's.
HB_EXPORT int hb_cache8_attention_any(const void* q, int dt, long ld_q, const void* kc, const void* vc, const float* ks, const float* vs, int ct,
                                      long n_pages, int Hkv, int page_size, int D, const int* bt, long ld_table, int table_rows, int table_width,
                                      const int* row_req, const int* pos, int n_rows, int G, int window, float scale, void* out, cudaStream_t st) {
  if (n_rows <= 0) return 0;
  if (Hkv < 1 || G < 1 || (long)Hkv * G > 65535 || page_size < 1 || D < 1 || D > 256)
    HB_FAIL("hb_cache8_attention_any: %d kv heads of %d for %d heads each, pages of %d", Hkv, D, G, page_size);
  C8_DISPATCH(ct, "hb_cache8_attention_any", HB_DISPATCH_1(dt, "hb_cache8_attention_any",
      hb_launch(cache8_attention_any_kernel<CT, TA>, dim3(n_rows, Hkv * G), dim3(C8A_KEYS), 0, st, (const TA*)q, ld_q, (const uint8_t*)kc,
                (const uint8_t*)vc, ks, vs, n_pages, Hkv, page_size, D, bt, ld_table, table_rows, table_width, row_req, pos, G, window, scale,
                (TA*)out)));
  HB_CHECK_LAUNCH("hb_cache8_attention_any");
  return 0;
}
