// Attention over a paged cache in 8 bits, of any sizes: 32-bit arithmetic on the plain units.
#include "cache8.cuh"

constexpr int C8A_KEYS = 128;      // keys of a pass, one a thread

// One block has a row and a query head: s_j = scale * ks_j * (q . kc_j) of 128 keys, a thread a key; the running maximum m and sum l of
// the softmax; o = sum_j e^(s_j - m) vs_j vc_j, a thread E dimensions of every `slices`-th key, as many as there are threads for, joined at the end.
// A key is seen if it is not behind the row's position, not at or before position - window, and its page is there; a row that sees none is 0.
// W codes of a key are loaded at a time (16 where a row is whole pieces of them, else 4 or 1), E of a value (4 or 1).
//
// For sizes that nothing else takes (heads of other than 64 and 128, pages of other than whole blocks): bound by the latency of a pass, two
// rounds of loads and three barriers. 8 requests of 2,000 tokens, 32 heads over 8 of 80: 89 us (278 with single codes and a thread a dimension).
template <typename CT, typename T, int W>
__global__ void __launch_bounds__(C8A_KEYS) cache8_attention_any_kernel(const T* q, long ld_q, const uint8_t* kc, const uint8_t* vc, const float* ks,
                                                                        const float* vs, long n_pages, int Hkv, int page_size, int D, const int* bt,
                                                                        long ld_table, int table_rows, int table_width, const int* row_req,
                                                                        const int* pos, int G, int window, float scale, T* out) {
  constexpr int E = W > 1 ? 4 : 1;
  __shared__ __align__(16) float q_sh[256];
  __shared__ float w_sh[C8A_KEYS], red[32], o_sh[C8A_KEYS * E];
  __shared__ long base_sh[C8A_KEYS];
  hb_pdl_launch();
  hb_pdl_wait();
  const int t = blockIdx.x, head = blockIdx.y, h = head / G, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = row_req ? row_req[t] : t, p = pos[t];
  const bool known = r >= 0 && r < table_rows;
  for (int d = tid; d < D; d += C8A_KEYS) q_sh[d] = hb_to_float(q[t * ld_q + (long)head * D + d]) * scale;
  __syncthreads();
  // dimensions d, d + 1 .. of every slices-th key from `slice` on; of more than 128 single ones a thread has those 128 on too
  const int pieces = D / E, slices = pieces < C8A_KEYS ? C8A_KEYS / pieces : 1, slice = tid / pieces, d = tid % pieces * E;
  constexpr int MORE = E == 1 ? 2 : 1, AHEAD = 8;
  float m = -INFINITY, l = 0.f, o[MORE][E] = {};
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
        const float key_scale = ks[block];
        value_scale = vs[block];
        float dot = 0.f;
        if constexpr (W == 1) {
          for (int i = 0; i < D; i++) dot = fmaf(q_sh[i], CT::value(kc[base + i]), dot);
        } else {
          const auto four = [&](uint32_t w, int i) {
            const float4 y = *(const float4*)(q_sh + i);
            float x[4];
            CT::values4(w, x);
            dot = fmaf(y.w, x[3], fmaf(y.z, x[2], fmaf(y.y, x[1], fmaf(y.x, x[0], dot))));
          };
#pragma unroll 4
          for (int i = 0; i < D; i += W) {
            if constexpr (W == 16) {
              const uint4 w = *(const uint4*)(kc + base + i);
              four(w.x, i), four(w.y, i + 4), four(w.z, i + 8), four(w.w, i + 12);
            } else {
              four(*(const uint32_t*)(kc + base + i), i);
            }
          }
        }
        s = dot * key_scale;
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
    const int n = (int)min((long)C8A_KEYS, last - j0 + 1);
#pragma unroll
    for (int c = 0; c < MORE; c++) {
#pragma unroll
      for (int e = 0; e < E; e++) o[c][e] *= f;
      if (slice < slices && d + c * C8A_KEYS < D) {
        for (int i0 = slice; i0 < n; i0 += AHEAD * slices) {      // (asked for together: one by one 8 requests took 181 us)
          uint32_t code[AHEAD];
          float weight[AHEAD];
#pragma unroll
          for (int u = 0; u < AHEAD; u++) {
            const int i = i0 + u * slices;
            const long from = i < n ? base_sh[i] : -1;
            code[u] = 0u, weight[u] = 0.f;
            if (from >= 0) {
              const uint8_t* at = vc + from + d + c * C8A_KEYS;
              weight[u] = w_sh[i];
              if constexpr (E == 1) code[u] = *at;
              else code[u] = *(const uint32_t*)at;
            }
          }
#pragma unroll
          for (int u = 0; u < AHEAD; u++) {
            float x[4] = {CT::value((uint8_t)code[u])};
            if constexpr (E == 4) CT::values4(code[u], x);
#pragma unroll
            for (int e = 0; e < E; e++) o[c][e] = fmaf(weight[u], x[e], o[c][e]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < MORE; c++) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++) o_sh[tid * E + e] = o[c][e];
    __syncthreads();
    for (int i = tid; i < D && i + c * C8A_KEYS < D && (E > 1 || i < C8A_KEYS); i += C8A_KEYS) {      // dimension i of slice n stands at n * pieces * E + i
      float x = 0.f;
      for (int n = 0; n < slices; n++) x += o_sh[n * pieces * E + i];
      out[((long)t * gridDim.y + head) * D + i + c * C8A_KEYS] = hb_from_float<T>(l == 0.f ? 0.f : x / l);
    }
  }
}

// q [n_rows][ld_q] with Hkv * G heads of D, out [n_rows][Hkv * G * D]; bt [table_rows][ld_table]; row_req null: row t is request t's.
HB_EXPORT int hb_cache8_attention_any(const void* q, int dt, long ld_q, const void* kc, const void* vc, const float* ks, const float* vs, int ct,
                                      long n_pages, int Hkv, int page_size, int D, const int* bt, long ld_table, int table_rows, int table_width,
                                      const int* row_req, const int* pos, int n_rows, int G, int window, float scale, void* out, cudaStream_t st) {
  if (n_rows <= 0) return 0;
  if (Hkv < 1 || G < 1 || (long)Hkv * G > 65535 || page_size < 1 || D < 1 || D > 256)
    HB_FAIL("hb_cache8_attention_any: %d kv heads of %d for %d heads each, pages of %d", Hkv, D, G, page_size);
  const auto pieces = [&](int n) { return D % n == 0 && !(((uintptr_t)kc | (uintptr_t)vc) & (n - 1)); };
#define C8A_LAUNCH(W)                                                                                                                              \
  hb_launch(cache8_attention_any_kernel<CT, TA, W>, dim3(n_rows, Hkv * G), dim3(C8A_KEYS), 0, st, (const TA*)q, ld_q, (const uint8_t*)kc,          \
            (const uint8_t*)vc, ks, vs, n_pages, Hkv, page_size, D, bt, ld_table, table_rows, table_width, row_req, pos, G, window, scale, (TA*)out)
  C8_DISPATCH(ct, "hb_cache8_attention_any", HB_DISPATCH_1(dt, "hb_cache8_attention_any", {
    if (pieces(16)) C8A_LAUNCH(16);
    else if (pieces(4)) C8A_LAUNCH(4);
    else C8A_LAUNCH(1);
  }));
#undef C8A_LAUNCH
  HB_CHECK_LAUNCH("hb_cache8_attention_any");
  return 0;
}
