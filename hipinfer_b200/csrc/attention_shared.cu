// Attention of a step's rows over a paged cache in which groups of requests share the pages of a long prefix, computed once for all rows of a
// group (csrc/shared_plan.cu makes the items).
//
//   over a range A of keys: m_A = max s_j, l_A = sum 2^(s_j - m_A), o_A = sum 2^(s_j - m_A) v_j, s_j = log2(e) scale q . k_j, all in 32 bits;
//   ranges are joined as o = sum_A 2^(m_A - m) o_A / sum_A 2^(m_A - m) l_A, m = max m_A.
//
// shared_items_kernel leaves (m, l) and o of every item's rows in the workspace; any head size up to 256, page size and group, both element
// types: 64 rows by 64 keys a tile in shared memory, or up to 16 rows without one; products on the FMA pipe, all numbers widened to 32 bits.
// bfloat16 heads of 64 and 128 go to the tensor cores instead (attention_shared_tc.cu).
// shared_join_kernel, one or four warps per row and head, adds the keys of the step's own rows (a row sees those up to itself, so that the
// items need no mask) and joins the parts in a fixed order: the same plan and inputs give the same bits.
#include "common.cuh"
#include "shared_plan.h"

#include <type_traits>

namespace {

constexpr int SI_KEYS = 64, SI_THREADS = 256, SI_FEW = 16;      // (rows: also in kernels/drafts.py)

__device__ __forceinline__ float exp2_of(float x) { return exp2f(x); }

// Four elements of a row of D from column c on, zeros behind its end.
template <typename T> __device__ __forceinline__ float4 row4(const T* row, int c, int D, bool vec) {
  if (vec && c + 4 <= D) return hb_load4(row + c);
  float4 v;
  v.x = c < D ? hb_to_float(row[c]) : 0.f;
  v.y = c + 1 < D ? hb_to_float(row[c + 1]) : 0.f;
  v.z = c + 2 < D ? hb_to_float(row[c + 2]) : 0.f;
  v.w = c + 3 < D ? hb_to_float(row[c + 3]) : 0.f;
  return v;
}

// Two numbers at a time: the FMA pipe takes as long, the issue slots are half of them.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ void copy16(void* dst, const void* src, bool some) {      // zeros where there is nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(some ? 16 : 0) : "memory");
}

template <int NC> struct ItemsShared {
  static constexpr int LD = 64 * NC + 4, LP = SI_KEYS + 4, TILE = SI_KEYS * LD, STAGES = NC <= 2 ? 2 : 1;
  static constexpr int BYTES = (64 * LD + 2 * STAGES * TILE + 64 * LP) * 4 + 2 * SI_KEYS * 8;
};

// 64 rows of an item, FMA-bound: 192 rows of 32 heads over 8 of 64 behind 8,192 tokens 369 us, 35 TFLOP/s of 72. A thread has four rows (4 ty ..) by four keys (tx, tx + 16, ..) of the scores, and four rows by 4 NC columns of the output. Tiles of K and V come by asynchronous copies a tile ahead, where rows start on 16 bytes, are 32-bit and two tiles fit (heads of up to
// 128); else through registers.
template <typename T, int NC>
__device__ __forceinline__ void item_rows(const SharedItem& e, int r0, float* sh, const T* q, long ldq, const T* kc, const T* vc, const int* bt,
                                          int bt_stride, int narrow, float* part_o, float2* part_ml, int G, int Hkv, int D, int page_size,
                                          float scale_log2, int vec) {
  using S = ItemsShared<NC>;
  constexpr int RM = 4, R = 16 * RM, DP = 64 * NC, LD = S::LD, LP = S::LP;
  constexpr bool CAN = S::STAGES == 2 && sizeof(T) == 4;
  float *sQ = sh, *sKV = sQ + 64 * LD, *sP = sKV + 2 * S::STAGES * S::TILE;     // stage s: K at 2 s, V at 2 s + 1
  long* sRow = (long*)(sP + 64 * LP);                                           // [stage][key]: where the key's row is, -1: nowhere
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, rows = e.tokens * G;
  const bool copies = CAN && vec;
  auto find = [&](int k0, int s) {                    // rows of the keys from k0 on
    if (threadIdx.x < SI_KEYS) {
      const int p = k0 + (int)threadIdx.x;
      sRow[s * SI_KEYS + threadIdx.x] =
          p < e.hi ? (((long)bt[(size_t)e.table * bt_stride + p / page_size] * Hkv + e.head) * page_size + p % page_size) * D : -1;
    }
  };
  auto bring = [&](int s) {                           // their keys and values into stage s
    float *sK = sKV + 2 * s * S::TILE, *sV = sK + S::TILE;
    for (int i = threadIdx.x; i < SI_KEYS * (DP / 4); i += SI_THREADS) {
      const int j = i / (DP / 4), c = 4 * (i % (DP / 4));
      const long row = sRow[s * SI_KEYS + j];
      if (copies) {
        const bool some = row >= 0 && c < D;
        copy16(sK + j * LD + c, kc + (some ? row + c : 0), some);
        copy16(sV + j * LD + c, vc + (some ? row + c : 0), some);
      } else {
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
        if (row >= 0) {
          k = row4(kc + row, c, D, vec);
          v = row4(vc + row, c, D, vec);
        }
        *(float4*)(sK + j * LD + c) = k;
        *(float4*)(sV + j * LD + c) = v;
      }
    }
    if (CAN) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  __syncthreads();
  find(e.lo, 0);
  for (int i = threadIdx.x; i < R * (DP / 4); i += SI_THREADS) {
    const int r = i / (DP / 4), c = 4 * (i % (DP / 4));
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < rows) v = row4(q + (size_t)(e.token + (r0 + r) / G) * ldq + (size_t)(e.head * G + (r0 + r) % G) * D, c, D, vec);
    *(float4*)(sQ + r * LD + c) = v;
  }
  __syncthreads();
  if (copies) bring(0);
  float m[RM], l[RM];
  uint64_t acc[RM][2 * NC];
  int last[RM];                                     // the last key that the row sees
#pragma unroll
  for (int i = 0; i < RM; i++) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    last[i] = e.pos == SP_NO_MASK ? SP_NO_MASK : e.pos + (r0 + ty * RM + i) / G;
#pragma unroll
    for (int c = 0; c < 2 * NC; c++) acc[i][c] = 0ull;
  }
  int stage = 0;
  for (int k0 = e.lo; k0 < e.hi; k0 += SI_KEYS) {
    if (copies) {
      if (k0 + SI_KEYS < e.hi) find(k0 + SI_KEYS, stage ^ 1);
      __syncthreads();                              // (the other stage has been read, too)
      if (k0 + SI_KEYS < e.hi) {
        bring(stage ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
    } else {
      if (k0 > e.lo) {
        __syncthreads();
        find(k0, 0);
        __syncthreads();
      }
      bring(0);
    }
    __syncthreads();
    const float *sK = sKV + 2 * stage * S::TILE, *sV = sK + S::TILE;
    if (copies) stage ^= 1;
    uint64_t s2[RM][4];
#pragma unroll
    for (int i = 0; i < RM; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) s2[i][j] = 0ull;
#pragma unroll 4
    for (int c = 0; c < DP; c += 4) {
      ulonglong2 a[RM], b[4];
#pragma unroll
      for (int i = 0; i < RM; i++) a[i] = *(const ulonglong2*)(sQ + (ty * RM + i) * LD + c);
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = *(const ulonglong2*)(sK + (tx + 16 * j) * LD + c);
#pragma unroll
      for (int i = 0; i < RM; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s2[i][j] = fma2(a[i].x, b[j].x, fma2(a[i].y, b[j].y, s2[i][j]));
    }
    float corr[RM];
#pragma unroll
    for (int i = 0; i < RM; i++) {
      float s[4], mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int p = k0 + tx + 16 * j;
        const float2 y = both(s2[i][j]);
        s[j] = p < e.hi && p <= last[i] ? (y.x + y.y) * scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[i], mx), sub = mn == -INFINITY ? 0.f : mn;
      corr[i] = exp2_of(m[i] - sub);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = exp2_of(s[j] - sub);
        sum += p;
        sP[(ty * RM + i) * LP + tx + 16 * j] = p;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = l[i] * corr[i] + sum;
    }
    __syncwarp();               // the 16 lanes that share a row of P are of one warp
#pragma unroll
    for (int i = 0; i < RM; i++) {
      const uint64_t w = pair(corr[i], corr[i]);
#pragma unroll
      for (int c = 0; c < 2 * NC; c++) acc[i][c] = fma2(acc[i][c], w, 0ull);
    }
    // a value behind a row is not multiplied by 0 (it may be an infinity or NaN), where rows do not see all keys
    auto products = [&](auto careful) {
#pragma unroll 2
      for (int j = 0; j < SI_KEYS; j += 4) {
        float pr[RM][4];
#pragma unroll
        for (int i = 0; i < RM; i++) *(float4*)pr[i] = *(const float4*)(sP + (ty * RM + i) * LP + j);
#pragma unroll
        for (int jj = 0; jj < 4; jj++)
#pragma unroll
          for (int n = 0; n < NC; n++) {
            const ulonglong2 v = *(const ulonglong2*)(sV + (j + jj) * LD + 64 * n + 4 * tx);
#pragma unroll
            for (int i = 0; i < RM; i++) {
              const uint64_t p = pair(pr[i][jj], pr[i][jj]);
              if (!decltype(careful)::value || pr[i][jj] != 0.f) {
                acc[i][2 * n] = fma2(p, v.x, acc[i][2 * n]);
                acc[i][2 * n + 1] = fma2(p, v.y, acc[i][2 * n + 1]);
              }
            }
          }
      }
    };
    if (e.pos == SP_NO_MASK) products(std::false_type());
    else products(std::true_type());
  }
#pragma unroll
  for (int i = 0; i < RM; i++) {
    const int r = r0 + ty * RM + i;
    if (r >= rows) continue;
    const size_t row = (size_t)e.part + r;
    if (tx == 0) {
      part_ml[row] = make_float2(m[i], l[i]);
      // a plan that was made for the tensor cores has a second part here (rows of q that TMA cannot address)
      if (e.tokens <= narrow) part_ml[row + rows] = make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int n = 0; n < NC; n++) {
      const float2 y[2] = {both(acc[i][2 * n]), both(acc[i][2 * n + 1])};
      const float o[4] = {y[0].x, y[0].y, y[1].x, y[1].y};
#pragma unroll
      for (int c = 0; c < 4; c++)
        if (64 * n + 4 * tx + c < D) part_o[row * D + 64 * n + 4 * tx + c] = o[c];
    }
  }
}

// Few rows of an item, RR at a time, without shared tiles: a lane has E columns of all RR rows of q and of O in registers, LPK lanes are a key, and
// a warp goes through eight keys at a time (four a half-warp; four a warp for heads above 64) on its own, the warps in turn. The sums over a key's
// lanes come by exchanging halves, so that every lane ends with whole scores of one row, and P goes round through 32 numbers of shared memory.
// The warps' results meet at the end. A tile through shared memory has one load of 16 bytes for four products where it serves few rows: 32 requests
// of one row behind 2,048 tokens of their own, 32 heads over 8 of 64 in 32 bits, 185 us through tiles, 66 so (4.1 TB/s); heads of 128 343 and 189.
// Up to 16 rows go this way (24, with the rest of a long prefix's rows, made 25 us 36).
template <int NC> struct FewRows {
  // (four rows leave two blocks an SM; more columns a lane have one in any case)
  static constexpr int RR = NC == 1 ? 4 : 8, LPK = NC == 1 ? 16 : 32, E = 64 * NC / LPK, HALVES = 32 / LPK, KEYS = 4 * HALVES;
  // what a warp has of the shared memory: m, l and O of its rows at the end; P before it
  static constexpr int FLOATS = RR * 2 + RR * 64 * NC;
};
template <typename T, int NC>
__device__ __forceinline__ void item_few_rows(const SharedItem& e, int r0, float* sh, const T* q, long ldq, const T* kc, const T* vc, const int* bt,
                                              int bt_stride, int narrow, float* part_o, float2* part_ml, int G, int Hkv, int D, int page_size,
                                              float scale_log2, int vec) {
  using F = FewRows<NC>;
  constexpr int RR = F::RR, LPK = F::LPK, E = F::E, E2 = E / 2, KEYS = F::KEYS, DP = 64 * NC, WARPS = SI_THREADS / 32;
  constexpr int PER = RR * 4 / LPK;                    // scores a lane ends with: of row `mine`, keys key0 ..
  static_assert(PER == 1 || PER == 2, "a lane's scores are of one row");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPK, half = lane / LPK, c = sub * E, rows = e.tokens * G;
  const int mine = sub * PER / 4, key0 = sub * PER % 4;
  float* own = sh + warp * F::FLOATS;
  __syncthreads();                                     // (the shared memory's last readers)
  auto load = [&](const T* row, uint64_t* x) {         // this lane's columns
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 v = row4(row, c + i, D, vec);
      x[i / 2] = pair(v.x, v.y);
      x[i / 2 + 1] = pair(v.z, v.w);
    }
  };
  uint64_t x[RR][E2], acc[RR][E2];
#pragma unroll
  for (int r = 0; r < RR; r++) {
    const int row = min(r0 + r, rows - 1);             // (the last row again behind it)
    load(q + (size_t)(e.token + row / G) * ldq + (size_t)(e.head * G + row % G) * D, x[r]);
#pragma unroll
    for (int i = 0; i < E2; i++) acc[r][i] = 0ull;
  }
  const int last = e.pos == SP_NO_MASK ? e.hi - 1 : min(e.hi - 1, e.pos + min(r0 + mine, rows - 1) / G);      // the last key that row `mine` sees
  float m = -INFINITY, l = 0.f;                        // of row `mine`; l of this lane's keys
  auto walk = [&](auto careful) {
    for (int k0 = e.lo + warp * KEYS; k0 < e.hi; k0 += WARPS * 32) {
      const int p = min(k0 + (lane / KEYS) * WARPS * KEYS + lane % KEYS, e.hi - 1), page = p / page_size;      // of this warp's keys of the next 256
      const long at = (((long)bt[(size_t)e.table * bt_stride + page] * Hkv + e.head) * page_size + (p - page * page_size)) * D;
      for (int j0 = 0, first = k0 + 4 * half; j0 < 32 && first - 4 * half < e.hi; j0 += KEYS, first += WARPS * KEYS) {      // (the last key again behind it)
        uint64_t k[4][E2], v[4][E2];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const long row = __shfl_sync(0xffffffffu, at, j0 + 4 * half + u);
          load(kc + row, k[u]);
          load(vc + row, v[u]);
        }
        float s[RR * 4];
#pragma unroll
        for (int r = 0; r < RR; r++)
#pragma unroll
          for (int u = 0; u < 4; u++) {
            uint64_t a = 0ull;
#pragma unroll
            for (int i = 0; i < E2; i++) a = fma2(x[r][i], k[u][i], a);
            const float2 y = both(a);
            s[4 * r + u] = y.x + y.y;
          }
        // sums over a key's lanes: who has the upper half of the lanes keeps the upper half of the sums
#pragma unroll
        for (int o = LPK / 2, n = RR * 2; o > 0; o >>= 1, n >>= 1) {
          const bool up = sub & o;
          if (n > 0) {
#pragma unroll
            for (int i = 0; i < n; i++) {
              const float keep = up ? s[n + i] : s[i], give = up ? s[i] : s[n + i];
              s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
          } else {
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; i++) {
          s[i] = first + key0 + i <= last ? s[i] * scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[i]);
        }
#pragma unroll
        for (int o = 4 / PER / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (F::HALVES == 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        if (__any_sync(0xffffffffu, mx > m)) {
          const float mn = fmaxf(m, mx), corr = m == mn ? 1.f : exp2_of(m - mn);
          m = mn;
          l *= corr;
#pragma unroll
          for (int r = 0; r < RR; r++) {
            const float f = __shfl_sync(0xffffffffu, corr, r * 4 / PER);
#pragma unroll
            for (int i = 0; i < E2; i++) acc[r][i] = fma2(acc[r][i], pair(f, f), 0ull);
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        __syncwarp();                                  // P's last readers
#pragma unroll
        for (int i = 0; i < PER; i++) {
          s[i] = exp2_of(s[i] - ref);
          l += s[i];
          own[half * RR * 4 + sub * PER + i] = s[i];
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < RR; r++) {
          const float4 w = *(const float4*)(own + half * RR * 4 + 4 * r);
          const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int u = 0; u < 4; u++)
            // a value behind a row is not multiplied by 0 (it may be an infinity or NaN), where rows do not see all keys
            if (!decltype(careful)::value || ws[u] != 0.f) {
#pragma unroll
              for (int i = 0; i < E2; i++) acc[r][i] = fma2(pair(ws[u], ws[u]), v[u][i], acc[r][i]);
            }
        }
      }
    }
  };
  if (e.pos == SP_NO_MASK) walk(std::false_type());
  else walk(std::true_type());
  // this warp's rows into its part of the shared memory
#pragma unroll
  for (int o = 4 / PER / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (F::HALVES == 2) l += __shfl_xor_sync(0xffffffffu, l, 16);
  __syncwarp();
  if (half == 0 && key0 == 0) {
    own[mine] = m;
    own[RR + mine] = l;
  }
#pragma unroll
  for (int r = 0; r < RR; r++)
#pragma unroll
    for (int i = 0; i < E2; i++) {
      float2 y = both(acc[r][i]);
      if (F::HALVES == 2) {
        y.x += __shfl_xor_sync(0xffffffffu, y.x, 16);
        y.y += __shfl_xor_sync(0xffffffffu, y.y, 16);
      }
      if (half == 0) *(float2*)(own + 2 * RR + r * DP + c + 2 * i) = y;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < RR * DP; i += SI_THREADS) {
    const int r = i / DP, col = i % DP;
    if (r0 + r >= rows) break;
    float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, sh[w * F::FLOATS + r]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = exp2_of(sh[w * F::FLOATS + r] - ref);              // 0 for a warp without keys
      sum = fmaf(f, sh[w * F::FLOATS + RR + r], sum);
      o = fmaf(f, sh[w * F::FLOATS + 2 * RR + i], o);
    }
    const size_t part = (size_t)e.part + r0 + r;
    if (col == 0) {
      part_ml[part] = make_float2(top, sum);
      if (e.tokens <= narrow) part_ml[part + rows] = make_float2(-INFINITY, 0.f);        // (as below)
    }
    if (col < D) part_o[part * D + col] = o;
  }
}

// An item's rows, 64 at a time, or where they are few, four or eight.
template <typename T, int NC>
__global__ void __launch_bounds__(SI_THREADS, NC == 1 ? 2 : 1) shared_items_kernel(const T* q, long ldq, const T* kc, const T* vc, const int* bt, int bt_stride,
                                                                  const SharedItem* items, const int* ctas, int narrow, float* part_o,
                                                                  float2* part_ml, int Hq, int Hkv, int D, int page_size, float scale_log2, int vec) {
  extern __shared__ __align__(16) float sh[];
  const int G = Hq / Hkv, it0 = ctas[blockIdx.x], it1 = ctas[blockIdx.x + 1];
  hb_pdl_wait();
  hb_pdl_launch();
  for (int it = it0; it < it1; it++) {
    const SharedItem e = items[it];
    const int rows = e.tokens * G;
    for (int r0 = blockIdx.y * 64; r0 < rows; r0 += gridDim.y * 64) {
      if (rows - r0 <= SI_FEW)
        for (int r = r0; r < rows; r += FewRows<NC>::RR)
          item_few_rows<T, NC>(e, r, sh, q, ldq, kc, vc, bt, bt_stride, narrow, part_o, part_ml, G, Hkv, D, page_size, scale_log2, vec);
      else
        item_rows<T, NC>(e, r0, sh, q, ldq, kc, vc, bt, bt_stride, narrow, part_o, part_ml, G, Hkv, D, page_size, scale_log2, vec);
    }
  }
}

// E elements of a row of D from column c on as floats; FULL: a row is 32 E elements and starts on 16 bytes.
template <int E, bool FULL, typename T> __device__ __forceinline__ void load_elements(const T* row, int c, int D, float* x) {
  if constexpr (!FULL) {
#pragma unroll
    for (int i = 0; i < E; i++) x[i] = c + i < D ? hb_to_float(row[c + i]) : 0.f;
  } else if constexpr (E >= 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 v = hb_load4(row + c + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else {
    float2 v;
    if constexpr (sizeof(T) == 4) v = *(const float2*)(row + c);
    else v = __bfloat1622float2(*(const __nv_bfloat162*)(row + c));
    x[0] = v.x; x[1] = v.y;
  }
}

constexpr int SJ_WARPS = 4;

// Four sums over the warp at a time, all of them in every lane: a lane that halves what it sums also halves the shuffles.
__device__ __forceinline__ void warp_sums(float* s, int lane) {
  const bool hi = lane & 16, odd = lane & 8;
  const float a0 = (hi ? s[2] : s[0]) + __shfl_xor_sync(0xffffffffu, hi ? s[0] : s[2], 16);
  const float a1 = (hi ? s[3] : s[1]) + __shfl_xor_sync(0xffffffffu, hi ? s[1] : s[3], 16);
  float c = (odd ? a1 : a0) + __shfl_xor_sync(0xffffffffu, odd ? a0 : a1, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
#pragma unroll
  for (int j = 0; j < 4; j++) s[j] = __shfl_sync(0xffffffffu, c, 8 * j);
}

// W warps per row of q and head (a block has SJ_WARPS); a lane has E columns. The parts go to the warps in turn, the keys of the step's own rows to
// the last warp; W > 1: the warps' results meet in shared memory, in their order. Latency is what it takes, a few loads that wait for one another:
// the pages of all own keys are looked up at once, a lane a key, and parts are asked for before their weights are known. The own keys come ahead
// of the wait for the items' kernel (behind_items: that one starts this one behind its own wait, when all they need is in place). 384 rows of 32
// heads with four parts each take 15 us, 8 rows 2.
template <typename T, int E, int W, bool FULL>
__global__ void __launch_bounds__(SJ_WARPS * 32, E <= 4 ? 8 : 4) shared_join_kernel(const T* q, long ldq, const T* kc, const T* vc, const int* bt, int bt_stride,
                                                                    const SharedToken* tokens, const float* part_o, const float2* part_ml, T* out, int Hq,
                                                                    int Hkv, int G, int D, int page_size, float scale_log2, int behind_items) {
  __shared__ float2 sh_ml[SJ_WARPS];
  __shared__ float sh_acc[W > 1 ? SJ_WARPS : 1][W > 1 ? 32 * E : 1];
  constexpr int AHEAD = W == 1 ? 4 : 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % W, c = lane * E;
  const int t = blockIdx.x, head = blockIdx.y * (SJ_WARPS / W) + warp / W, h = head / G, g = head - h * G;
  const bool some = head < Hq;
  const SharedToken e = tokens[t];                   // (of the plan: in place before the step's first kernel)
  float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int i = 0; i < E; i++) acc[i] = 0.f;
  if (!behind_items) hb_pdl_wait();

  // the keys of the step's own rows
  if (some && mine == W - 1 && e.fresh > 0) {
    static_assert(SP_FRESH <= 32, "a lane a key");
    float x[E];
    load_elements<E, FULL>(q + (size_t)t * ldq + (size_t)head * D, c, D, x);
    const int p = e.first + min(lane, e.fresh - 1);
    const int page = p / page_size;
    const long at = (((long)bt[(size_t)e.table * bt_stride + page] * Hkv + h) * page_size + (p - page * page_size)) * D;
    for (int j0 = 0; j0 < e.fresh; j0 += 4) {
      float k[4][E], v[4][E], s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; j++) {              // (the last key again behind it, without a branch)
        const long row = __shfl_sync(0xffffffffu, at, j0 + j);
        load_elements<E, FULL>(kc + row, c, D, k[j]);
        load_elements<E, FULL>(vc + row, c, D, v[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < E; i++) s[j] = fmaf(x[i], k[j][i], s[j]);
      if (j0 + 1 < e.fresh) warp_sums(s, lane);
      else s[0] = hb_warp_sum(s[0]);
      float mx = m;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        s[j] = j0 + j < e.fresh ? s[j] * scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[j]);
      }
      const float sub = mx == -INFINITY ? 0.f : mx, corr = exp2_of(m - sub);
      m = mx;
      l *= corr;
#pragma unroll
      for (int i = 0; i < E; i++) acc[i] *= corr;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j0 + j < e.fresh) {
          const float p = exp2_of(s[j] - sub);
          l += p;
#pragma unroll
          for (int i = 0; i < E; i++) acc[i] = fmaf(p, v[j][i], acc[i]);
        }
    }
  }
  if (behind_items) hb_pdl_wait();
  hb_pdl_launch();

  // this warp's parts, 32 at a time: a lane holds one's maximum and sum
  const int all = some ? e.pre_n + e.own_n : 0, n = (all - mine + W - 1) / W;
  const int pre0 = e.pre_base + h * e.pre_n * e.pre_rows + g, own0 = e.own_base + (h * e.own_n - e.pre_n) * e.own_rows + g;
  auto row_of = [&](int k) { return k < e.pre_n ? pre0 + k * e.pre_rows : own0 + k * e.own_rows; };
  for (int k0 = 0; k0 < n; k0 += 32) {
    const int k = (k0 + lane) * W + mine, in = min(32, n - k0);
    const float2 ml = k < all ? part_ml[row_of(k)] : make_float2(-INFINITY, 0.f);
    float o[AHEAD][E];
    auto ask = [&](int j0) {
#pragma unroll
      for (int j = 0; j < AHEAD; j++)
        load_elements<E, FULL>(part_o + (size_t)row_of((k0 + min(j0 + j, in - 1)) * W + mine) * D, c, D, o[j]);
    };
    ask(0);
    const float mx = hb_warp_max(fmaxf(ml.x, m)), sub = mx == -INFINITY ? 0.f : mx, corr = exp2_of(m - sub);
    // a part without a visible key has sum 0 and no output; one whose sum is NaN makes the row NaN
    const float w = ml.y == 0.f ? 0.f : ml.y != ml.y ? ml.y : exp2_of(ml.x - sub);
    m = mx;
    l = l * corr + hb_warp_sum(w == 0.f ? 0.f : w * ml.y);
#pragma unroll
    for (int i = 0; i < E; i++) acc[i] *= corr;
    for (int j0 = 0; j0 < in; j0 += AHEAD) {
      if (j0) ask(j0);
#pragma unroll
      for (int j = 0; j < AHEAD; j++) {
        const float wj = __shfl_sync(0xffffffffu, w, j0 + j);       // (0 behind the last part)
        if (wj != 0.f) {
#pragma unroll
          for (int i = 0; i < E; i++) acc[i] = fmaf(wj, o[j][i], acc[i]);
        }
      }
    }
  }
  if (W > 1) {
    if (lane == 0) sh_ml[warp] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < E; i++) sh_acc[warp][c + i] = acc[i];
    __syncthreads();
    if (mine != 0) return;
    for (int k = warp; k < warp + W; k++) m = fmaxf(m, sh_ml[k].x);
    const float sub = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) acc[i] = 0.f;
    for (int k = warp; k < warp + W; k++) {
      const float2 ml = sh_ml[k];
      if (ml.y == 0.f) continue;
      const float w = ml.y != ml.y ? ml.y : exp2_of(ml.x - sub);
      l = fmaf(w, ml.y, l);
#pragma unroll
      for (int i = 0; i < E; i++) acc[i] = fmaf(w, sh_acc[k][c + i], acc[i]);
    }
  }
  if (!some) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;       // a row that sees nothing is 0
  T* dst = out + ((size_t)t * Hq + head) * D;
#pragma unroll
  for (int i = 0; i < E; i++) acc[i] *= inv;
  if constexpr (FULL && E >= 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) hb_store4(dst + c + i, make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < E; i++)
      if (c + i < D) dst[c + i] = hb_from_float<T>(acc[i]);
  }
}

template <typename T, int NC>
int launch_items(const void* q, long ldq, const void* kc, const void* vc, const int* bt, int bt_stride, const SharedItem* items, const int* cta_items,
                 int ctas, int max_rows, int narrow, float* part_o, float2* part_ml, int Hq, int Hkv, int D, int page_size, float scale_log2, int vec, cudaStream_t s) {
  constexpr int smem = ItemsShared<NC>::BYTES;
  auto kern = shared_items_kernel<T, NC>;
  static bool configured[64] = {};      // the attribute belongs to a device: set once on each
  int dev = -1;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) HB_FAIL("hb_shared_items: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int blocks = (max_rows + 63) / 64;
  const cudaError_t e = hb_launch(kern, dim3(ctas, blocks < 65535 ? blocks : 65535), SI_THREADS, smem, s, (const T*)q, ldq, (const T*)kc, (const T*)vc, bt,
                                  bt_stride, items, cta_items, narrow, part_o, part_ml, Hq, Hkv, D, page_size, scale_log2, vec);
  if (e != cudaSuccess) HB_FAIL("hb_shared_items: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace

// What a call has of its plan, in host memory: the numbers that the launches want.
struct SharedLaunch { int T, ctas, max_rows, narrow, parts, tensor_cores, dt, Hq, Hkv, D, page_size, off_items, off_ctas, off_tokens, masked; };

// q [T, ldq] (heads of D side by side), caches [num_pages, Hkv, page_size, D], bt [R, bt_stride], plan on the device (see shared_plan.cu) and `h` of it;
// workspace parts * (D + 2) + 4 floats, 16-byte aligned; out [T, Hq, D]. aligned: rows of q, pages and out start on 16 bytes. `status` is set to 1 if
// a bounded wait ran out.
HB_EXPORT int hb_attention_shared(const void* q, long ldq, const void* kc, const void* vc, long num_pages, const int* bt, int bt_stride, const int* plan,
                                  const SharedLaunch* h, float* workspace, void* out, float scale, int aligned, int* status, cudaStream_t s) {
  const int Hq = h->Hq, Hkv = h->Hkv, D = h->D, ps = h->page_size, T = h->T;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv) HB_FAIL("hb_attention_shared: %d heads are not a multiple of %d kv heads", Hq, Hkv);
  if (D < 1 || D > 256 || ps < 1) HB_FAIL("hb_attention_shared: heads of %d (1 to 256 are supported), pages of %d", D, ps);
  if (!(scale >= 0.f && scale < INFINITY)) HB_FAIL("hb_attention_shared: a scale of %g", scale);
  if (T <= 0) return 0;
  const long warps = (long)T * Hq;
  if (warps > (1l << 30) || Hq > 65535) HB_FAIL("hb_attention_shared: %d rows of %d heads are beyond the grid limit", T, Hq);
  if (h->parts > 0 && (!workspace || ((uintptr_t)workspace & 15))) HB_FAIL("hb_attention_shared: the workspace must be 16-byte aligned");
  float* part_o = workspace;
  float2* part_ml = (float2*)(workspace + ((long)h->parts * D + 3) / 4 * 4);
  const SharedItem* items = (const SharedItem*)(plan + h->off_items);
  const int* cta_items = plan + h->off_ctas;
  const SharedToken* tokens = (const SharedToken*)(plan + h->off_tokens);
  const int vec = aligned && D % 4 == 0;
  const float sl2 = fmaxf(scale * 1.4426950408889634f, 1.17549435e-38f);      // (masked scores are -inf ahead of it: 0 would make them NaN)
  if (T == 1) ldq = (long)Hq * D;                        // (one row has no stride)
  // rows of q that lie over each other (one row for all, say) have no copies by boxes: they go the way of those off 16 bytes
  if (h->ctas > 0 && h->tensor_cores && aligned && ldq >= (long)Hq * D) {
    if (hb_shared_items_tc(q, ldq, kc, vc, num_pages, bt, bt_stride, items, cta_items, h->ctas, h->masked, T, part_o, part_ml, Hq, Hkv, D, ps, sl2, status, s)) return -1;
  } else if (h->ctas > 0) {
    int r = -1;
#define SI_LAUNCH(NC) \
  r = launch_items<TA, NC>(q, ldq, kc, vc, bt, bt_stride, items, cta_items, h->ctas, h->max_rows, h->narrow, part_o, part_ml, Hq, Hkv, D, ps, sl2, vec, s)
    HB_DISPATCH_1(h->dt, "hb_attention_shared", { if (D <= 64) SI_LAUNCH(1); else if (D <= 128) SI_LAUNCH(2); else SI_LAUNCH(4); });
#undef SI_LAUNCH
    if (r) return r;
  }
  cudaError_t e = cudaSuccess;
  // few rows of many parts: four warps share one's (8 rows of 32 heads behind 24,560 tokens 26.7 -> 23.8 us a call; 190 rows of 24 heads with 5 parts
  // 34.8 -> 44: more blocks than a round)
  const int W = warps > 1024 || h->parts < 6 * warps ? 1 : 4;
#define SJ_LAUNCH(E, W, FULL)                                                                                                                    \
  e = hb_launch(shared_join_kernel<TA, E, W, FULL>, dim3((unsigned)T, (unsigned)((Hq * W + SJ_WARPS - 1) / SJ_WARPS)), SJ_WARPS * 32, 0, s, (const TA*)q, ldq, \
                (const TA*)kc, (const TA*)vc, bt, bt_stride, tokens, part_o, part_ml, (TA*)out, Hq, Hkv, Hq / Hkv, D, ps, sl2, (int)(h->ctas > 0))
#define SJ_LAUNCH_W(E)                                       \
  do {                                                       \
    if (!(aligned && D == 32 * E)) SJ_LAUNCH(E, 1, false);   \
    else if (W == 1) SJ_LAUNCH(E, 1, true);                  \
    else SJ_LAUNCH(E, 4, true);                              \
  } while (0)
  HB_DISPATCH_1(h->dt, "hb_attention_shared", { if (D <= 64) SJ_LAUNCH_W(2); else if (D <= 128) SJ_LAUNCH_W(4); else SJ_LAUNCH_W(8); });
#undef SJ_LAUNCH
#undef SJ_LAUNCH_W
  if (e != cudaSuccess) HB_FAIL("hb_attention_shared: %s", cudaGetErrorString(e));
  HB_CHECK_LAUNCH("hb_attention_shared");
  return 0;
}
