// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Request r has n drafted tokens d_1 .. d_n and n + 1 rows of logits. p_i = softmax(logits_i / t); at t = 0, and where a row's largest logit
// is not finite (NaN counts as above all), p_i is a point mass on the lowest index of the largest. q_i is the distribution the draft was drawn
// from, or a point mass on d_i. Draft i is accepted iff all before it are and u_i q_i(d_i) < p_i(d_i); the token behind the accepted ones is
//     argmax_v w_v / e_v,   w = max(p_i - q_i, 0) at the first draft refused (p_i where that is 0 everywhere), w = p_{n+1} if none was,
// with e_v ~ Exp(1) given: the smallest of exponential variables of rates w_v is v with probability w_v / sum w.
//
// Two kernels. verify_rows_kernel reads every logit once: a block leaves a slice's maximum, its lowest index, and the sum of exponentials
// under that maximum. verify_pick_kernel has every block join its request's rows and decide (a few hundred numbers, the same in all of them),
// then go through a slice of the one row that the last token is drawn from; the blocks meet in an atomic maximum of ordered 64-bit keys
// (score, lowest index first), which does not depend on their order, and the last one to arrive writes the results.
#include "common.cuh"

namespace {

constexpr int VD_THREADS = 256, VD_MAX_DRAFTS = 63;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t ordered(float x) {          // larger numbers have larger keys, NaN the largest, 0 and -0 the same
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return x != x ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return k == 0xffffffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 key_of(uint32_t value, int index) { return (u64)value << 32 | (uint32_t)~index; }
__device__ __forceinline__ int index_of(u64 key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ u64 warp_max(u64 k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  return k;
}

struct RowPart { u64 key; float sum; int pad; };     // a slice's largest logit and its place; sum of 2^((x - largest) c)

// 16 bytes of a row as floats.
__device__ __forceinline__ void unpack(uint4 v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __bfloat1622float2(*(const __nv_bfloat162*)&w[i]);
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ int clamped(int n, int K) { return n < 0 ? 0 : n > K ? K : n; }

// A slice is VD_THREADS * U vectors of 16 bytes, counted from the row's first 16-byte boundary at or before its start (a row of an odd
// vocabulary starts anywhere): whole vectors are one load each, the two at the row's ends are read element by element.
template <typename T, int U>
__global__ void __launch_bounds__(VD_THREADS) verify_rows_kernel(const T* logits, long ld, int T_rows, int V, const int* start, const int* n_drafts, int K,
                                                                 const float* temperature, RowPart* parts, int slices, u64* keys, int* arrived) {
  constexpr int N = 16 / sizeof(T);
  __shared__ u64 sh_key[VD_THREADS / 32];
  __shared__ float sh_sum[VD_THREADS / 32];
  hb_pdl_wait();
  hb_pdl_launch();
  const int r = blockIdx.z, i = blockIdx.y, s = blockIdx.x;
  if (s == 0 && i == 0 && threadIdx.x == 0) {
    keys[2 * r] = keys[2 * r + 1] = 0;
    arrived[r] = 0;
  }
  const int row = start[r] + i;
  if (i > clamped(n_drafts[r], K) || row < 0 || row >= T_rows) return;
  const T* x = logits + (size_t)row * ld;
  const int off = (int)(((uintptr_t)x & 15) / sizeof(T));           // elements between the boundary and the row's first
  const float t = temperature[r], c = 1.4426950408889634f / (t > 0.f ? t : 1.f);
  float v[U][N];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int at = ((s * U + u) * VD_THREADS + (int)threadIdx.x) * N - off;
    if (at >= 0 && at + N <= V) unpack(*(const uint4*)(x + at), v[u]);
    else {
#pragma unroll
      for (int j = 0; j < N; j++) v[u][j] = at + j >= 0 && at + j < V ? hb_to_float(x[at + j]) : -INFINITY;
    }
  }
  // the maximum and its lowest index
  float mx = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < N; j++) {
      mx = fmaxf(mx, v[u][j]);
      nan |= v[u][j] != v[u][j];
    }
  int best = 0x7fffffff;
#pragma unroll
  for (int u = U - 1; u >= 0; u--)
#pragma unroll
    for (int j = N - 1; j >= 0; j--) {
      const int at = ((s * U + u) * VD_THREADS + (int)threadIdx.x) * N - off + j;
      if ((nan ? v[u][j] != v[u][j] : v[u][j] == mx) && at >= 0 && at < V) best = at;
    }
  u64 key = best == 0x7fffffff ? 0 : key_of(nan ? 0xffffffffu : ordered(mx), best);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  key = warp_max(key);
  if (lane == 0) sh_key[warp] = key;
  __syncthreads();
  key = warp_max(lane < VD_THREADS / 32 ? sh_key[lane] : 0);
  const float top = key ? unordered((uint32_t)(key >> 32)) : -INFINITY, sub = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < U; u++) {
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) part += exp2f((v[u][j] - sub) * c);
    sum += part;
  }
  sum = hb_warp_sum(sum);
  if (lane == 0) sh_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < VD_THREADS / 32; w++) total += sh_sum[w];
    RowPart p;
    p.key = key;
    p.sum = total;
    p.pad = 0;
    parts[((size_t)r * (K + 1) + i) * slices + s] = p;
  }
}

// The candidate v with weight w and noise e: key 0 means none.
__device__ __forceinline__ u64 candidate(float w, float e, int v) {
  if (!(w > 0.f)) return 0;
  const float s = __fdiv_rn(w, e);
  return key_of(s > 0.f ? __float_as_uint(s) + 1u : 1u, v);          // (a score that is NaN counts as 0)
}

template <typename T, typename Q>
__global__ void __launch_bounds__(VD_THREADS) verify_pick_kernel(const T* logits, long ld, int T_rows, int V, const int* start, const int* n_drafts,
                                                                 const int* drafts, int K, const float* temperature, const float* uniform,
                                                                 const float* noise, long noise_ld, const Q* probs, long probs_r, long probs_i,
                                                                 const RowPart* parts, int slices, u64* keys, int* arrived, int* tokens, int* counts,
                                                                 float* logprobs) {
  __shared__ u64 row_key[VD_MAX_DRAFTS + 1];
  __shared__ float row_sum[VD_MAX_DRAFTS + 1], row_logp[VD_MAX_DRAFTS + 1];
  __shared__ int row_ok[VD_MAX_DRAFTS + 1];
  __shared__ u64 sh_key[2][VD_THREADS / 32];
  __shared__ int sh_last;
  hb_pdl_wait();
  hb_pdl_launch();
  const int r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = start[r], n = min(clamped(n_drafts[r], K), T_rows - 1 - row0);
  const bool any = row0 >= 0 && n >= 0;                               // rows outside the logits: no token
  const float t = temperature[r], c = 1.4426950408889634f / (t > 0.f ? t : 1.f);
  // the rows' statistics and decisions, a warp a row
  for (int i = warp; any && i <= n; i += VD_THREADS / 32) {
    u64 key = 0;
    float sum = 0.f;
    for (int s0 = 0; s0 < slices; s0 += 32) {
      const RowPart p = s0 + lane < slices ? parts[((size_t)r * (K + 1) + i) * slices + s0 + lane] : RowPart{0, 0.f, 0};
      const u64 all = warp_max(p.key > key ? p.key : key);
      const float top = unordered((uint32_t)(all >> 32)), sub = top == -INFINITY ? 0.f : top;
      const float mine = p.key ? unordered((uint32_t)(p.key >> 32)) : -INFINITY, before = key ? unordered((uint32_t)(key >> 32)) : -INFINITY;
      sum = (sum == 0.f ? 0.f : sum * exp2f((before - sub) * c)) + hb_warp_sum(p.key && p.sum != 0.f ? p.sum * exp2f((mine - sub) * c) : 0.f);
      key = all;
    }
    if (lane == 0) {
      const float top = unordered((uint32_t)(key >> 32));
      const bool point = !(t > 0.f) || !isfinite(top);
      row_key[i] = key;
      row_sum[i] = sum;
      if (i < n) {
        const int d = drafts[(size_t)r * K + i];
        const bool in = d >= 0 && d < V;
        const float x = in ? hb_to_float(logits[(size_t)(row0 + i) * ld + d]) : -INFINITY;
        const float p = !in ? 0.f : point ? (d == index_of(key) ? 1.f : 0.f) : exp2f((x - top) * c) / sum;
        const float qd = !probs ? 1.f : in ? hb_to_float(probs[(size_t)r * probs_r + (size_t)i * probs_i + d]) : 0.f;
        row_ok[i] = uniform[(size_t)r * K + i] * qd < p;
        row_logp[i] = isfinite(top) ? (x - top) * (c * 0.6931471805599453f) - logf(sum) : 0.f;
      }
    }
  }
  __syncthreads();
  int taken = 0;
  while (any && taken < n && row_ok[taken]) taken++;
  const u64 top_key = any ? row_key[taken] : 0;
  const float top = unordered((uint32_t)(top_key >> 32)), sum = any ? row_sum[taken] : 1.f;
  const bool point = any && (!(t > 0.f) || !isfinite(top));
  const T* x = logits + (size_t)(row0 + taken) * ld;
  int final = -1;
  if (any && point) final = index_of(top_key);
  if (!any || point) {
    if (blockIdx.x > 0) return;
  } else {
    const bool refused = taken < n, dist = refused && probs;
    const int d = refused && !probs ? drafts[(size_t)r * K + taken] : -1;
    const Q* q = dist ? probs + (size_t)r * probs_r + (size_t)taken * probs_i : nullptr;
    const float* e = noise + (size_t)r * noise_ld;
    const float inv = 1.f / sum;
    u64 rest = 0, whole = 0;               // of max(p - q, 0) and of p
    const int per = (V + gridDim.x - 1) / gridDim.x, end = min(V, (int)(blockIdx.x + 1) * per);
    for (int v0 = blockIdx.x * per; v0 < end; v0 += 4 * VD_THREADS) {
      float xs[4], es[4], qs[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int v = v0 + u * VD_THREADS + (int)threadIdx.x;
        xs[u] = v < end ? hb_to_float(x[v]) : -INFINITY;
        es[u] = v < end ? e[v] : 1.f;
        qs[u] = v < end && dist ? hb_to_float(q[v]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int v = v0 + u * VD_THREADS + (int)threadIdx.x;
        const float p = exp2f((xs[u] - top) * c) * inv;
        const u64 a = candidate(p, es[u], v), b = dist ? candidate(fmaxf(p - qs[u], 0.f), es[u], v) : v == d ? 0 : a;
        whole = a > whole ? a : whole;
        rest = b > rest ? b : rest;
      }
    }
    rest = warp_max(rest);
    whole = warp_max(whole);
    if (lane == 0) {
      sh_key[0][warp] = rest;
      sh_key[1][warp] = whole;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < VD_THREADS / 32; w++) {
        rest = sh_key[0][w] > rest ? sh_key[0][w] : rest;
        whole = sh_key[1][w] > whole ? sh_key[1][w] : whole;
      }
      if (rest) atomicMax(&keys[2 * r], rest);
      if (whole) atomicMax(&keys[2 * r + 1], whole);
      __threadfence();
      sh_last = atomicAdd(&arrived[r], 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!sh_last) return;
    if (threadIdx.x == 0) {
      __threadfence();
      const u64 a = atomicMax(&keys[2 * r], 0ull), b = atomicMax(&keys[2 * r + 1], 0ull);
      final = index_of(a ? a : b ? b : top_key);
    }
  }
  // the results: drafts, the token behind them, -1
  for (int i = threadIdx.x; i <= K; i += VD_THREADS) {
    int token = -1;
    float lp = 0.f;
    if (any && i < taken) {
      token = drafts[(size_t)r * K + i];
      lp = row_logp[i];
    }
    if (i != taken || !any) {
      tokens[(size_t)r * (K + 1) + i] = token;
      logprobs[(size_t)r * (K + 1) + i] = lp;
    }
  }
  if (threadIdx.x == 0) {
    counts[r] = any ? taken + 1 : 0;
    if (any) {
      tokens[(size_t)r * (K + 1) + taken] = final;
      logprobs[(size_t)r * (K + 1) + taken] = isfinite(top) ? (hb_to_float(x[final]) - top) * (c * 0.6931471805599453f) - logf(sum) : 0.f;
    }
  }
}

// Vectors a thread: four are in flight at once; a few rows are cut finer so that there are blocks enough.
int vd_unroll(int V, int dt, int rows) {
  const int n = dt == HB_BF16 ? 8 : 4;
  for (int u = 8; u > 1; u >>= 1)
    if ((long)rows * ((V + n * VD_THREADS * u - 1) / (n * VD_THREADS * u)) >= 4 * 148) return u;
  return 1;
}
int vd_slices(int V, int dt, int u) {
  const int n = (dt == HB_BF16 ? 8 : 4) * VD_THREADS * u;
  return (V + (dt == HB_BF16 ? 8 : 4) - 1 + n - 1) / n;          // a row may begin up to a vector behind its boundary
}

}  // namespace

// Bytes of workspace for R requests of up to K drafts.
HB_EXPORT long hb_verify_drafts_workspace(int R, int K, int V, int dt) {
  const int s = vd_slices(V, dt, vd_unroll(V, dt, R * (K + 1)));
  return (long)R * (K + 1) * s * (long)sizeof(RowPart) + (long)R * 24;
}

HB_EXPORT int hb_verify_drafts(const void* logits, int dt, long ld, int T_rows, int V, const int* start, const int* n_drafts, const int* drafts, int R,
                               int K, const float* temperature, const float* uniform, const float* noise, long noise_ld, const void* probs,
                               int probs_dt, long probs_r, long probs_i, void* workspace, int* tokens, int* counts, float* logprobs,
                               cudaStream_t s) {
  if (R <= 0) return 0;
  if (V <= 0 || K < 0 || K > VD_MAX_DRAFTS) HB_FAIL("hb_verify_drafts: a vocabulary of %d, %d drafts (at most %d)", V, K, VD_MAX_DRAFTS);
  if (R > 65535) HB_FAIL("hb_verify_drafts: %d requests are beyond the grid limit", R);
  if (!workspace || ((uintptr_t)workspace & 15)) HB_FAIL("hb_verify_drafts: the workspace must be 16-byte aligned");
  const int u = vd_unroll(V, dt, R * (K + 1)), slices = vd_slices(V, dt, u);
  if (V > (1 << 30)) HB_FAIL("hb_verify_drafts: a vocabulary of %d", V);
  RowPart* parts = (RowPart*)workspace;
  u64* keys = (u64*)(parts + (size_t)R * (K + 1) * slices);
  int* arrived = (int*)(keys + 2 * (size_t)R);
  cudaError_t e = cudaSuccess;
#define VD_ROWS(U) e = hb_launch(verify_rows_kernel<TA, U>, dim3(slices, K + 1, R), VD_THREADS, 0, s, (const TA*)logits, ld, T_rows, V, start, n_drafts, K, \
                                 temperature, parts, slices, keys, arrived)
  HB_DISPATCH_1(dt, "hb_verify_drafts", { if (u == 8) VD_ROWS(8); else if (u == 4) VD_ROWS(4); else if (u == 2) VD_ROWS(2); else VD_ROWS(1); });
#undef VD_ROWS
  if (e != cudaSuccess) HB_FAIL("hb_verify_drafts: %s", cudaGetErrorString(e));
  int blocks = (V + 4 * VD_THREADS - 1) / (4 * VD_THREADS);
  const int most = (8 * 148 + R - 1) / R;
  if (blocks > most) blocks = most;
  HB_DISPATCH_2(dt, probs ? probs_dt : HB_F32, "hb_verify_drafts",
                e = hb_launch(verify_pick_kernel<TA, TB>, dim3(blocks, R), VD_THREADS, 0, s, (const TA*)logits, ld, T_rows, V, start, n_drafts, drafts, K,
                              temperature, uniform, noise, noise_ld, (const TB*)probs, probs_r, probs_i, parts, slices, keys, arrived, tokens,
                              counts, logprobs));
  if (e != cudaSuccess) HB_FAIL("hb_verify_drafts: %s", cudaGetErrorString(e));
  HB_CHECK_LAUNCH("hb_verify_drafts");
  return 0;
}
