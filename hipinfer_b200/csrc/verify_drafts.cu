// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Request r has n drafted tokens d_1 .. d_n and n + 1 rows of logits. p_i = softmax(logits_i / t); at t = 0, and where a row's largest logit
// is not finite (NaN counts as above all), p_i is a point mass on the lowest index of the largest. q_i is the distribution the draft was drawn
// from, or a point mass on d_i. Draft i is accepted iff all before it are and u_i q_i(d_i) < p_i(d_i); the token behind the accepted ones is
//     argmax_v w_v / e_v,   w = max(p_i - q_i, 0) at the first draft refused (p_i where that is 0 everywhere), w = p_{n+1} if none was,
// with e_v ~ Exp(1) given: the smallest of exponential variables of rates w_v is v with probability w_v / sum w.
//
// Bytes bound it: every logit once, one row of q and the noise a request. 24 requests of up to five drafts over 128,256 entries, 32-bit, take 17.5 us
// (3.7 TB/s), 96 of up to seven over 50,021 in bfloat16 28 (2.6: half of the blocks are drafts that are not there, and an exponential, a
// conversion and two sums for two bytes keep the issue slots half full). One request of three takes 6: two kernels and what they wait for.
//
// Two kernels. verify_rows_kernel reads every logit once: a block has a slice of a row in registers and leaves its maximum and sum of
// exponentials. verify_pick_kernel, a cluster a request, has every CTA join the rows' slices and decide (a few hundred numbers, the same in all
// of them), then go through a part of the one row that the last token is drawn from beside the noise and q; the best candidates meet through
// distributed shared memory, and the cluster's first CTA writes the results. (One kernel for both was slower from eight requests on.)
#include "tc_common.cuh"

#include <type_traits>

namespace {

constexpr int VD_WARPS = 8, VD_THREADS = VD_WARPS * 32, VD_MAX_DRAFTS = 63;
constexpr int VP_WARPS = 8, VP_THREADS = VP_WARPS * 32, VP_MAX_RANKS = 16, VP_U = 8;
constexpr float VD_LOG2E = 1.4426950408889634f, VD_LN2 = 0.6931471805599453f;
constexpr int VD_NONE = 0x7fffffff;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t ordered(float x) {          // larger numbers have larger keys, NaN the largest, 0 and -0 the same
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return x != x ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 key_of(uint32_t value, int index) { return (u64)value << 32 | (uint32_t)~index; }     // the lowest index wins a tie
__device__ __forceinline__ int index_of(u64 key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 warp_larger(u64 k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = larger(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

__device__ __forceinline__ float reciprocal(float x) {      // of the special-function unit (a rounding or two; of 0 infinity, of infinity 0)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 16 bytes of a row as pairs of floats, and the largest of them.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float, uint4 v, int j) { return j ? pair(v.z, v.w) : pair(v.x, v.y); }
__device__ __forceinline__ uint64_t pair_of(__nv_bfloat16, uint4 v, int j) {
  const uint32_t w = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
  return pair(w << 16, w & 0xffff0000u);
}
__device__ __forceinline__ float max_of(float, uint4 v) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ float max_of(__nv_bfloat16, uint4 v) {
  const __nv_bfloat162 m = __hmax2(__hmax2(*(const __nv_bfloat162*)&v.x, *(const __nv_bfloat162*)&v.y), __hmax2(*(const __nv_bfloat162*)&v.z, *(const __nv_bfloat162*)&v.w));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float warp_max(float x) {        // one instruction on sm_100a
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint4 minus_inf(float) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 minus_inf(__nv_bfloat16) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ float unordered(uint32_t k) {
  return k == 0xffffffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// A slice's largest logit (with its lowest index, where the request is greedy or the number not finite), and the sum of 2^((x - m) c), c = log2(e) / t.
// The subtraction comes before the factor: at the largest logit the exponent is 0 at any temperature, where x c minus a rounded m c is
// off by 2^-24 |m c| (above 126 from m / t of 1.5e9 on: sums of 0 and infinity).
struct RowPart { u64 key; float sum; int pad; };
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
// (c is finite and not 0, so that neither 0 c nor -inf c is NaN)
__device__ __forceinline__ float factor(float t) { return fminf(fmaxf(VD_LOG2E / (t > 0.f ? t : 1.f), 1.17549435e-38f), 3.40282347e38f); }
__device__ __forceinline__ int clamped(int n, int K) { return n < 0 ? 0 : n > K ? K : n; }
__device__ __forceinline__ void cluster_sync() {       // (the barrier's instructions want whole warps)
  __syncwarp();
  hb_cluster_sync();
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// The lanes' parts as one.
__device__ __forceinline__ RowPart warp_join(u64 key, float sum, float c) {
  RowPart r;
  r.key = warp_larger(key);
  const float m = unordered((uint32_t)(key >> 32)), top = unordered((uint32_t)(r.key >> 32));
  r.sum = hb_warp_sum(key == 0 || sum == 0.f ? 0.f : sum * hb_exp2((m - base_of(top)) * c));
  r.pad = 0;
  return r;
}

// A row is some elements up to its first 16-byte boundary (a row of an odd vocabulary starts anywhere), whole vectors, of which a slice has
// U * VD_THREADS (the last one what is left), and some elements more.
template <typename T, int U>
__global__ void __launch_bounds__(VD_THREADS) verify_rows_kernel(const T* logits, long ld, int T_rows, int V, const int* start, const int* n_drafts, int K,
                                                                 const float* temperature, RowPart* parts, int slices) {
  constexpr int N = 16 / sizeof(T);
  __shared__ u64 sh_key[VD_WARPS];
  __shared__ float sh_sum[VD_WARPS];
  hb_pdl_wait();
  hb_pdl_launch();
  const int r = blockIdx.z, i = blockIdx.y, s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = start[r] + i;
  if (i > clamped(n_drafts[r], K) || row < 0 || row >= T_rows) return;
  const T* x = logits + (size_t)row * ld;
  // `head` elements, n whole vectors, and the rest; of the vectors this thread has U at most: lo, lo + VD_THREADS, .. below hi
  const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T)), n = (V - head) / N;
  const int lo = s * U * VD_THREADS + (int)threadIdx.x, hi = n;
  const uint4* vec = (const uint4*)(x + head) + lo;
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    raw[u] = minus_inf(T());
    if (lo < hi - u * VD_THREADS) raw[u] = vec[u * VD_THREADS];
  }
  // the elements at the ends: the first slice's first threads
  const int rest = V - head - n * N, edge = s == 0 && (int)threadIdx.x < head + rest ? (int)threadIdx.x + ((int)threadIdx.x < head ? 0 : n * N) : -1;
  const float ex = edge >= 0 ? hb_to_float(x[edge]) : -INFINITY;
  const float t = temperature[r];
  const bool greedy = !(t > 0.f);
  const float c = factor(t);
  float mx[U], m = ex;
#pragma unroll
  for (int u = 0; u < U; u++) {
    mx[u] = max_of(T(), raw[u]);
    m = fmaxf(m, mx[u]);
  }
  m = warp_max(m);
  const float base = base_of(m);
  const uint64_t c2 = pair(__float_as_uint(c), __float_as_uint(c)), minus2 = pair(__float_as_uint(-base), __float_as_uint(-base));
  uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < N / 2; j++) {
      const float2 y = both(mul2(add2(pair_of(T(), raw[u], j), minus2), c2));
      sums[j & 1] = add2(sums[j & 1], pair(__float_as_uint(hb_exp2(y.x)), __float_as_uint(hb_exp2(y.y))));
    }
  const float2 ab = both(add2(sums[0], sums[1]));
  const float sum = hb_warp_sum(ab.x + ab.y + hb_exp2((ex - base) * c));
  const bool odd = !(fabsf(m) < INFINITY) || sum != sum;           // (NaN hides from the maximum and shows in the sum)
  uint32_t value = ordered(m);
  int at = VD_NONE;
  if (odd || greedy) {                 // the place: of a finite number, where a vector's largest is it, else of the largest key of all
    uint32_t best = edge >= 0 ? ordered(ex) : 0;
    at = edge >= 0 ? edge : VD_NONE;
#pragma unroll
    for (int u = 0; u < U; u++)
      if ((odd || mx[u] == m) && lo < hi - u * VD_THREADS) {
#pragma unroll
        for (int j = 0; j < N; j++) {
          const float2 two = both(pair_of(T(), raw[u], j / 2));
          const uint32_t key = ordered(j & 1 ? two.y : two.x);
          const int p = head + (lo + u * VD_THREADS) * N + j;
          if (key > best || (key == best && p < at)) { best = key; at = p; }
        }
      }
    value = __reduce_max_sync(0xffffffffu, best);
    at = (int)__reduce_min_sync(0xffffffffu, (unsigned)(best == value ? at : VD_NONE));
  }
  if (lane == 0) {
    sh_key[warp] = value ? key_of(value, at) : 0;                  // (nothing of the row: no key)
    sh_sum[warp] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    const RowPart p = warp_join(lane < VD_WARPS ? sh_key[lane] : 0, lane < VD_WARPS ? sh_sum[lane] : 0.f, c);
    if (lane == 0) parts[((size_t)r * (K + 1) + i) * slices + s] = p;
  }
}

template <typename T, typename Q>
__global__ void __launch_bounds__(VP_THREADS, 4) verify_pick_kernel(const T* logits, long ld, int T_rows, int V, const int* start, const int* n_drafts,
                                                                 const int* drafts, int K, const float* temperature, const float* uniform,
                                                                 const float* noise, long noise_ld, const Q* probs, long probs_r, long probs_i,
                                                                 const RowPart* parts, int slices, int* tokens, int* counts, float* logprobs) {
  struct Row { float m, s; int at, ok, d; float logp; };
  __shared__ Row rows[VD_MAX_DRAFTS + 1];
  __shared__ u64 warp_key[VP_WARPS], rank_key[VP_MAX_RANKS];
  cluster_arrive();                                   // this CTA runs: the others may write to it
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t ranks;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  const int rank = (int)hb_cluster_ctarank(), shift = __ffs(ranks) - 1, r = blockIdx.x >> shift;      // (a power of two)
  // The rows' kernel lets this one start behind its own wait: everything but its parts is in place.
  const int row0 = start[r], n = min(clamped(n_drafts[r], K), T_rows - 1 - row0);
  const bool any = row0 >= 0 && n >= 0;                               // the first row outside of the logits: no token (the last ones: fewer drafts)
  const float t = temperature[r];
  const bool greedy = !(t > 0.f);
  const float c = factor(t);
  const float* e = noise + (size_t)r * noise_ld;
  const int share = (V >> shift) + 1, begin = min(V, rank * share), end = min(V, begin + share);
  // what a draft is decided by: lane j of warp w has row w + VP_WARPS j
  const int mine = warp + VP_WARPS * lane;
  int d = -1;
  float xd = -INFINITY, qd = 0.f, ud = 0.f;
  if (any && mine < n) {
    d = drafts[(size_t)r * K + mine];
    ud = uniform[(size_t)r * K + mine];
    if (d >= 0 && d < V) {
      xd = hb_to_float(logits[(size_t)(row0 + mine) * ld + d]);
      qd = probs ? hb_to_float(probs[(size_t)r * probs_r + (size_t)mine * probs_i + d]) : 1.f;
    }
  }
  float es[VP_U];                // the noise of the first candidates
#pragma unroll
  for (int u = 0; u < VP_U; u++) {
    es[u] = 1.f;
    if (!greedy && (int)threadIdx.x < end - begin - u * VP_THREADS) es[u] = e[begin + (int)threadIdx.x + u * VP_THREADS];
  }
  hb_pdl_wait();
  hb_pdl_launch();
  // the rows' statistics and the decisions, a warp a row
  for (int i = warp; any && i <= n; i += VP_WARPS) {
    RowPart all = {0, 0.f, 0};
    for (int s0 = 0; s0 < slices; s0 += 31) {                         // (lane 31 holds what there is so far)
      RowPart p = all;
      if (lane < 31) {
        p.key = 0;
        if (s0 + lane < slices) p = parts[((size_t)r * (K + 1) + i) * slices + s0 + lane];
      }
      all = warp_join(p.key, p.sum, c);
    }
    if (lane == i / VP_WARPS) {
      const float m = unordered((uint32_t)(all.key >> 32)), y = (xd - base_of(m)) * c;
      const bool finite = fabsf(m) < INFINITY;
      Row w;
      w.m = finite ? m : INFINITY;
      w.s = finite ? all.sum : 1.f;
      w.at = index_of(all.key);
      w.d = d;
      const float p = d < 0 || d >= V ? 0.f : greedy || !finite ? (d == w.at ? 1.f : 0.f) : hb_exp2(y) / all.sum;
      w.ok = ud * qd < p;
      w.logp = finite ? y * VD_LN2 - logf(all.sum) : 0.f;
      rows[i] = w;
    }
  }
  __syncthreads();
  cluster_wait();                                     // and they run
  int taken = 0;
  while (taken < n && rows[taken].ok) taken++;
  const Row s = any ? rows[taken] : Row{INFINITY, 1.f, -1, 0, -1, 0.f};
  const bool point = greedy || !(s.m < INFINITY);
  const T* x = logits + (size_t)(row0 + taken) * ld;
  int final = s.at;
  if (!point) {
    const bool dist = taken < n && probs;
    const Q* q = dist ? probs + (size_t)r * probs_r + (size_t)taken * probs_i : nullptr;
    const float inv = 1.f / s.s;
    u64 best = 0;
    for (int attempt = 0;; attempt++) {
      // First the scores above 0 of max(p - q, 0); where there is none in the whole vocabulary, those of 0 too (their noise is infinite), and
      // then p stands in for what q has left nothing of. A thread's candidates come in rising order.
      float top = attempt ? -1.f : 0.f;
      int at = VD_NONE;
      const int skip = attempt < 2 && taken < n && !probs ? s.d - begin : VD_NONE;      // (places from `begin` on)
      auto walk = [&](auto flag, auto unroll) {
        constexpr bool WITH_Q = decltype(flag)::value;
        constexpr int U = decltype(unroll)::value, STEP = U * VP_THREADS;
        const T* xp = x + begin;
        const Q* qp = q + begin;
        const int all = end - begin;
        auto chunk = [&](int k, auto whole) {           // U candidates a thread, all of them there or not
          constexpr bool WHOLE = decltype(whole)::value;
          float xs[U], qs[U];
#pragma unroll
          for (int u = 0; u < U; u++) {
            const bool in = WHOLE || k < all - u * VP_THREADS;
            xs[u] = -INFINITY;
            qs[u] = 0.f;
            if (in) xs[u] = hb_to_float(xp[k + u * VP_THREADS]);
            if (WITH_Q && in) qs[u] = hb_to_float(qp[k + u * VP_THREADS]);
            if (U == 1 && in) es[u] = e[begin + k];
          }
#pragma unroll
          for (int u = 0; u < U; u++) {
            float w = hb_exp2((xs[u] - s.m) * c);                  // (the sum matters beside q alone)
            if (WITH_Q) w = fmaf(w, inv, -qs[u]);
            float score = w * reciprocal(es[u]);                      // infinite without noise
            if (U == 1) score = w > 0.f ? fmaxf(score, 0.f) : -1.f;   // (attempts after the first; NaN counts as 0)
            if (score > top && k + u * VP_THREADS != skip) {
              top = score;
              at = k + u * VP_THREADS;
            }
          }
        };
        int k = threadIdx.x, from = 0;
        for (; U > 1 && from + STEP <= all; from += STEP, k += STEP) {
          chunk(k, std::true_type());
          const bool more = from + 2 * STEP <= all;
#pragma unroll
          for (int u = 0; u < U; u++)
            if (more || k < all - STEP - u * VP_THREADS) es[u] = e[begin + k + STEP + u * VP_THREADS];
        }
        for (; k < all; k += STEP) chunk(k, std::false_type());
      };
      if (attempt == 0 && dist) walk(std::true_type(), std::integral_constant<int, VP_U>());
      else if (attempt == 0) walk(std::false_type(), std::integral_constant<int, VP_U>());
      else if (attempt == 1 && dist) walk(std::true_type(), std::integral_constant<int, 1>());
      else walk(std::false_type(), std::integral_constant<int, 1>());
      best = warp_larger(at == VD_NONE ? 0 : key_of(__float_as_uint(top) + 1u, begin + at));
      if (lane == 0) warp_key[warp] = best;
      __syncthreads();
      if (warp == 0) {
        best = warp_larger(lane < VP_WARPS ? warp_key[lane] : 0);
        if (lane < (int)ranks)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(hb_mapa(&rank_key[rank], lane)), "l"(best) : "memory");
      }
      cluster_sync();
      best = warp_larger(lane < (int)ranks ? rank_key[lane] : 0);
      if (best || attempt == 2) break;
      cluster_sync();                                  // all have read
    }
    final = best ? index_of(best) : 0;
  }
  if (rank != 0 || warp != 0) return;
  for (int i = lane; i <= K; i += 32) {           // drafts, the token behind them, -1
    int token = -1;
    float lp = 0.f;
    if (any && i < taken) {
      token = rows[i].d;
      lp = rows[i].logp;
    } else if (any && i == taken) {
      token = final;
      if (s.m < INFINITY) lp = (hb_to_float(x[final]) - s.m) * c * VD_LN2 - logf(s.s);
    }
    tokens[(size_t)r * (K + 1) + i] = token;
    logprobs[(size_t)r * (K + 1) + i] = lp;
  }
  if (lane == 0) counts[r] = any ? taken + 1 : 0;
}

// The cut: U vectors a thread (32 elements where that leaves blocks for all SMs, 64 of bfloat16 would take
// the registers of half of the warps; few rows are cut finer), and CTAs a request for the last token, up to 16 of
// at least 1,024 candidates, as many as one round of the SMs has (two rounds: 96 requests 31 us instead of 28).
struct Cut { int u, slices, ranks; };
Cut cut(int V, int dt, int R, int K) {
  const int n = V / (dt == HB_BF16 ? 8 : 4);
  Cut c;
  for (c.u = dt == HB_BF16 ? 4 : 8; c.u > 1; c.u >>= 1)
    if ((long)R * (K + 1) * (n / (c.u * VD_THREADS)) >= 4 * 148) break;
  c.slices = n / (c.u * VD_THREADS) + 1;
  c.ranks = 1;
  while (c.ranks < VP_MAX_RANKS && (long)R * c.ranks * 2 <= 4 * 148 && V > c.ranks * 1024) c.ranks *= 2;
  return c;
}

template <typename T, typename Q>
cudaError_t launch_pick(const Cut& k, const void* logits, long ld, int T_rows, int V, const int* start, const int* n_drafts, const int* drafts, int R, int K,
                        const float* temperature, const float* uniform, const float* noise, long noise_ld, const void* probs, long probs_r,
                        long probs_i, const RowPart* parts, int* tokens, int* counts, float* logprobs, cudaStream_t s) {
  auto kern = verify_pick_kernel<T, Q>;
  static bool configured[64] = {};      // the attribute belongs to a device: set once on each
  int dev = -1;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return hb_launch_cluster(kern, dim3((unsigned)R * k.ranks), VP_THREADS, 0, s, dim3(k.ranks, 1, 1), (const T*)logits, ld, T_rows, V, start, n_drafts, drafts, K,
                           temperature, uniform, noise, noise_ld, (const Q*)probs, probs_r, probs_i, parts, k.slices, tokens, counts, logprobs);
}

}  // namespace

// Floats of workspace for R requests of up to K drafts, or -1 beyond the limits.
HB_EXPORT int hb_verify_drafts_workspace(int R, int K, int V, int dt) {
  if (R < 1 || R > 65535 || K < 0 || K > VD_MAX_DRAFTS || V < 1 || V > (1 << 30)) return -1;
  const long n = (long)R * (K + 1) * cut(V, dt, R, K).slices * (long)(sizeof(RowPart) / 4);
  return n < 0x7fffffff ? (int)n : -1;
}

// logits [T_rows, V] with rows `ld` elements apart; start, n_drafts, temperature [R]; drafts, uniform [R, K]; noise [R, V] with rows noise_ld apart; probs
// [R, K, V] with the strides probs_r, probs_i, or none; tokens, logprobs [R, K + 1], counts [R].
HB_EXPORT int hb_verify_drafts(const void* logits, int dt, long ld, int T_rows, int V, const int* start, const int* n_drafts, const int* drafts, int R,
                               int K, const float* temperature, const float* uniform, const float* noise, long noise_ld, const void* probs,
                               int probs_dt, long probs_r, long probs_i, void* workspace, int* tokens, int* counts, float* logprobs,
                               cudaStream_t s) {
  if (R <= 0) return 0;
  if (V <= 0 || V > (1 << 30) || K < 0 || K > VD_MAX_DRAFTS) HB_FAIL("hb_verify_drafts: a vocabulary of %d, %d drafts (at most %d)", V, K, VD_MAX_DRAFTS);
  if (R > 65535) HB_FAIL("hb_verify_drafts: %d requests are beyond the grid limit", R);
  if (hb_verify_drafts_workspace(R, K, V, dt) < 0) HB_FAIL("hb_verify_drafts: %d requests of %d drafts, a vocabulary of %d: too many parts", R, K, V);
  if (!workspace || ((uintptr_t)workspace & 15)) HB_FAIL("hb_verify_drafts: the workspace must be 16-byte aligned");
  const Cut k = cut(V, dt, R, K);
  RowPart* parts = (RowPart*)workspace;
  cudaError_t e = cudaSuccess;
#define VD_LAUNCH_ROWS(U) e = hb_launch(verify_rows_kernel<TA, U>, dim3(k.slices, K + 1, R), VD_THREADS, 0, s, (const TA*)logits, ld, T_rows, V, start, \
                                        n_drafts, K, temperature, parts, k.slices)
  HB_DISPATCH_1(dt, "hb_verify_drafts", { if (k.u == 8 && sizeof(TA) == 4) VD_LAUNCH_ROWS(sizeof(TA) == 4 ? 8 : 4); else if (k.u == 4) VD_LAUNCH_ROWS(4); else if (k.u == 2) VD_LAUNCH_ROWS(2); else VD_LAUNCH_ROWS(1); });
#undef VD_LAUNCH_ROWS
  if (e != cudaSuccess) HB_FAIL("hb_verify_drafts: %s", cudaGetErrorString(e));
  HB_DISPATCH_2(dt, probs ? probs_dt : HB_F32, "hb_verify_drafts",
                e = (launch_pick<TA, TB>(k, logits, ld, T_rows, V, start, n_drafts, drafts, R, K, temperature, uniform, noise, noise_ld, probs, probs_r, probs_i,
                                         parts, tokens, counts, logprobs, s)));
  if (e != cudaSuccess) HB_FAIL("hb_verify_drafts: %s", cudaGetErrorString(e));
  HB_CHECK_LAUNCH("hb_verify_drafts");
  return 0;
}
