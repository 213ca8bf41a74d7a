// The items of the shared-prefix attention (shared_plan.cu, attention_shared.cu) on the 5th-generation tensor cores: bfloat16, heads of 64 or 128.
//
// Persistent CTAs, one an SM, walk the items that the plan gives them. An item is up to 2 x 128 query rows (consecutive tokens times the heads
// of a kv head) against a range of keys, in tiles of 128 absolute positions. Two CHAINS, a softmax warpgroup, an MMA warp, score tiles, an
// accumulator and running maxima and sums each, work beside each other in STEPS of 128 rows by 64 keys: where an item has more rows than 128 a
// chain has half of them and takes a tile in two steps, and the tile of K and V that was loaded once serves both; where it has fewer, both
// chains have the same rows, each a half of every tile's keys, and each leaves a part of the result.
//   softmax warps   a thread owns a query row: reads a step's scores from tensor memory, masks them where the tile reaches over the item's range or the
//                   row's position, exponentiates in 32 bits, and writes P as bfloat16 over the scores, from where the second product reads
//                   it as its A operand (shared memory then feeds Q, K and V alone);
//   an MMA warp a chain   O += P V of a step as soon as its P is written, and right behind it S = Q K^T of the step after the next into the
//                   same tensor memory (the tensor core works in the order of issue), which is done while the softmax warps are at the next step;
//   K and V loaders TMA, a page and 64 columns a box, a lane holds a page's number; Q comes with K, one box of (64 columns, heads, tokens).
// The accumulator is rescaled only when a row's maximum grew by more than a power of 2 (any reference value gives the same quotient).
// V rows outside of the item's range, which may hold anything, are set to zero in shared memory by the softmax threads that mask them: P
// is 0 there, and 0 times an infinity is no 0. For the same reason, where a step has keys that some rows of the item do not see (portions of more
// than SP_FRESH rows), values that are not finite are looked for, set to zero, and make the rows that do see them NaN (scan_values).
// That is an instance of the kernel by itself: a portion of 4,096 rows of 32 heads of 128 takes 210 us, 194 without, and the registers cost
// steps without such keys 2 to 5 %. Every wait is bounded; both chains wait for and release every tile and every Q, so that a barrier is never
// more than a phase ahead of one that waits for it.
//
// What bounds it: with many rows the softmax (a step is 64 exponentials of 128 rows for two products of 128 x 64 x D; two warps share a scheduler):
// 384 rows of 32 heads over 8 of 128 behind 24,560 shared tokens take 143 us, 1,082 TFLOP/s. With few rows the memory: 32 requests of one row
// behind 8,192 tokens of their own 170 us, 6.3 TB/s. In short calls latency: an item's first tile and its end, 2 us each. A chain takes
// 64 keys a step so that its scores fit into registers beside the running numbers; two chains an SM, since one alone leaves the tensor core idle during
// its softmax and four, with the registers for half of the keys each, were slower.
#include "shared_plan.h"
#include "tc_common.cuh"

namespace {

constexpr int ST_ROWS = 128, ST_KEYS = 128, ST_THREADS = 384, ST_KEPT = 64;

template <int D> struct StSizes {
  static constexpr int TILE = 128 * 64 * 2;                 // [128][64] bfloat16; an operand of D columns is D / 64 of them
  static constexpr int OPND = D / 64 * TILE;
  static constexpr int NK = D == 128 ? 2 : 4, NV = D == 128 ? 3 : 8;
};
template <int D> struct StBars {
  uint64_t q_full[2], q_free[2], k_full[StSizes<D>::NK], k_free[StSizes<D>::NK], v_full[StSizes<D>::NV], v_free[StSizes<D>::NV];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];      // [chain][step & 1]
  uint64_t scanned[2];                                     // a chain's warps have all looked through a step's values
  alignas(8) uint32_t bad[StSizes<D>::NV][4];              // a tile's values that are not finite, a bit a row
  uint32_t tmem_slot;
  int abort_flag;
  alignas(16) SharedItem kept[ST_KEPT];
};
template <int D> constexpr int st_smem() { return (2 + StSizes<D>::NK + StSizes<D>::NV) * StSizes<D>::OPND + (int)sizeof(StBars<D>); }
static_assert(st_smem<128>() <= 227 * 1024 && st_smem<64>() <= 227 * 1024, "shared memory of a block");

// MN-major operand with the 128-byte swizzle (V as it lies in its pages): 64 contiguous elements of the head a row, eight keys per 1,024-byte
// group; the next 64 columns lie a tile further.
__device__ __forceinline__ uint64_t desc_mn128(uint32_t smem_addr, int next) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D[tensor memory] (+)= A[tensor memory: a lane a row, two bfloat16 a column] B[shared memory]; one thread.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 columns of this thread's lane, not waited for, and back.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(taddr));
}
__device__ __forceinline__ void ld32_fence(uint32_t* r) { asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory"); }
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
// 16 lanes by 64 columns: of each eight columns a thread has two neighbours (2 (lane % 4)) of rows lane / 4 and lane / 4 + 8.
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(taddr));
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {   // two fmaf, each rounded by itself
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest of three numbers, NaN if there is one.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^t of two numbers, t <= 8, on the FMA pipe: t = n + f with n its nearest integer, 2^f for |f| <= 1/2 as a polynomial of degree 4 that is 1 at 0
// (fitted to the least relative error, 2.9e-6), n added to the exponent. Below -127, -inf too, it is 0; of NaN it is any number.
__device__ __forceinline__ void exp2_poly(uint64_t t2, float& p0, float& p1) {
  float t0, t1;
  unpack2(t2, t0, t1);
  t0 = fmaxf(t0, -127.f);
  t1 = fmaxf(t1, -127.f);
  const uint64_t t = pack2(t0, t1), magic = pack2(12582912.f, 12582912.f), minus = pack2(-12582912.f, -12582912.f);
  const uint64_t y = add2(t, magic), n = add2(y, minus), f = fma2(n, pack2(-1.f, -1.f), t);
  uint64_t p = fma2(f, pack2(0.009582818485796452f, 0.009582818485796452f), pack2(0.05590637028217316f, 0.05590637028217316f));
  p = fma2(p, f, pack2(0.24024099111557007f, 0.24024099111557007f));
  p = fma2(p, f, pack2(0.6931241750717163f, 0.6931241750717163f));
  p = fma2(p, f, pack2(1.f, 1.f));
  float y0, y1;
  unpack2(y, y0, y1);
  unpack2(p, p0, p1);
  p0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(y0) << 23));
  p1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(y1) << 23));
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(hb_smem_u32(dst)), "l"((uint64_t)m), "r"(hb_smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Whether a phase is over, without waiting; and a wait, of which only the first look stands in line (a loop at every place it is used made the
// kernel 60 KB of code, and every role's instructions came late).
__device__ __forceinline__ bool is_over(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(hb_smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, volatile int* abort) { return hb_mbar_wait(bar, parity, abort); }
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return hb_mbar_try_wait(bar, parity) || wait_longer(bar, parity, abort);
}

// A warp's rows of O from tensor memory to `dst`, the first n of 32. A store of a thread's own row would touch 32 lines of 128 bytes (256 rows of
// 128 took 9,500 cycles): here four threads have 64 bytes of a row, neighbours having swapped two columns of eight for two of the next eight.
template <int D> __device__ __noinline__ void store_rows(uint32_t tmem_o, float* dst, int n) {
  const int lane = threadIdx.x & 31, r = lane >> 2, odd = lane & 1;
  dst += r * D + 8 * odd + 4 * (lane >> 1 & 1);
  for (int half = 0; half < 2 && 16 * half < n; half++) {
#pragma unroll 1
    for (int q = 0; q < D / 64; q++) {
      uint32_t o[32];
      ld16(tmem_o + ((uint32_t)(16 * half) << 16) + q * 64, o);
      hb_tmem_ld_wait();
      ld32_fence(o);
#pragma unroll
      for (int i = 0; i < 32; i += 8)          // two eights of columns
#pragma unroll
        for (int k = 0; k < 4; k += 2) {       // the thread's two rows
          const uint32_t x0 = __shfl_xor_sync(0xffffffffu, odd ? o[i + k] : o[i + 4 + k], 1);
          const uint32_t x1 = __shfl_xor_sync(0xffffffffu, odd ? o[i + k + 1] : o[i + 5 + k], 1);
          const uint4 v = odd ? make_uint4(x0, x1, o[i + 4 + k], o[i + 5 + k]) : make_uint4(o[i + k], o[i + k + 1], x0, x1);
          if (r + 16 * half + 4 * k < n) *(uint4*)(dst + (16 * half + 4 * k) * D + q * 64 + 2 * i) = v;
        }
    }
  }
}

// This thread's row of O times `by`.
template <int D> __device__ __noinline__ void scale_rows(uint32_t tmem_o, float by) {
#pragma unroll 1
  for (int q = 0; q < D / 32; q++) {
    uint32_t o[32];
    ld32(tmem_o + q * 32, o);
    hb_tmem_ld_wait();
    ld32_fence(o);
#pragma unroll
    for (int d = 0; d < 32; d++) o[d] = __float_as_uint(__uint_as_float(o[d]) * by);
    st32(tmem_o + q * 32, o);
  }
}

// The values of a step that not all rows of the item see, keys [lo, hi) of its 64: those that are not finite are set to zero. Two threads have a row
// of V; what they find they mark in `bad` first, so that the other chain, which goes through the same tile of a wide item, knows of rows
// that this one has emptied. 1: there is one among the keys up to `last`, which this thread's row sees; 2: a wait ran out.
template <int D> __device__ __noinline__ int scan_values(uint8_t* rows, uint32_t* bad, uint64_t* bar, uint32_t parity, int lo, int hi, int last, volatile int* abort) {
  const int row = (threadIdx.x & 127) >> 1;
  const uint32_t mine = hb_smem_u32(rows) + row * 128 + (threadIdx.x & 1) * (D == 128 ? StSizes<D>::TILE : 64);
  if (row >= lo && row < hi) {
    uint32_t found = 0;
#pragma unroll
    for (int q = 0; q < D / 16; q++) {
      uint32_t x[4];
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(mine + q * 16) : "memory");
#pragma unroll
      for (int i = 0; i < 4; i++) found |= __vcmpeq2(x[i] & 0x7f807f80u, 0x7f807f80u);
    }
    if (found) {
      atomicOr(bad + (row >> 5), 1u << (row & 31));
      __threadfence_block();
    }
  }
  __syncwarp();
  if ((threadIdx.x & 31) == 0) hb_mbar_arrive(bar);
  if (!__all_sync(0xffffffffu, wait_for(bar, parity, abort))) return 2;
  const unsigned long long all = *(volatile unsigned long long*)bad;
  if (!all) return 0;
  if (all >> row & 1) {
#pragma unroll
    for (int q = 0; q < D / 16; q++) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(mine + q * 16), "r"(0) : "memory");
  }
  return last >= 0 && (all & (~0ull >> (63 - min(last, 63)))) != 0;
}

// The CTA's items: the first ST_KEPT of them are in shared memory.
struct Items {
  const SharedItem *kept, *all;
  int n, tokens_a_chain, tokens_low;
};
struct Work {      // an item as the roles go through it
  SharedItem e;
  int kt0, tiles;  // its key tiles
  bool wide;       // a chain has half of the rows (else half of a tile's keys)
  bool low;        // at most 64 rows: chain 1 has them in its rows 64 .., so that the two chains' warps are not of the same schedulers
};
__device__ __forceinline__ Work work_of(const Items& items, int it) {
  Work w;
  const int4* src = (const int4*)(it < ST_KEPT ? items.kept + it : items.all + it);
  *(int4*)&w.e = src[0];
  *((int4*)&w.e + 1) = src[1];
  w.kt0 = w.e.lo / ST_KEYS;
  w.tiles = (w.e.hi - 1) / ST_KEYS - w.kt0 + 1;
  w.wide = w.e.tokens > items.tokens_a_chain;
  w.low = w.e.tokens <= items.tokens_low;
  return w;
}

// MASKED: there are items whose rows do not see all keys.
template <int D, bool MASKED>
__global__ void __launch_bounds__(ST_THREADS, 1) shared_items_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                        const __grid_constant__ CUtensorMap map_v, const int* bt, int bt_stride,
                                                                        const SharedItem* plan_items, const int* ctas, float* part_o, float2* part_ml,
                                                                        int Hkv, int G, int page_size, float scale_log2, float slack, int* status) {
  using S = StSizes<D>;
  constexpr int NH = D / 64, TILE = S::TILE, OPND = S::OPND, NK = S::NK, NV = S::NV;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *sK = smem, *sQ = sK + NK * OPND, *sV = sQ + 2 * OPND;      // (chain 1 of a low item reads 64 rows from below Q: K, whatever is there)
  StBars<D>* bar = (StBars<D>*)(sV + NV * OPND);
  volatile int* abort_flag = &bar->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (hb_smem_u32(smem) & 1023) {   // never seen; the tiles would not be where the tensor core expects them
    hb_pdl_wait();
    hb_pdl_launch();
    if (threadIdx.x == 0) atomicExch(status, 1);
    return;
  }
  if (threadIdx.x == 0) {
    // (what is loaded has to be let go by both chains)
    for (int b = 0; b < 2; b++) {
      hb_mbar_init(&bar->q_full[b], 1); hb_mbar_init(&bar->q_free[b], 2); hb_mbar_init(&bar->scanned[b], 4);
      for (int h = 0; h < 2; h++) { hb_mbar_init(&bar->s_full[b][h], 1); hb_mbar_init(&bar->p_full[b][h], 4); hb_mbar_init(&bar->pv_done[b][h], 1); }
    }
    for (int b = 0; b < NK; b++) { hb_mbar_init(&bar->k_full[b], 1); hb_mbar_init(&bar->k_free[b], 2); }
    for (int b = 0; b < NV; b++) { hb_mbar_init(&bar->v_full[b], 1); hb_mbar_init(&bar->v_free[b], 2); }
    bar->abort_flag = 0;
    hb_fence_barrier_init();
  }
  if (warp == 8 && lane == 0) { hb_tma_prefetch_desc(&map_q); hb_tma_prefetch_desc(&map_k); hb_tma_prefetch_desc(&map_v); }
  if (warp == 10) {
    hb_tmem_alloc(&bar->tmem_slot, 512);
    hb_tmem_relinquish();
  }
  // (the plan is copied before the step's first kernel begins: it may be read ahead of the wait; block tables are read behind it)
  const int it0 = ctas[blockIdx.x], RT = ST_ROWS / G;
  Items items = {bar->kept, plan_items + it0, ctas[blockIdx.x + 1] - it0, RT, 64 / G};
  for (int i = threadIdx.x; i < 2 * min(items.n, ST_KEPT); i += ST_THREADS) ((int4*)bar->kept)[i] = ((const int4*)items.all)[i];
  hb_tc_fence_before();
  __syncthreads();
  hb_tc_fence_after();
  const uint32_t tmem = bar->tmem_slot;   // S and P of chain c at c * 128, its O at 256 + c * 128
  hb_pdl_wait();
  hb_pdl_launch();

  // Key tiles are numbered through all items of the CTA, a chain's steps too. Q buffers: a wide item has both, a narrow one the one that the narrow item
  // before did not have.
  if (warp >= 8) {
  if (warp < 10) {  // ---------------- TMA
    const bool is_k = warp == 8;
    const CUtensorMap* map = is_k ? &map_k : &map_v;
    uint64_t *full = is_k ? bar->k_full : bar->v_full, *free = is_k ? bar->k_free : bar->v_free;
    uint8_t* ring = is_k ? sK : sV;
    const uint32_t stages = is_k ? NK : NV;
    const int places = ST_KEYS / page_size;
    uint32_t stage = 0, parity = 1, q_parity = 3, qb = 0;
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t p) { return ok = __all_sync(0xffffffffu, wait_for(b, p, abort_flag)); };
    // the page of this lane's place in tile t, asked for a tile ahead
    auto page = [&](const Work& w, int t) {
      const int pg = (w.kt0 + t) * places + lane;
      return lane < places && pg * page_size < w.e.hi && (pg + 1) * page_size > w.e.lo ? bt[(size_t)w.e.table * bt_stride + pg] : -1;
    };
    Work w = work_of(items, 0);
    int ahead = page(w, 0);
    for (int it = 0, t = 0; it < items.n && ok;) {
      if (is_k && t == 0) {
        for (int c = 0; c < (w.wide ? 2 : 1); c++) {
          const uint32_t b = w.wide ? (uint32_t)c : qb;
          if (!wait(&bar->q_free[b], q_parity >> b & 1)) break;
          q_parity ^= 1u << b;
          if (hb_elect()) {
            hb_mbar_expect_tx(&bar->q_full[b], (uint32_t)(RT * G * D * 2));
#pragma unroll
            for (int hf = 0; hf < NH; hf++)
              tma_load_3d(sQ + b * OPND + hf * TILE, &map_q, &bar->q_full[b], hf * 64, w.e.head * G, w.e.token + c * RT);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (!w.wide) qb ^= 1;
      }
      const uint32_t boxes = __ballot_sync(0xffffffffu, ahead >= 0);
      const int row = (ahead * Hkv + w.e.head) * page_size;
      if (++t == w.tiles) {
        t = 0;
        if (++it < items.n) w = work_of(items, it);
      }
      if (it < items.n) ahead = page(w, t);
      if (!wait(&free[stage], parity)) break;
      if (MASKED && !is_k && lane < 4) bar->bad[stage][lane] = 0;
      __syncwarp();
      if (hb_elect()) hb_mbar_expect_tx(&full[stage], (uint32_t)__popc(boxes) * page_size * D * 2);
      __syncwarp();
      for (int p = 0; p < places; p += 4) {       // four boxes an election
        int from[4];
#pragma unroll
        for (int j = 0; j < 4; j++) from[j] = __shfl_sync(0xffffffffu, row, (p + j) & 31);
        if (hb_elect()) {
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (p + j < places && (boxes >> (p + j) & 1)) {
              uint8_t* dst = ring + stage * OPND + (p + j) * page_size * 128;            // rows of 128 bytes in each 64-column tile
#pragma unroll
              for (int hf = 0; hf < NH; hf++) hb_tma_load_2d(dst + hf * TILE, map, &full[stage], hf * 64, from[j]);
            }
        }
        __syncwarp();
      }
      if (++stage == stages) { stage = 0; parity ^= 1; }
    }
  } else {  // ---------------- tensor cores: warp 10 + c issues the products of chain c
    if (hb_elect()) {
      const uint32_t c = warp - 10, tmem_s = tmem + c * 128, tmem_o = tmem + 256 + c * 128;
      constexpr uint32_t idesc_s = hb_umma_idesc_bf16(ST_ROWS, 64), idesc_o = hb_umma_idesc_bf16(ST_ROWS, D) | (1u << 16);      // (V is MN-major)
      const uint64_t q_desc = hb_umma_desc_k128(hb_smem_u32(sQ)), k_desc = hb_umma_desc_k128(hb_smem_u32(sK)), v_desc = desc_mn128(hb_smem_u32(sV), TILE);
      // Where the scores are, and where the products: an item's tiles and kind, the tile in it and its half, the tile's stage and the parity of
      // the stage's use.
      struct At {
        int it, tile, tiles;
        uint32_t wide, half, stage, parity, below;
      };
      auto item = [&](At& a) {
        const Work w = work_of(items, a.it);
        a.tile = 0;
        a.tiles = w.tiles;
        a.wide = w.wide;
        a.half = w.wide ? 0 : c;
        a.below = w.low && c ? 64 * 128 >> 4 : 0;
      };
      auto next = [&](At& a, uint32_t stages) {
        if (a.wide && a.half == 0) {
          a.half = 1;
          return;
        }
        if (++a.stage == stages) { a.stage = 0; a.parity ^= 1; }
        a.half = a.wide ? 0 : c;
        if (++a.tile == a.tiles && ++a.it < items.n) item(a);
      };
      At s = {0, 0, 0, 0, 0, 0, 0, 0}, o;
      item(s);
      o = s;
      uint32_t q_parity = 0, qb = 0;               // of the two Q buffers as bits; the narrow items' buffer
      uint32_t ms = 0, mo = 0, polls = 0;          // steps whose scores, and whose products, were issued: at most two of the former ahead
      while (o.it < items.n) {
        polls++;
        const bool first = !s.wide || s.half == 0;           // the step is its tile's first of this chain
        const uint32_t b = s.wide ? c : qb;
        if (s.it < items.n && ms < mo + 2 &&
            (!first || (is_over(&bar->k_full[s.stage], s.parity) &&
                        (s.tile > 0 || (is_over(&bar->q_full[b], q_parity >> b & 1) && (!s.wide || is_over(&bar->q_full[b ^ 1], q_parity >> (b ^ 1) & 1))))))) {
          if (s.tile == 0 && first) q_parity ^= s.wide ? 3u : 1u << b;
          hb_tc_fence_after();
          const uint64_t dq = q_desc + b * (OPND >> 4) - s.below, dk = k_desc + s.stage * (OPND >> 4) + s.half * (64 * 128 >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++)     // 16 columns a step: four steps in each 64-column tile
            hb_umma_bf16(tmem_s + (ms & 1) * 64, dq + (kk >> 2) * (TILE >> 4) + 2 * (kk & 3), dk + (kk >> 2) * (TILE >> 4) + 2 * (kk & 3), idesc_s, kk != 0);
          hb_umma_commit(&bar->s_full[c][ms & 1]);
          if (!s.wide || s.half) {
            hb_umma_commit(&bar->k_free[s.stage]);
            if (s.tile == s.tiles - 1) {
              hb_umma_commit(&bar->q_free[b]);
              if (s.wide) hb_umma_commit(&bar->q_free[b ^ 1]);
              else qb ^= 1;
            }
          }
          next(s, NK);
          ms++;
          polls = 0;
        }
        if (mo < ms && is_over(&bar->p_full[c][mo & 1], mo >> 1 & 1) && is_over(&bar->v_full[o.stage], o.parity)) {
          hb_tc_fence_after();
          const uint32_t fresh = o.tile == 0 && (!o.wide || o.half == 0);           // the accumulator's first step
          const uint64_t dv = v_desc + o.stage * (OPND >> 4) + o.half * (64 * 128 >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; kk++)          // 16 keys: eight columns of P, 16 rows of V
            umma_ts(tmem_o, tmem_s + (mo & 1) * 64 + 8 * kk, dv + kk * (16 * 128 >> 4), idesc_o, kk != 0 || !fresh);
          hb_umma_commit(&bar->pv_done[c][mo & 1]);
          if (!o.wide || o.half) hb_umma_commit(&bar->v_free[o.stage]);
          next(o, NV);
          mo++;
          polls = 0;
        }
        if ((polls & 63) == 63 && *abort_flag) break;
        if (polls > 16 * HB_WAIT_LIMIT) {          // (these looks do not suspend)
          *abort_flag = 1;
          break;
        }
      }
    }
  }
  } else {  // ---------------- softmax: warpgroup c is chain c, a thread a query row
    const int c = warp >> 2, w4 = warp & 3;
    const uint32_t lanes = (uint32_t)(w4 * 32) << 16, tmem_s = tmem + c * 128 + lanes, tmem_o = tmem + 256 + c * 128 + lanes;
    uint32_t m = 0, scans = 0, v_stage = 0, v_parity = 0;       // steps, and those whose values were looked through; where V is
    bool ok = true;                // every wait's outcome is made uniform over the warp: the tensor-memory accesses below are warp-wide
    auto wait = [&](uint64_t* b, uint32_t parity) { return ok = __all_sync(0xffffffffu, wait_for(b, parity, abort_flag)); };
    const uint64_t scale2 = pack2(scale_log2, scale_log2);
    for (int it = 0; it < items.n && ok; it++) {
      const Work w = work_of(items, it);
      const int first = w.wide ? c * RT : 0, rows = min(RT, w.e.tokens - first) * G;           // the chain's rows
      const int below = w.low && c ? 64 : 0, r = (int)(threadIdx.x & 127) - below;      // the thread's row of the chain's
      const bool idle = w4 * 32 < below || w4 * 32 - below >= rows;
      const int last_key = !MASKED || w.e.pos == SP_NO_MASK ? w.e.hi - 1 : min(w.e.hi - 1, w.e.pos + first + r / G);
      const int sure = !MASKED || w.e.pos == SP_NO_MASK ? w.e.hi : min(w.e.hi, w.e.pos + first + 1);      // the keys below are seen by all rows
      float m_run = -INFINITY, l_run = 0.f;
      const uint32_t m0 = m;
      for (int i = 0; i < w.tiles && ok; i++) {
        const int tile = (w.kt0 + i) * ST_KEYS;
        for (int h = w.wide ? 0 : c; h < (w.wide ? 2 : c + 1); h++, m++) {
          const int k_base = tile + 64 * h;
          const uint32_t sp = tmem_s + (m & 1) * 64;           // S and P of the step
          if (!wait(&bar->s_full[c][m & 1], m >> 1 & 1)) break;
          hb_tc_fence_after();
          const bool cut = k_base < w.e.lo || k_base + 64 > w.e.hi;
          const bool open = MASKED && k_base + 64 > w.e.pos + 1;      // some row does not see all keys (the same steps for both chains of a wide item)
          if (cut || open) {
            if (!wait(&bar->v_full[v_stage], v_parity)) break;
            // the rows of V, of the step's keys, where the item does not reach: a thread has half of one
            const int row = 64 * h + ((threadIdx.x & 127) >> 1);
            if (tile + row < w.e.lo || tile + row >= w.e.hi) {
              const uint32_t dst = hb_smem_u32(sV + v_stage * OPND) + row * 128 + (threadIdx.x & 1) * (D == 128 ? TILE : 64);
#pragma unroll
              for (int q = 0; q < D / 16; q++)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + q * 16), "r"(0) : "memory");
            }
            if (open) {
              const int found = scan_values<D>(sV + v_stage * OPND + 64 * h * 128, &bar->bad[v_stage][2 * h], &bar->scanned[c], scans++ & 1,
                                               max(w.e.lo, w.e.pos + 1) - k_base, w.e.hi - k_base, last_key - k_base, abort_flag);
              if (!(ok = found != 2)) break;
              if (found == 1) l_run = __uint_as_float(0x7fc00000u);
            }
            hb_fence_proxy_async();
          }
          if (!idle) {
            uint32_t x[64];
#pragma unroll
            for (int q = 0; q < 64; q += 32) ld32(sp + q, x + q);
            hb_tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 64; q += 32) ld32_fence(x + q);
            if (cut || k_base + 64 > sure) {
              const int lo_j = w.e.lo - k_base, hi_j = last_key - k_base;
#pragma unroll
              for (int j = 0; j < 64; j++)
                if (j < lo_j || j > hi_j) x[j] = __float_as_uint(-INFINITY);
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 64; j += 2) mx[(j >> 1) & 3] = max_nan(mx[(j >> 1) & 3], __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
            const float m_step = max_nan(max_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale_log2;
            if (!(m_step < INFINITY)) l_run = __uint_as_float(0x7fc00000u);      // a score that is NaN or infinite: so is the row
            const bool grow = m_step > m_run + slack;   // also the first step with a visible key: m_run is -inf
            if (__any_sync(0xffffffffu, grow)) {
              const float m_new = grow ? m_step : m_run, corr = grow ? hb_exp2(m_run - m_new) : 1.f;      // 0 while nothing has been summed
              m_run = m_new;
              l_run *= corr;
              if (m > m0) {       // the rows of O so far
                if (!wait(&bar->pv_done[c][(m - 1) & 1], (m - 1) >> 1 & 1)) break;
                hb_tc_fence_after();
                scale_rows<D>(tmem_o, corr);
              }
            }
            const float sub = m_run == -INFINITY ? 0.f : m_run;
            const uint64_t sub2 = pack2(-sub, -sub);
            uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
            for (int j = 0; j < 64; j += 4) {              // masked scores are -inf: 2^-inf = 0
              float p0, p1, p2, p3;
              const uint64_t t0 = fma2(pack2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), scale2, sub2);
              const uint64_t t1 = fma2(pack2(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])), scale2, sub2);
              if (j % 12 == 0) {       // 6 of 16 groups: the special-function unit has 8 cycles for each of the others (none 150 us, these 143, half of them 148: 384 rows behind 24,560 tokens)
                exp2_poly(t0, p0, p1);
                exp2_poly(t1, p2, p3);
              } else {
                unpack2(t0, p0, p1);
                unpack2(t1, p2, p3);
                p0 = hb_exp2(p0); p1 = hb_exp2(p1); p2 = hb_exp2(p2); p3 = hb_exp2(p3);
              }
              sum2[0] = add2(sum2[0], pack2(p0, p1));
              sum2[1] = add2(sum2[1], pack2(p2, p3));
              // P is rounded to bfloat16, the operand's type; the sum is of the unrounded numbers
              x[j >> 1] = hb_pack_bf16(p0, p1);
              x[(j >> 1) + 1] = hb_pack_bf16(p2, p3);
            }
            st32(sp, x);
            hb_tmem_st_wait();
            float s0, s1, s2, s3;
            unpack2(sum2[0], s0, s1);
            unpack2(sum2[1], s2, s3);
            l_run += (s0 + s1) + (s2 + s3);
          }
          hb_tc_fence_before();
          __syncwarp();
          if (lane == 0) hb_mbar_arrive(&bar->p_full[c][m & 1]);
        }
        if (++v_stage == NV) { v_stage = 0; v_parity ^= 1; }
      }
      if (!ok) break;
      // ---- the item's end: the rows' parts
      const size_t part = (size_t)w.e.part + (w.wide ? c * RT * G : c * rows);
      if (!wait(&bar->pv_done[c][(m - 1) & 1], (m - 1) >> 1 & 1)) break;
      hb_tc_fence_after();
      if (r >= 0 && r < rows) part_ml[part + r] = make_float2(m_run, l_run);
      if (!idle) {
        store_rows<D>(tmem_o, part_o + (part + w4 * 32 - below) * D, rows - (w4 * 32 - below));
        hb_tc_fence_before();
      }
    }
  }

  hb_tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(status, 1);
    __nanosleep(100000);
  }
  if (warp == 10) {
    __syncwarp();
    hb_tmem_dealloc(tmem, 512);
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (EncodeFn)p;
  }
  return fn;
}
// A bfloat16 map with the 128-byte swizzle; strides in bytes of dimension 1 (and 2).
int make_map(CUtensorMap* out, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  EncodeFn fn = encode_fn();
  if (!fn) HB_FAIL("cuTensorMapEncodeTiled is not available from this driver");
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) HB_FAIL("hb_shared_items_tc: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return 0;
}

}  // namespace

// Whether the kernel takes these sizes (whatever they are, rows of q and pages have to lie on 16 bytes).
HB_EXPORT int hb_shared_items_tc_supported(int Hq, int Hkv, int D, int page_size) {
  return Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= ST_ROWS && (D == 64 || D == 128) && page_size >= 8 && page_size <= ST_KEYS &&
         (page_size & (page_size - 1)) == 0;
}

int hb_shared_items_tc(const void* q, long ldq, const void* kc, const void* vc, long num_pages, const int* bt, int bt_stride, const SharedItem* items,
                       const int* cta_items, int ctas, int masked, int T, float* part_o, float2* part_ml, int Hq, int Hkv, int D, int page_size, float scale_log2, int* status, cudaStream_t s) {
  if (!hb_shared_items_tc_supported(Hq, Hkv, D, page_size))
    HB_FAIL("hb_shared_items_tc: %d/%d heads of %d with pages of %d are not supported", Hq, Hkv, D, page_size);
  if (ctas <= 0 || T <= 0) return 0;
  if (!status) HB_FAIL("hb_shared_items_tc: no status word");
  if ((((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15) || (ldq * 2) % 16 || ldq < (long)Hq * D)
    HB_FAIL("hb_shared_items_tc: rows of q and pages have to lie on 16 bytes");
  const long rows = num_pages * Hkv * page_size;
  if (rows > 0x7fffffff) HB_FAIL("hb_shared_items_tc: %ld pages are beyond the maps' limit", num_pages);
  const int G = Hq / Hkv;
  CUtensorMap mq, mk, mv;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)T}, strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(ST_ROWS / G)};
    if (make_map(&mq, q, 3, dims, strides, box)) return -1;
  }
  {
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)D * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)page_size};
    if (make_map(&mk, kc, 2, dims, strides, box) || make_map(&mv, vc, 2, dims, strides, box)) return -1;
  }
  // How far a row's maximum may lie above the reference of its exponentials, as a power of 2. A term of 1 is rounded to bfloat16 without an error, so that
  // a near reference is the more exact one (behind 5,648 tokens 1.18 instead of 1.33 times the error of the output's own rounding), but each
  // new one waits for the product before: 64 users 33 us at 8, 39 at 2. Calls of fewer than 256 rows times heads take as long with either.
  const float slack = (long)T * Hq < 256 ? 1.f : 8.f;
  cudaError_t e = cudaSuccess;
  int dev = -1;
  cudaGetDevice(&dev);
#define ST_LAUNCH(DD, M)                                                                                                                    \
  do {                                                                                                                                      \
    static bool configured[64] = {}; /* the attribute belongs to a device: set once on each */                                              \
    if (dev < 0 || dev >= 64 || !configured[dev]) {                                                                                         \
      e = cudaFuncSetAttribute(shared_items_tc_kernel<DD, M>, cudaFuncAttributeMaxDynamicSharedMemorySize, st_smem<DD>());                  \
      if (e != cudaSuccess) HB_FAIL("hb_shared_items_tc: %s", cudaGetErrorString(e));                                                       \
      if (dev >= 0 && dev < 64) configured[dev] = true;                                                                                     \
    }                                                                                                                                       \
    e = hb_launch(shared_items_tc_kernel<DD, M>, ctas, ST_THREADS, st_smem<DD>(), s, mq, mk, mv, bt, bt_stride, items, cta_items,           \
                  part_o, part_ml, Hkv, G, page_size, scale_log2, slack, status);                                                           \
  } while (0)
  if (D == 64 && masked) ST_LAUNCH(64, true);
  else if (D == 64) ST_LAUNCH(64, false);
  else if (masked) ST_LAUNCH(128, true);
  else ST_LAUNCH(128, false);
#undef ST_LAUNCH
  if (e != cudaSuccess) HB_FAIL("hb_shared_items_tc: %s", cudaGetErrorString(e));
  HB_CHECK_LAUNCH("hb_shared_items_tc");
  return 0;
}
