// Storing rows into a cache in 8 bits, and reading pages of it back as numbers.
#include "cache8.cuh"

#include <type_traits>

// Rows of K and V [T][Hkv * D] go to the places slot[t] = page * page_size + place, in any order; of several rows for one place the last
// counts. A block (16 places of a page) is taken over by the first row of the call that goes to it: the CTAs of that row look through all
// slots for the others (a block's places are consecutive slots), and each of their warps has one kv head of K or V: it takes the largest |x| of
// the block's rows, a; the block's scale becomes max(a, 1e-30) / M where a row goes to its first place, else the larger of that and what
// it was, and where it grew the block's codes are rounded once more, to r(code * (old / new)); then the rows' codes, r(x * (1 / scale)),
// overwrite theirs. Numbers that are not finite have no part in a; infinities become the largest code, NaN 0. All arithmetic is 32-bit,
// each operation rounded by itself (no contraction), so that a block's bits are a matter of its rows and what it held alone.
//
// What bounds it: few rows, a chain of a few loads (one row, 8 heads of 128, 2.8 us; 64 rows of 64 requests 3.6); many, issue slots (6,000 rows of a prompt 10.9 us,
// 5.6 by bandwidth, 58 % of the slots used). The maximum is taken of the numbers' bits, two of 16 bits at a time, and a block's rows stay in registers.
constexpr int C8S_WARPS = 8, C8S_ROWS = 16, C8S_LOOK = 8;

// E numbers side by side as they are in memory (16 bytes of them, or one), as floats, and as codes to memory.
template <typename T, int E> struct C8Piece {
  using Raw = std::conditional_t<E == 1, T, uint4>;
  static __device__ __forceinline__ void floats(const Raw& r, float* x) {
    if constexpr (E == 1) {
      x[0] = hb_to_float(r);
    } else {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (E == 4) x[i] = __uint_as_float(w[i]);
        else x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  // NaN becomes 0 and what is beyond +-most becomes that; of bf16 the number nearest to it, which is off by 2^-8 of it at most, less than half the
  // step to the code below (1 of 127, or 32 of 448) or above
  static __device__ __forceinline__ uint32_t finite(uint32_t w, uint32_t most) {
    const uint32_t a = w & 0x7fffffffu;
    return a > 0x7f800000u ? 0u : (w ^ a) | min(a, most);
  }
  static __device__ __forceinline__ void finite(Raw& r, float most) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
    const uint32_t m = E == 4 ? __float_as_uint(most) : min((__float_as_uint(most) + 0x8000u) & 0xffff0000u, 0x7f7f0000u);
#pragma unroll
    for (int i = 0; i < 4; i++)
      w[i] = E == 4 ? finite(w[i], m) : finite(w[i] & 0xffff0000u, m) | finite(w[i] << 16, m) >> 16;
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename CT, int E> __device__ __forceinline__ void c8_store(uint8_t* p, const float* x) {
  if constexpr (E == 8) *(uint2*)p = make_uint2(CT::code4(x), CT::code4(x + 4));
  else if constexpr (E == 4) *(uint32_t*)p = CT::code4(x);
  else *p = CT::code(*x);
}

// E numbers are loaded at a time; ITEMS > 0: a lane's numbers of a block (16 rows of D are 32 lanes x ITEMS x E) stay in registers between
// the maximum and the rounding; 0: any D, loaded twice.
template <typename CT, typename T, int E, int ITEMS>
__global__ void __launch_bounds__(32 * C8S_WARPS) cache8_store_kernel(const T* k, const T* v, long ld_k, long ld_v, const int* slot, int n_rows, int rows_cta,
                                                                      int Hkv, int page_size, int D, long n_slots, uint8_t* kc, uint8_t* vc, float* ks,
                                                                      float* vs) {
  __shared__ int win[C8_BLOCK], earlier;
  hb_pdl_launch();
  hb_pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, pair = blockIdx.y * C8S_WARPS + (tid >> 5), h = pair >> 1;
  const bool mine = h < Hkv, is_v = pair & 1;
  const T* x = (is_v ? v : k) + (long)h * D;
  const long ld = is_v ? ld_v : ld_k;
  // rows that are stored and go to another block than the row before, of the CTA's `rows_cta` (at most 31): a lane has a row
  const int t0 = blockIdx.x * rows_cta;
  int lo_mine = -1;                                              // a block's places are slots lo .. lo + places - 1
  {
    const int row = t0 - 1 + lane, s = row >= 0 && lane <= rows_cta && row < n_rows ? slot[row] : -1;
    if (s >= 0 && s < n_slots) lo_mine = s - s % page_size % C8_BLOCK;
  }
  const int lo_before = __shfl_up_sync(0xffffffffu, lo_mine, 1);
  for (uint32_t heads = __ballot_sync(0xffffffffu, lane > 0 && lo_mine >= 0 && lo_mine != lo_before); heads; heads &= heads - 1) {
    const int at_lane = __ffs(heads) - 1, t = t0 - 1 + at_lane, lo = __shfl_sync(0xffffffffu, lo_mine, at_lane);
    const int page = lo / page_size, first = lo % page_size, places = min(C8_BLOCK, page_size - first);
    __syncthreads();
    if (tid < C8_BLOCK) win[tid] = -1;
    if (tid == C8_BLOCK) earlier = 0;
    __syncthreads();
    for (int i0 = tid; i0 < n_rows; i0 += C8S_LOOK * 32 * C8S_WARPS) {      // (asked for eight at a time: one by one, 6,000 rows took 44 us)
      int s_of[C8S_LOOK];
#pragma unroll
      for (int j = 0; j < C8S_LOOK; j++) s_of[j] = i0 + j * 32 * C8S_WARPS < n_rows ? slot[i0 + j * 32 * C8S_WARPS] : -1;
#pragma unroll
      for (int j = 0; j < C8S_LOOK; j++) {
        const unsigned place = (unsigned)(s_of[j] - lo);
        if (place < (unsigned)places) {
          const int i = i0 + j * 32 * C8S_WARPS;
          if (i < t) earlier = 1;
          atomicMax(&win[place], i);
        }
      }
    }
    __syncthreads();
    if (earlier) continue;                                       // (uniform; the next round's first barrier is behind every read)
    if (!mine) continue;
    uint8_t* at = (is_v ? vc : kc) + ((long)page * Hkv + h) * page_size * D + (long)first * D;
    float* scale = (is_v ? vs : ks) + ((long)page * Hkv + h) * c8_blocks(page_size) + first / C8_BLOCK;
    const bool fresh = win[0] >= 0;
    const float old = fresh ? 0.f : *scale;
    const int pieces = D / E, items = places * pieces;           // piece i: place i / pieces, numbers i % pieces * E ..
    using Piece = C8Piece<T, E>;
    using Raw = typename Piece::Raw;
    Raw kept[ITEMS ? ITEMS : 1];
    float most = 0.f;
    const auto largest = [&](const Raw& r) {                     // of the finite ones
      float y[E];
      Piece::floats(r, y);
#pragma unroll
      for (int e = 0; e < E; e++)
        if (fabsf(y[e]) <= 3.402823466e38f) most = fmaxf(most, fabsf(y[e]));
    };
    bool odd = false;                                            // some of the numbers kept are not finite
    const auto load = [&](int i) { return *(const Raw*)(x + win[i / pieces] * ld + i % pieces * E); };
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int j = 0; j < ITEMS; j++) {
        kept[j] = Raw{};
        if (win[(j * 32 + lane) / pieces] >= 0) kept[j] = load(j * 32 + lane);
      }
      // the largest |x| by its bits, of 16-bit numbers two at a time; only where one is not finite are they looked at one by one
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < ITEMS; j++) {
        const uint32_t w[4] = {kept[j].x, kept[j].y, kept[j].z, kept[j].w};
#pragma unroll
        for (int i = 0; i < 4; i++) bits = sizeof(T) == 4 ? max(bits, w[i] & 0x7fffffffu) : __vmaxu2(bits, w[i] & 0x7fff7fffu);
      }
      if (sizeof(T) == 2) bits = max(bits & 0xffff0000u, bits << 16);
      bits = __reduce_max_sync(0xffffffffu, bits);
      odd = bits >= 0x7f800000u;
      most = __uint_as_float(bits);
      if (odd) {
        most = 0.f;
#pragma unroll
        for (int j = 0; j < ITEMS; j++) largest(kept[j]);
        most = hb_warp_max(most);
      }
    } else {
      for (int i = lane; i < items; i += 32)
        if (win[i / pieces] >= 0) largest(load(i));
      most = hb_warp_max(most);
    }
    float now = __fdiv_rn(fmaxf(most, C8_LEAST), CT::MOST);
    if (!fresh && now > old) {
      const float f = __fdiv_rn(old, now);
      using Codes = std::conditional_t<E == 8, uint2, std::conditional_t<E == 4, uint32_t, uint8_t>>;
      const auto again = [&](int i, const Codes& c) {
        float z[E];
        if constexpr (E == 8) CT::values4(c.x, z), CT::values4(c.y, z + 4);
        else if constexpr (E == 4) CT::values4(c, z);
        else z[0] = CT::value(c);
#pragma unroll
        for (int e = 0; e < E; e++) z[e] = __fmul_rn(z[e], f);
        c8_store<CT, E>(at + (long)i * E, z);
      };
      if constexpr (ITEMS > 0) {
        constexpr int AHEAD = ITEMS < 8 ? ITEMS : 8;             // asked for before the first is used
#pragma unroll 1
        for (int j = 0; j < ITEMS; j += AHEAD) {
          Codes c[AHEAD];
#pragma unroll
          for (int n = 0; n < AHEAD; n++) c[n] = *(const Codes*)(at + ((j + n) * 32 + lane) * E);
#pragma unroll
          for (int n = 0; n < AHEAD; n++)
            if (win[((j + n) * 32 + lane) / pieces] < 0) again((j + n) * 32 + lane, c[n]);
        }
      } else {
        for (int i = lane; i < items; i += 32)
          if (win[i / pieces] < 0) again(i, at[i]);
      }
    } else if (!fresh) {
      now = old;
    }
    if (lane == 0) *scale = now;
    const float inv = __fdiv_rn(1.f, now);
    if constexpr (ITEMS > 0)
      if (odd) {
#pragma unroll
        for (int j = 0; j < ITEMS; j++) Piece::finite(kept[j], fminf(__fmul_rn(now, CT::MOST), 3.402823466e38f));
      }
    const auto put = [&](int i, const Raw& r) {
      float y[E], z[E];
      Piece::floats(r, y);
#pragma unroll
      for (int e = 0; e < E; e++) {
        z[e] = __fmul_rn(y[e], inv);
        // (numbers kept are finite by now, and no more than a rounding beyond the largest code, which they become)
        if constexpr (ITEMS == 0) z[e] = z[e] != z[e] ? 0.f : fminf(fmaxf(z[e], -CT::MOST), CT::MOST);
      }
      c8_store<CT, E>(at + (long)i * E, z);
    };
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int j = 0; j < ITEMS; j++)
        if (win[(j * 32 + lane) / pieces] >= 0) put(j * 32 + lane, kept[j]);
    } else {
      for (int i = lane; i < items; i += 32)
        if (win[i / pieces] >= 0) put(i, load(i));
    }
  }
}

// ct: HB_I8 or HB_E4M3; dt: the rows' type. n_pages * page_size places; slots outside of them (negative ones among them) store nothing.
HB_EXPORT int hb_cache8_store(const void* k, const void* v, long ld_k, long ld_v, int dt, const int* slot, int n_rows, int Hkv, int page_size,
                              int D, long n_pages, int ct, void* kc, void* vc, float* ks, float* vs, cudaStream_t st) {
  if (n_rows <= 0) return 0;
  if (Hkv < 1 || Hkv > 65535 || page_size < 1 || D < 1 || n_pages * page_size > 0x7fffffffL)
    HB_FAIL("hb_cache8_store: %d kv heads of %d, %ld pages of %d", Hkv, D, n_pages, page_size);
  const size_t size = dt == HB_F32 ? 4 : 2;
  // 16 bytes of a row at a time
  const bool wide = (D == 64 || D == 128) && page_size % C8_BLOCK == 0 &&
                    !(((uintptr_t)k | (uintptr_t)v | ld_k * size | ld_v * size | (uintptr_t)kc | (uintptr_t)vc) & 15);
  // a row a CTA while those that have nothing to do are few, else as many as a block has places
  const int rows_cta = n_rows <= 512 ? 1 : C8S_ROWS;
  const dim3 grid((n_rows + rows_cta - 1) / rows_cta, (2 * Hkv + C8S_WARPS - 1) / C8S_WARPS);
#define C8S_LAUNCH(E, ITEMS)                                                                                                                        \
  hb_launch(cache8_store_kernel<CT, TA, E, ITEMS>, grid, dim3(32 * C8S_WARPS), 0, st, (const TA*)k, (const TA*)v, ld_k, ld_v, slot, n_rows, rows_cta, \
            Hkv, page_size, D, n_pages * page_size, (uint8_t*)kc, (uint8_t*)vc, ks, vs)
  C8_DISPATCH(ct, "hb_cache8_store", HB_DISPATCH_1(dt, "hb_cache8_store", {
    constexpr int E = 16 / sizeof(TA);
    if (wide && D == 64) C8S_LAUNCH(E, 64 / (2 * E));
    else if (wide) C8S_LAUNCH(E, 128 / (2 * E));
    else C8S_LAUNCH(1, 0);
  }));
#undef C8S_LAUNCH
  HB_CHECK_LAUNCH("hb_cache8_store");
  return 0;
}

// Page i of the output [n][Hkv][page_size][D] is page table[i] of the cache; a number outside of the
// cache's pages gives zeros. E codes at a time: 8 of them are a load of 8 bytes and a store of 16 (bf16) or two, so that a warp's stores are
// whole lines; a page of one plane is a block's, or a few blocks' where pages are few. Bound by
// bandwidth where pages are many (4,000 pages of 8 heads of 128 66 us, 60 by a copy's; 380 8.2, of 5.7), else by one round of loads (64 pages 3.1 us).
constexpr int C8E_AHEAD = 4;      // pieces that a thread asks for before it uses the first
// CTAs that share `pieces` of 8 bytes: one piece a thread while there are few of them, all of them one CTA's when they are many (64 pages of 8 heads of
// 128 3.1 us, with one CTA a page and plane 4.6; 4,000 pages 66 us either way). A thread's numbers of pieces end less than C8E_BEYOND behind the last.
constexpr int C8E_SPLIT = 64, C8E_BEYOND = C8E_SPLIT * 256 * (C8E_AHEAD + 1);
static int c8_split(long ctas, long pieces) {
  const long most = (pieces + 255) / 256, room = 8L * 148 / ctas;
  return (int)(room < 1 ? 1 : room < most ? (room < C8E_SPLIT ? room : C8E_SPLIT) : most < C8E_SPLIT ? most : C8E_SPLIT);
}
template <typename CT, typename T, int E>
__global__ void __launch_bounds__(256) cache8_expand_kernel(const uint8_t* kc, const uint8_t* vc, const float* ks, const float* vs, const int* table,
                                                            long n_pages, int Hkv, int page_size, int D, T* k, T* v) {
  hb_pdl_launch();
  hb_pdl_wait();
  const long i = blockIdx.x;
  const bool is_v = blockIdx.y;
  const int step = gridDim.z * 256;
  const int pieces = Hkv * page_size * D / E, row_pieces = D / E, blocks = c8_blocks(page_size);
  const bool whole = page_size % C8_BLOCK == 0;
  T* out = (is_v ? v : k) + i * pieces * E;
  const long page = table[i];
  const bool there = page >= 0 && page < n_pages;
  const uint8_t* codes = (is_v ? vc : kc) + (there ? page : 0) * pieces * E;
  const float* scales = (is_v ? vs : ks) + (there ? page : 0) * Hkv * blocks;
  for (int j0 = blockIdx.z * 256 + threadIdx.x; j0 < pieces; j0 += C8E_AHEAD * step) {
    uint2 w[C8E_AHEAD];
    float f[C8E_AHEAD];
#pragma unroll
    for (int k = 0; k < C8E_AHEAD; k++) {
      const int j = j0 + k * step;
      w[k] = make_uint2(0u, 0u), f[k] = 0.f;
      if (there && j < pieces) {
        if constexpr (E == 8) w[k] = *(const uint2*)(codes + (long)j * E);
        else w[k].x = codes[j];
        const int row = j / row_pieces;                          // of the page's rows, head by head
        f[k] = scales[whole ? row / C8_BLOCK : row / page_size * blocks + row % page_size / C8_BLOCK];
      }
    }
#pragma unroll
    for (int k = 0; k < C8E_AHEAD; k++) {
      const int j = j0 + k * step;
      if (j >= pieces) break;
      if constexpr (E == 8) {
        float x[8];
        CT::values4(w[k].x, x);
        CT::values4(w[k].y, x + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = there ? x[e] * f[k] : 0.f;
        if constexpr (sizeof(T) == 4) {
          *(float4*)(out + (long)j * E) = make_float4(x[0], x[1], x[2], x[3]);
          *(float4*)(out + (long)j * E + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
          __nv_bfloat162 y[4];
#pragma unroll
          for (int e = 0; e < 4; e++) y[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
          *(uint4*)(out + (long)j * E) = *(const uint4*)y;
        }
      } else {
        out[j] = hb_from_float<T>(there ? CT::value((uint8_t)w[k].x) * f[k] : 0.f);
      }
    }
  }
}

HB_EXPORT int hb_cache8_expand(const void* kc, const void* vc, const float* ks, const float* vs, int ct, const int* table, long n, long n_pages,
                               int Hkv, int page_size, int D, void* k, void* v, int dt, cudaStream_t st) {
  if (n <= 0) return 0;
  if (n > 0x7fffffffL || Hkv < 1 || page_size < 1 || D < 1 || (long)Hkv * page_size * D > 0x7fffffffL - C8E_BEYOND || n_pages < 1)
    HB_FAIL("hb_cache8_expand: %ld of %ld pages of %d heads, %d places and %d", n, n_pages, Hkv, page_size, D);
  const bool wide = D % 8 == 0 && !(((uintptr_t)kc | (uintptr_t)vc) & 7) && !(((uintptr_t)k | (uintptr_t)v) & 15);
#define C8E_LAUNCH(E)                                                                                                                                   \
  hb_launch(cache8_expand_kernel<CT, TA, E>, dim3(n, 2, c8_split(2 * n, (long)Hkv * page_size * D / E)), dim3(256), 0, st, (const uint8_t*)kc,            \
            (const uint8_t*)vc, ks, vs, table, n_pages, Hkv, page_size, D, (TA*)k, (TA*)v)
  C8_DISPATCH(ct, "hb_cache8_expand", HB_DISPATCH_1(dt, "hb_cache8_expand", {
    if (wide) C8E_LAUNCH(8);
    else C8E_LAUNCH(1);
  }));
#undef C8E_LAUNCH
  HB_CHECK_LAUNCH("hb_cache8_expand");
  return 0;
}

// What the flash kernel for portions wants of a cache: the codes of pages table[index[i]] as bf16, which holds them exactly, and the scales of
// their blocks, scale[h][C8_AHEAD + i * blocks + block] of n * blocks and C8_AHEAD on either side: {K's times `scale_log2`, log2 of V's, 1 / V's, 0}, K's negative where
// the page is not there. A weight is made times its value's scale and in bf16, so that a scale near the least (a block of zeros has 1e-30 / M) would lose all weights
// but the largest, and one near the greatest would leave the type: outside of 2^-60 .. 2^60 a scale comes times 2^60 or 2^-60 and the block's codes the other way,
// exactly. Where a scale is 0 (a block that nothing was stored to) or not a number it is 1 and the codes are 0 (0 times a masked score is not a number); places that nothing
// was stored to may hold anything, and so codes that are not numbers become 0; what lies on either side, for tiles that reach over a request's ends, are ones.
//
// `beside`: the kernel ahead is cache8_attention_mma_kernel for a step's other rows, which lets this one start when it has itself waited for what came
// before it: the cache is as this kernel wants it, and the two run side by side (a step of two portions and four single rows 7 us of 119). Its 380 pages of 8 heads of
// 128 take 8 us; with a page's work shared by blocks it took the single rows' blocks their place (104 us the step, 108). This
// kernel still does not end before that one has.
constexpr int C8_AHEAD = 32;
struct C8Shifted {
  float scale, codes;          // what a block's scale and its codes are multiplied with
};
__device__ __forceinline__ C8Shifted c8_shifted(float s) {
  constexpr float UP = 1.152921504606846976e18f;                 // 2^60
  if (!(s > 0.f && s <= 3.402823466e38f)) return {0.f, 0.f};
  return s < 1.f / UP ? C8Shifted{UP, 1.f / UP} : s > UP ? C8Shifted{1.f / UP, UP} : C8Shifted{1.f, 1.f};
}
template <typename CT>
__global__ void __launch_bounds__(256) cache8_portions_kernel(const uint8_t* kc, const uint8_t* vc, const float* ks, const float* vs, const int* table,
                                                              const int* index, long n, long n_pages, int Hkv, int page_size, int D, float scale_log2,
                                                              __nv_bfloat16* k, __nv_bfloat16* v, float4* scale, bool beside) {
  hb_pdl_launch();
  if (!beside) hb_pdl_wait();
  const long i = blockIdx.x;
  const int blocks = c8_blocks(page_size);
  const long ld = n * blocks + 2 * C8_AHEAD;
  const int step = gridDim.y * 256;
  if (i == n) {
    if (blockIdx.y == 0)
      for (int j = threadIdx.x; j < Hkv * 2 * C8_AHEAD; j += 256) {
        const int at = j % (2 * C8_AHEAD);
        scale[j / (2 * C8_AHEAD) * ld + (at < C8_AHEAD ? at : n * blocks + at)] = make_float4(1.f, 0.f, 1.f, 0.f);
      }
    if (beside) hb_pdl_wait();
    return;
  }
  const long page = table[index[i]];
  const bool there = page >= 0 && page < n_pages;
  const int pieces = Hkv * page_size * D / 8, block_log2 = D == 64 ? 7 : 8;      // 2^block_log2 pieces of a block, 2 D
  // whether some block of the page has a scale that comes times something: looked up once for all (asked for with every piece a step took 4 us more, of 102)
  bool odd = false;
  for (int j = threadIdx.x; there && j < 2 * Hkv * blocks; j += 256)
    odd |= c8_shifted((j >= Hkv * blocks ? vs : ks)[page * Hkv * blocks + (j >= Hkv * blocks ? j - Hkv * blocks : j)]).codes != 1.f;
  odd = __syncthreads_or(odd);
  for (int j0 = blockIdx.y * 256 + threadIdx.x; j0 < 2 * pieces; j0 += C8E_AHEAD * step) {
    uint2 w[C8E_AHEAD];
#pragma unroll
    for (int u = 0; u < C8E_AHEAD; u++) {
      const int j = j0 + u * step;
      w[u] = there && j < 2 * pieces ? *(const uint2*)((j >= pieces ? vc : kc) + (page * pieces + (j >= pieces ? j - pieces : j)) * 8L) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < C8E_AHEAD; u++) {
      const int j = j0 + u * step;
      if (j >= 2 * pieces) break;
      float x[8];
      CT::values4(w[u].x, x);
      CT::values4(w[u].y, x + 4);
      __nv_bfloat162 y[4];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = there && x[e] == x[e] ? x[e] : 0.f;
      if (odd) {
        const float times = c8_shifted((j >= pieces ? vs : ks)[page * Hkv * blocks + ((j >= pieces ? j - pieces : j) >> block_log2)]).codes;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= times;
      }
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
      *(uint4*)((j >= pieces ? v : k) + (i * pieces + (j >= pieces ? j - pieces : j)) * 8L) = *(const uint4*)y;
    }
  }
  for (int j = blockIdx.y * 256 + threadIdx.x; j < Hkv * blocks; j += step) {
    const auto number = [](float s) {
      const C8Shifted f = c8_shifted(s);
      return f.scale == 0.f ? 1.f : s * f.scale;
    };
    // (K's stays above 0 whatever the softmax's scale: it multiplies masked scores, which are infinite)
    const float x = there ? fmaxf(number(ks[page * Hkv * blocks + j]) * scale_log2, 1.17549435e-38f) : -1.f, y = there ? number(vs[page * Hkv * blocks + j]) : 1.f;
    scale[j / blocks * ld + C8_AHEAD + i * blocks + j % blocks] = make_float4(x, log2f(y), 1.f / y, 0.f);
  }
  if (beside) hb_pdl_wait();
}

// scale: 4 floats x Hkv x (n * blocks of a page + 2 C8_AHEAD), 16-byte aligned as k and v are; kc, vc 8-byte aligned; D 64 or 128, pages of whole
// blocks, as the flash kernel takes them.
HB_EXPORT int hb_cache8_portions(const void* kc, const void* vc, const float* ks, const float* vs, int ct, const int* table, const int* index, long n,
                                 long n_pages, int Hkv, int page_size, int D, float scale, void* k, void* v, void* scales, int beside,
                                 cudaStream_t st) {
  if (n <= 0) return 0;
  if (n >= 0x7fffffffL || Hkv < 1 || page_size < 1 || page_size % C8_BLOCK || (D != 64 && D != 128) || 2L * Hkv * page_size * D > 0x7fffffffL - C8E_BEYOND || n_pages < 1)
    HB_FAIL("hb_cache8_portions: %ld of %ld pages of %d heads, %d places and %d", n, n_pages, Hkv, page_size, D);
  C8_DISPATCH(ct, "hb_cache8_portions",
      hb_launch(cache8_portions_kernel<CT>, dim3(n + 1, beside ? 1 : c8_split(n + 1, 2L * Hkv * page_size * D / 8)), dim3(256), 0, st, (const uint8_t*)kc, (const uint8_t*)vc, ks, vs, table, index, n, n_pages, Hkv,
                page_size, D, scale * 1.4426950408889634f, (__nv_bfloat16*)k, (__nv_bfloat16*)v, (float4*)scales, beside != 0));
  HB_CHECK_LAUNCH("hb_cache8_portions");
  return 0;
}
