// Attention over a paged cache in 8 bits on warp MMAs: heads of 64 or 128, pages of whole blocks. Single tokens and short portions, whose time
// is the reading of the cache.
//
// A TILE is up to 8 NT (row, query head) pairs of one request and kv head; a cluster of C blocks has a tile, and their warps take its keys in units
// of 16 places (a block of the cache: one scale for K, one for V), every (4 C)th unit a warp. A warp keeps its own softmax of the units it has
// seen and the warps and blocks are joined at the end, through shared memory and through the cluster's: no workspace, one launch.
//
// Scores are S^T = K Q^T and results O^T = V^T P^T, so that the 16 rows of an MMA are keys (or dimensions) and its 8 columns the pairs: eight
// query heads fill it, where Q as the rows would leave half of it empty. The order of the dimensions within a product is free, and so K's
// operand is what ldmatrix gives of bytes: four codes of key g and of key g + 8 a register. V's needs two keys' codes of one dimension side by side:
// bytes of four loads are interleaved.
//
// A warp's units come by cp.async through a ring of its own in shared memory, two or three units ahead, so that nothing waits for another warp and the
// registers are left to the products: with the units ahead in registers (166 of them, 12 warps an SM) every second stall was for a result of the
// warp's own, and 64 requests of 8,000 tokens (128) took 208 us, 163 now. 16-byte pieces are exchanged within a unit so that the reads of a product's operand
// touch every bank once.
//
// Codes are integers (or e4m3 numbers) of at most 8 significant bits, exact in f16. The query of a pair is scaled by a power of two to below 2^10 and
// split into f16 parts: one holds all of a bf16 query, two hold 22 bits of a 32-bit one. A bf16 query meets int8 keys as they are: it is rounded to
// 16 bits of its pair's largest number, two int8 parts (2^-16 of that number is less than what bf16 keeps of it), whose products with the codes are
// exact in integers; the keys' conversion was a sixth of all instructions. A weight is 2^(score - sub), where sub lies 2 (in base 2) below
// a score that was the largest once and is raised only when a weight passes 2^10, so that raising it, which costs a pass over the accumulators, is
// rare. It is made times its unit's V scale over a reference, that of an earlier unit, which is exchanged (another pass) only where the two are more
// than 2^5 apart: at most 2^15 in f16 (two parts where the rows are 32-bit, the second times 2^12). A weight keeps its bits down to 2^-16 of the largest that its
// warp has seen (2^-28 in two parts); what is less is off by 2^-27 (2^-39) of that one, which counts where nearly all weight is on keys whose values are all but nothing beside the others'. A unit's sum is divided
// by that ratio again. Scales, sums and accumulators are 32-bit.
//
// What bounds it: with many long requests the copy bandwidth (64 of 8,000 tokens, 8 kv heads of 128: 163 us, 6.4 TB/s, 98 % of a copy's; heads of 64 96 us,
// 84 %, with half the issue slots used); with few the chain from the positions to the join (one of 700, heads of 64: 4.4 us within a graph, 5.4 launched by itself; 8 of 2,000: 8.5);
// with several rows a request the warps' own products and softmax (16 of 2,300 with 5 rows each, heads of 64: 18.3 us for 38 MB).
#include "cache8.cuh"
#include "tc_common.cuh"

#include <cuda_fp16.h>


constexpr int C8M_WARPS = 4, C8M_RANKS = 16;     // warps of a block; blocks of a cluster at most

struct C8Attend {
  const void* q;
  long ld_q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  long n_pages;
  int Hkv, upp, upp_log2;      // kv heads, units of a page; -1: no power of two
  const int* bt;
  long ld_table;
  int table_rows, table_width;
  const int* pos;
  const int4* tiles;           // (request, row and query head of a kv head's G of the first pair, pairs); null: row t is request t's, tiles_row tiles each
  int first_tile, tiles_row, G, window;
  uint32_t g_inv;              // 2^32 / G, rounded up
  float scale_log2;
  void* out;
  int q_aligned, out_aligned;
  int beside;                  // the kernel behind this one is cache8_portions_kernel, which does not wait: it may start when this one has waited
};

// D += A B, f16 operands; D = A B without an addend.
__device__ __forceinline__ void c8_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void c8_mma_zero(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t c8_transpose(uint32_t x) {      // an 8 x 8 of f16, two numbers a thread
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Four codes (two pairs) as two f16x2. int8: with the sign bit turned a byte u is code + 128, and f16 0x6400 | u is 1024 + u, exactly.
template <typename CT> __device__ __forceinline__ void c8_halves(uint32_t w, uint32_t& lo, uint32_t& hi);
template <> __device__ __forceinline__ void c8_halves<C8Int8>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 off = __half2half2(__ushort_as_half(0x6480));      // 1152
  const __half2 x = __hsub2(*(const __half2*)&a, off), y = __hsub2(*(const __half2*)&b, off);
  lo = *(const uint32_t*)&x;
  hi = *(const uint32_t*)&y;
}
template <> __device__ __forceinline__ void c8_halves<C8E4m3>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
}

// PARTS numbers of f16 whose sum, the second over TIMES, is x, two x at a time. The second part of a weight comes times 2^12 (and meets its codes over 2^12, exactly): by itself
// it would end where f16 does, and of a weight of 2^-22 of the row's largest neither part kept more than two bits.
template <int PARTS, int TIMES = 1> __device__ __forceinline__ void c8_split(float x, float y, uint32_t* part) {
  __half2 h = __floats2half2_rn(x, y);
  part[0] = *(const uint32_t*)&h;
  if constexpr (PARTS == 2) {
    const float2 f = __half22float2(h);
    h = __floats2half2_rn((x - f.x) * TIMES, (y - f.y) * TIMES);
    part[1] = *(const uint32_t*)&h;
  }
}
constexpr int C8M_TIMES = 4096;

// Products of 32 int8 dimensions.
__device__ __forceinline__ void c8_imma(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void c8_imma_zero(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}

// A unit in shared memory: keys' codes [16][D], then values'. Piece c (16 bytes) of row r lies at: (K is read by ldmatrix, eight rows of a piece
// together; V by pieces, or halves of them, of rows 2 tq.)
template <int D> __device__ __forceinline__ uint32_t c8_at_k(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : (r >> 1) * 128 + (((r & 1) * 4 + (c ^ (r >> 1 & 3))) << 4);
}
template <int D> __device__ __forceinline__ uint32_t c8_at_v(int r, int c) {
  if constexpr (D == 128) return c8_at_k<D>(r, c);
  const int p = (r >> 1) + (r & 1) * 8;                               // the rows that a product reads together stand side by side
  return p * 64 + ((c ^ (p & 2)) << 4);
}
template <int D> __device__ __forceinline__ void c8_fetch(uint32_t stage, const uint8_t* kc, const uint8_t* vc, int at, int lane) {
  const uint8_t *k = kc + (size_t)at * (C8_BLOCK * D), *v = vc + (size_t)at * (C8_BLOCK * D);
#pragma unroll
  for (int j = 0; j < D / 32; j++) {
    const int i = j * 32 + lane, r = i / (D / 16), c = i % (D / 16);
    hb_cp_async16(stage + c8_at_k<D>(r, c), k + i * 16);
    hb_cp_async16(stage + C8_BLOCK * D + c8_at_v<D>(r, c), v + i * 16);
  }
}
__device__ __forceinline__ uint4 c8_lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 c8_lds8(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}

template <typename CT, typename T, int D, int NT> struct C8Sizes {
  static constexpr bool Q_INT = sizeof(T) == 2 && CT::MOST == C8Int8::MOST;                       // the query in int8 parts
  static constexpr int PARTS = sizeof(T) == 4 || Q_INT ? 2 : 1, W_PARTS = sizeof(T) == 4 ? 2 : 1;  // of the query, of the weights
  static constexpr int STEPS = D / 16, Q_STEPS = Q_INT ? D / 32 : D / 16;
  // units of a stage, stages of a ring. 4 KB a stage; one unit of 2 KB at 32 pairs, whose registers two do not fit in (16 requests of 2,300 tokens with 8 rows
  // each, heads of 64: 23.7 us with two, 22.8 with one; at 24 pairs 17.9 and 17.7, and 64 such requests with 5 rows 58 and 64)
  static constexpr int U = D == 128 || NT == 4 ? 1 : 2, STAGES = 3;
  static constexpr bool Q_REGS = NT == 1 && (Q_INT || PARTS == 1);
  static constexpr int QUERY = Q_REGS ? 0 : PARTS * NT * Q_STEPS * 32 * 8, UNIT = 2 * C8_BLOCK * D, RING = C8M_WARPS * STAGES * U * UNIT;
  static constexpr int PITCH = D + 4, JOINED = C8M_WARPS * 8 * NT * PITCH * 4;
  static constexpr int WORK = QUERY + RING > JOINED ? QUERY + RING : JOINED;
  static constexpr int INBOX = 16 * (2 * NT * D + C8M_RANKS), SMEM = WORK + INBOX + INBOX / 2;     // (items of a tile, rounded up for every rank)
  static constexpr int BLOCKS = NT == 1 ? 4 : D == 64 ? (NT == 2 ? 4 : 3) : NT == 2 ? 3 : 2;      // an SM, by registers
};

template <typename CT, typename T, int D, int NT>
__global__ void __launch_bounds__(32 * C8M_WARPS, C8Sizes<CT, T, D, NT>::BLOCKS) cache8_attention_mma_kernel(const C8Attend a) {
  using Z = C8Sizes<CT, T, D, NT>;
  constexpr int PARTS = Z::PARTS, W_PARTS = Z::W_PARTS, STEPS = Z::STEPS, Q_STEPS = Z::Q_STEPS, PAIRS = 8 * NT, PITCH = Z::PITCH, STAGES = Z::STAGES, U = Z::U;
  extern __shared__ __align__(128) uint8_t smem[];
  uint2* q_sh = (uint2*)smem;                                           // [part][nt][step][lane]
  float* o_sh = (float*)smem;                                           // [warp][pair][PITCH], over the query when it is done with
  __shared__ float col_sh[Z::Q_REGS ? 1 : PAIRS];
  __shared__ float2 ml_sh[C8M_WARPS][PAIRS];                            // a warp's bounds and sums
  float4* inbox = (float4*)(smem + Z::WORK);                            // [rank][share]: the parts that this block joins
  float2* inbox_ml = (float2*)(smem + Z::WORK + Z::INBOX);              // and their bounds and sums
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3, h = blockIdx.y;
  const int ranks = gridDim.x, rank = blockIdx.x;
  const auto cluster_wait = [] { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); };
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  hb_pdl_wait();
  if (a.beside) hb_pdl_launch();
  int r, t0, head0, n;                                                  // n pairs, from head0 of row t0 on
  if (a.tiles) {
    const int4 t = a.tiles[a.first_tile + blockIdx.z];
    r = t.x, t0 = t.y, head0 = t.z, n = t.w;
  } else {
    const int z = a.first_tile + blockIdx.z;
    r = t0 = a.tiles_row == 1 ? z : z / a.tiles_row;
    head0 = (z - t0 * a.tiles_row) * PAIRS, n = min(PAIRS, a.G - head0);
  }
  const auto row_of = [&](int pair) { return t0 + (a.G == 1 ? pair : (int)__umulhi(head0 + pair, a.g_inv)); };      // (head0 + pair) / G, below 2^16
  const auto page_of = [&](int unit) { return a.upp_log2 >= 0 ? unit >> a.upp_log2 : unit / a.upp; };
  // all that does not depend on the rows' positions is asked for together with them, and ahead of the cache's units, whose traffic it would have to
  // wait behind (the query asked for after them: 8 requests of 2,000 tokens, 8 kv heads of 64, 9.6 us instead of 8.3): the query, and where all keys are seen the first pages
  const int p_lo = a.pos[t0], p_hi = a.pos[row_of(n - 1)];             // (positions of a request's rows ascend)
  constexpr int BATCH = 32 / U;
  const int id = rank * C8M_WARPS + warp, stride = ranks * C8M_WARPS;
  const bool early = a.window <= 0, known = r >= 0 && r < a.table_rows;
  const int* table = a.bt + r * a.ld_table;
  int early_page = -1;
  if (early && known) {
    const int i = page_of((id + lane / U * stride) * U + lane % U);
    if (i < a.table_width) early_page = table[i];
  }
  int col_hi[NT][2];                                                    // positions of the rows of columns 2 tq, 2 tq + 1
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int i = nt * 8 + 2 * tq + c;
      col_hi[nt][c] = i < n ? a.pos[row_of(i)] : -1;
    }
  using QRaw = std::conditional_t<sizeof(T) == 2, uint2, float4>;       // four numbers
  QRaw q_raw[STEPS];
  const bool q_mine = Z::Q_REGS || warp < NT;                           // each warp has its own query, or a warp 8 pairs for all
  const int q_pair = (Z::Q_REGS ? 0 : warp * 8) + g;                    // pair g of a tile of 8, the dimensions of this thread's codes
  if (q_mine && q_pair < n) {
    const int row = row_of(q_pair);
    const T* p = (const T*)a.q + row * a.ld_q + ((long)h * a.G + head0 + q_pair - (row - t0) * a.G) * D + tq * 4;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      if (a.q_aligned) {
        q_raw[i] = *(const QRaw*)(p + i * 16);
      } else {
        T x[4] = {p[i * 16], p[i * 16 + 1], p[i * 16 + 2], p[i * 16 + 3]};
        memcpy(&q_raw[i], x, sizeof(QRaw));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < STEPS; i++) q_raw[i] = QRaw{};
  }
  // the keys that any of its rows sees, and those that all of them see
  const int window = a.window > 0 ? a.window : 0x7fffffff;
  const int see_lo = max(0, p_lo < window ? 0 : p_lo - window + 1), all_lo = p_hi < window ? 0 : p_hi - window + 1;
  const int u_lo = see_lo / C8_BLOCK;
  const int u_hi = known && p_hi >= 0 ? (int)min((long)(p_hi / C8_BLOCK), (long)a.table_width * a.upp - 1) : -1;

  const uint32_t ring = hb_smem_u32(smem) + Z::QUERY + warp * STAGES * U * Z::UNIT;
  // this warp's stages: U units each, the id-th and every (ranks * WARPS)th from there; a lane looks up one unit of 32, 32 units ahead
  const int first = u_lo / U + id, last = u_hi < 0 ? -1 : u_hi / U;
  const auto has = [&](int i) { return first + i * stride <= last; };   // stage i
  struct Units { int at; float k_scale, v_scale; };
  const auto look = [&](int i) {                                        // stages i .. i + BATCH - 1
    Units x = {-1, 0.f, 0.f};
    const int unit = (first + (i + lane / U) * stride) * U + lane % U;
    if (unit >= u_lo && unit <= u_hi) {
      const int p = page_of(unit), page = early && i == 0 ? early_page : table[p];
      if (page >= 0 && page < a.n_pages) {
        x.at = (page * a.Hkv + h) * a.upp + unit - p * a.upp;
        x.k_scale = a.ks[x.at];
        x.v_scale = a.vs[x.at];
      }
    }
    return x;
  };
  // (V's scales as powers of two only where they are used: nothing waits for them ahead of the units' fetches; of a block that nothing was stored to: 0)
  const auto v_power = [](float s) { return __log2f(fmaxf(s, 1e-37f)); };
  Units now = look(0), next = {-1, 0.f, 0.f};
  if (has(BATCH)) next = look(BATCH);
  const auto fetch = [&](int i, int base, int slot) {                   // stage i, of the BATCH from `base` on or the next
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = __shfl_sync(0xffffffffu, i - base < BATCH ? now.at : next.at, i % BATCH * U + u);
      if (at >= 0 && has(i)) c8_fetch<D>(ring + (slot * U + u) * Z::UNIT, a.kc, a.vc, at, lane);
    }
    hb_cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) fetch(i, 0, i);

  uint2 q_reg[Z::Q_REGS ? PARTS : 1][Z::Q_REGS ? Q_STEPS : 1];
  float col[NT][2];                                                     // of columns 2 tq, 2 tq + 1: score = product * col * the unit's scale
  if (q_mine) {
    const int nt = Z::Q_REGS ? 0 : warp;
    float x[STEPS][4], most = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      if constexpr (sizeof(T) == 2) {
        x[i][0] = __uint_as_float(q_raw[i].x << 16), x[i][1] = __uint_as_float(q_raw[i].x & 0xffff0000u);
        x[i][2] = __uint_as_float(q_raw[i].y << 16), x[i][3] = __uint_as_float(q_raw[i].y & 0xffff0000u);
      } else {
        x[i][0] = q_raw[i].x, x[i][1] = q_raw[i].y, x[i][2] = q_raw[i].z, x[i][3] = q_raw[i].w;
      }
    }
    bool odd = false;
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        most = fmaxf(most, fabsf(x[s][e]));
        odd |= !(fabsf(x[s][e]) <= 3.402823466e38f);
      }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    odd = __shfl_xor_sync(0xffffffffu, (int)odd, 1) | odd;
    odd = __shfl_xor_sync(0xffffffffu, (int)odd, 2) | odd;
    float up, down;
    if constexpr (Z::Q_INT) {
      most = fmaxf(most, 1e-33f);
      up = odd ? 0.f : 32512.f / most, down = a.scale_log2 * (most / 32512.f);
    } else {                                                            // 2^e <= most < 2^(e + 1); the query times 2^(9 - e)
      const int e = max(-100, (int)(__float_as_uint(most) >> 23) - 127);
      up = odd ? 0.f : __uint_as_float((uint32_t)(9 - e + 127) << 23), down = a.scale_log2 * __uint_as_float((uint32_t)(e - 9 + 127) << 23);
    }
    if (odd) down = NAN;                                                // a query that is not finite: its scores are NaN
    const auto keep = [&](int part, int step, uint2 v) {
      if constexpr (Z::Q_REGS) q_reg[part][step] = v;
      else q_sh[((part * NT + nt) * Q_STEPS + step) * 32 + lane] = v;
    };
    {
      if constexpr (Z::Q_INT) {
#pragma unroll
        for (int s = 0; s < Q_STEPS; s++) {
          uint32_t hi[2] = {0u, 0u}, lo[2] = {0u, 0u};
#pragma unroll
          for (int w = 0; w < 2; w++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int n16 = odd ? 0 : __float2int_rn(x[2 * s + w][e] * up), n8 = (n16 + 128) >> 8;
              hi[w] |= (uint32_t)(n8 & 255) << (8 * e);
              lo[w] |= (uint32_t)((n16 - n8 * 256) & 255) << (8 * e);
            }
          keep(0, s, make_uint2(hi[0], hi[1]));
          keep(1, s, make_uint2(lo[0], lo[1]));
        }
      } else {
#pragma unroll
        for (int s = 0; s < Q_STEPS; s++) {
          uint32_t lo[PARTS], hi[PARTS];
          c8_split<PARTS>(odd ? 0.f : x[s][0] * up, odd ? 0.f : x[s][1] * up, lo);
          c8_split<PARTS>(odd ? 0.f : x[s][2] * up, odd ? 0.f : x[s][3] * up, hi);
#pragma unroll
          for (int p = 0; p < PARTS; p++) keep(p, s, make_uint2(lo[p], hi[p]));
        }
      }
    }
    if constexpr (Z::Q_REGS) col[0][0] = __shfl_sync(0xffffffffu, down, 8 * tq), col[0][1] = __shfl_sync(0xffffffffu, down, 8 * tq + 4);
    else if (tq == 0) col_sh[nt * 8 + g] = down;
  }
  if constexpr (!Z::Q_REGS) {
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; nt++) col[nt][0] = col_sh[nt * 8 + 2 * tq], col[nt][1] = col_sh[nt * 8 + 2 * tq + 1];
  }

  float o[STEPS][NT][4], sub[NT][2], most[NT][2], l[NT][2];             // most: the largest exponent of a weight, 10; -inf while there is no score yet
  float v_top = -INFINITY;                                              // the largest of V's scales so far
  float v_ref = 0.f;                                                    // V's reference scale, which o is to be multiplied with, as a power of two
  bool none = true;                                                     // no unit yet
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    sub[nt][0] = sub[nt][1] = l[nt][0] = l[nt][1] = 0.f;
    most[nt][0] = most[nt][1] = -INFINITY;
#pragma unroll
    for (int i = 0; i < STEPS; i++) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
  }

  // the scores of a unit over col and its scale, in 32 bits
  const uint32_t k_lane = c8_at_k<D>((lane >> 3 & 1) * 8 + (lane & 7), lane >> 4);      // ldmatrix: rows 0-7 and 8-15 of a piece, then of the next
  const auto products = [&](uint32_t stage, float (&s)[NT][4]) {
    int si[2][NT][4];                                                   // two chains of products: of int8 parts, or of every second step
    float sf[2][NT][4];
    const auto query = [&](int part, int nt, int step) {
      if constexpr (Z::Q_REGS) return q_reg[part][step];
      else return q_sh[((part * NT + nt) * Q_STEPS + step) * 32 + lane];
    };
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
      uint32_t w[4];                                                    // four codes of keys g and g + 8, and those 16 dimensions on
      hb_ldmatrix_x4(w, (stage + k_lane) ^ (j * 32));
      if constexpr (Z::Q_INT) {
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            const uint2 b = query(p, nt, j);
            if (j == 0) c8_imma_zero(si[p][nt], w, b.x, b.y);
            else c8_imma(si[p][nt], w, b.x, b.y);
          }
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint32_t f[4];
          c8_halves<CT>(w[2 * i], f[0], f[2]);
          c8_halves<CT>(w[2 * i + 1], f[1], f[3]);
#pragma unroll
          for (int p = 0; p < PARTS; p++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const uint2 b = query(p, nt, j * 2 + i);
              if (j == 0 && p == 0) c8_mma_zero(sf[i][nt], f, b.x, b.y);
              else c8_mma(sf[i][nt], f, b.x, b.y);
            }
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 4; c++)
        s[nt][c] = Z::Q_INT ? (float)(si[0][nt][c] * 256 + si[1][nt][c]) : sf[0][nt][c] + sf[1][nt][c];
  };
  // U units side by side in shared memory, whose first place is key0; at < 0: one that is not there
  const auto compute = [&](uint32_t stage, int key0, const int (&at)[U], const float (&k_scale)[U], const float (&v_log2)[U]) {
    float w[U][NT][4];                                                  // scores, then the weights' exponents, then the weights
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (at[u] >= 0) {
        products(stage + u * Z::UNIT, w[u]);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int c = 0; c < 4; c++) w[u][nt][c] = fmaf(w[u][nt][c], col[nt][c & 1] * k_scale[u], -sub[nt][c & 1]);
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) w[u][nt][0] = w[u][nt][1] = w[u][nt][2] = w[u][nt][3] = -INFINITY;
      }
    }
    const bool whole = key0 >= all_lo && key0 + U * C8_BLOCK - 1 <= p_lo;
    if (!whole) {                                                       // not all of it is seen by all rows
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int key = key0 + u * C8_BLOCK + g + (c >> 1) * 8, hi = col_hi[nt][c & 1];
            if (key > hi || hi - key >= window) w[u][nt][c] = -INFINITY;
          }
    }
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float mx = fmaxf(w[0][nt][c], w[0][nt][c + 2]);
#pragma unroll
        for (int u = 1; u < U; u++) mx = fmaxf(mx, fmaxf(w[u][nt][c], w[u][nt][c + 2]));
        raise |= mx > most[nt][c];
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float mx = fmaxf(w[0][nt][c], w[0][nt][c + 2]);
#pragma unroll
          for (int u = 1; u < U; u++) mx = fmaxf(mx, fmaxf(w[u][nt][c], w[u][nt][c + 2]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          if (mx > most[nt][c]) {
            const float up = mx - 2.f, f = most[nt][c] == -INFINITY ? 0.f : hb_exp2(-up);      // 0 while nothing has been summed
            most[nt][c] = 10.f;
            sub[nt][c] += up;
            l[nt][c] *= f;
#pragma unroll
            for (int u = 0; u < U; u++) w[u][nt][c] -= up, w[u][nt][c + 2] -= up;
#pragma unroll
            for (int i = 0; i < STEPS; i++) o[i][nt][c] *= f, o[i][nt][c + 2] *= f;
          }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (at[u] < 0) continue;
      // A scale of less than 2^-60 of the largest counts as that: what it multiplies is then off by 2^-53 of the largest value at most, and o, which is
      // divided by the reference, stays below 2^100 (blocks of zeros have a scale of 1e-30 / M, those that nothing was stored to 0).
      const float v_now = fmaxf(v_log2[u], v_top - 60.f);
      v_top = fmaxf(v_top, v_now);
      float ratio = v_now - v_ref;                                       // of V's scale to the reference
      if (none || !(fabsf(ratio) <= 5.f)) {
        const float f = none ? 0.f : hb_exp2(-ratio);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int i = 0; i < STEPS; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[i][nt][c] *= f;
        v_ref = v_now;
        none = false;
        ratio = 0.f;
      }
      const float back = hb_exp2(-ratio);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int c = 0; c < 4; c++) w[u][nt][c] = hb_exp2(w[u][nt][c] + ratio);
        l[nt][0] = fmaf(w[u][nt][0] + w[u][nt][2], back, l[nt][0]);
        l[nt][1] = fmaf(w[u][nt][1] + w[u][nt][3], back, l[nt][1]);
      }
      uint32_t b[W_PARTS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        uint32_t x[W_PARTS], y[W_PARTS];
        c8_split<W_PARTS, C8M_TIMES>(w[u][nt][0], w[u][nt][1], x);
        c8_split<W_PARTS, C8M_TIMES>(w[u][nt][2], w[u][nt][3], y);
#pragma unroll
        for (int p = 0; p < W_PARTS; p++) b[p][nt][0] = c8_transpose(x[p]), b[p][nt][1] = c8_transpose(y[p]);
      }
      uint32_t v[4][D / 32];                                            // codes of keys 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9: dimensions g D / 8 ..
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 2 * tq + (i >> 1) * 8 + (i & 1);
        const uint32_t from = stage + u * Z::UNIT + C8_BLOCK * D;
        if constexpr (D == 128) {
          const uint4 x = c8_lds16(from + c8_at_v<D>(r, g));
          v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
        } else {
          const uint2 x = c8_lds8(from + c8_at_v<D>(r, g >> 1) + (g & 1) * 8);
          v[i][0] = x.x, v[i][1] = x.y;
        }
        if constexpr (CT::MOST == C8E4m3::MOST) {                       // a place that nobody sees may hold a NaN
          const int key = key0 + u * C8_BLOCK + r;
          if (!whole && (key < see_lo || key > p_hi))
#pragma unroll
            for (int j = 0; j < D / 32; j++) v[i][j] = 0u;
        }
      }
#pragma unroll
      for (int j = 0; j < D / 32; j++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const uint32_t sel = half ? 0x7362 : 0x5140;
          const uint32_t x = __byte_perm(v[0][j], v[1][j], sel), y = __byte_perm(v[2][j], v[3][j], sel);
          uint32_t f[4];
          c8_halves<CT>(x, f[0], f[1]);
          c8_halves<CT>(y, f[2], f[3]);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) c8_mma(o[2 * j + half][nt], f, b[0][nt][0], b[0][nt][1]);
          if constexpr (W_PARTS == 2) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const __half2 z = __hmul2(*(const __half2*)&f[i], __float2half2_rn(1.f / C8M_TIMES));
              f[i] = *(const uint32_t*)&z;
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) c8_mma(o[2 * j + half][nt], f, b[1][nt][0], b[1][nt][1]);
          }
        }
      }
    }
  };

  now.v_scale = v_power(now.v_scale);
#pragma unroll 1
  for (int i = 0, base = 0, slot = 0, ahead = STAGES - 1; has(i); i++) {      // (not unrolled: three times the code was 12 % slower)
    if (i - base == BATCH) {
      base = i;
      now = next;
      now.v_scale = v_power(now.v_scale);
      next = look(base + BATCH);
    }
    hb_cp_async_wait<STAGES - 2>();
    __syncwarp();                                                       // the stage is there for all lanes, and all are done with the one before
    fetch(i + STAGES - 1, base, ahead);
    int at[U];
    float fk[U], fv[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int l = i % BATCH * U + u;
      at[u] = __shfl_sync(0xffffffffu, now.at, l);
      fk[u] = __shfl_sync(0xffffffffu, now.k_scale, l), fv[u] = __shfl_sync(0xffffffffu, now.v_scale, l);
    }
    compute(ring + slot * U * Z::UNIT, (first + i * stride) * U * C8_BLOCK, at, fk, fv);
    ahead = slot;
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  hb_cp_async_wait<0>();

  // What comes next may start on the SMs that are done and load its weights; sooner, its blocks are in this one's way: a decode step of 8 requests of 2,048
  // tokens (16 layers, heads of 64) 0.84 to 0.88 ms, 0.92 with the launch ahead of the wait, 0.88 behind it.
  if (!a.beside) hb_pdl_launch();
  // the warps' results, then the blocks'
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
      l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
      l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
    }
  const float v_scale = none ? 0.f : hb_exp2(v_ref);
  __syncthreads();                                                      // rings and query are read no more
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int pair = nt * 8 + 2 * tq + (c & 1);
      if (g == 0 && c < 2) ml_sh[warp][pair] = make_float2(most[nt][c] == -INFINITY ? -INFINITY : sub[nt][c], l[nt][c]);
      // dimension d = g D / 8 + 2 i + e lies at 16 i + 8 e + g: the lanes of a store in different banks
#pragma unroll
      for (int i = 0; i < STEPS; i++) o_sh[(warp * PAIRS + pair) * PITCH + i * 16 + (c >> 1) * 8 + g] = o[i][nt][c] * v_scale;
    }
  __syncthreads();
  const auto place = [](int d) { return d % (D / 8) / 2 * 16 + d % 2 * 8 + d / (D / 8); };
  const auto factor = [](float m, float mx) { return mx == -INFINITY ? 1.f : hb_exp2(m - mx); };      // (NaN sums without a bound count)
  T* out = (T*)a.out;
  const auto put = [&](int pair, int d, const float (&x)[4], float sum) {
    const int row = row_of(pair);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    T* to = out + ((long)row * a.Hkv * a.G + (long)h * a.G + head0 + pair - (row - t0) * a.G) * D + d;
    if (a.out_aligned) {
      hb_store4(to, make_float4(x[0] * f, x[1] * f, x[2] * f, x[3] * f));
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) to[e] = hb_from_float<T>(x[e] * f);
    }
  };
  // rank r of the cluster ends the items (pair, four dimensions) r * share .. ; the others' parts come into its inbox
  const int items = n * (D / 4), share = (items + ranks - 1) / ranks;
  const float share_inv = __fdividef(1.f, (float)share);               // (i + 1/2) / share is 1/2048 or more off a whole number, its rounding less)
  if (ranks > 1) cluster_wait();                                        // the others have started
  for (int i = tid; i < items; i += 32 * C8M_WARPS) {
    const int pair = i / (D / 4), d = i % (D / 4) * 4;
    float mx = -INFINITY, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < C8M_WARPS; w++) mx = fmaxf(mx, ml_sh[w][pair].x);
#pragma unroll
    for (int w = 0; w < C8M_WARPS; w++) {
      const float2 ml = ml_sh[w][pair];
      const float f = factor(ml.x, mx);
      sum = fmaf(ml.y, f, sum);
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = fmaf(o_sh[(w * PAIRS + pair) * PITCH + place(d + e)], f, x[e]);
    }
    if (ranks == 1) {
      put(pair, d, x, sum);
      continue;
    }
    const int to = (int)(((float)i + 0.5f) * share_inv), at = rank * share + i - to * share;
    uint32_t box = hb_mapa(inbox + at, to), ml = hb_mapa(inbox_ml + at, to);
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(box), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]) : "memory");
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(ml), "f"(mx), "f"(sum) : "memory");
  }
  if (ranks == 1) return;
  hb_cluster_sync();                                                    // (nobody's memory is touched behind it)
  for (int i = tid; i < share && rank * share + i < items; i += 32 * C8M_WARPS) {
    float mx = -INFINITY, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < ranks; c++) mx = fmaxf(mx, inbox_ml[c * share + i].x);
    for (int c = 0; c < ranks; c++) {
      const float2 ml = inbox_ml[c * share + i];
      const float4 y = inbox[c * share + i];
      const float f = factor(ml.x, mx);
      sum = fmaf(ml.y, f, sum);
      x[0] = fmaf(y.x, f, x[0]), x[1] = fmaf(y.y, f, x[1]), x[2] = fmaf(y.z, f, x[2]), x[3] = fmaf(y.w, f, x[3]);
    }
    put((rank * share + i) / (D / 4), (rank * share + i) % (D / 4) * 4, x, sum);
  }
}

template <typename CT, typename T, int D, int NT>
static cudaError_t configure() {                                        // once on each device
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && configured[dev])) return e;
  e = cudaFuncSetAttribute(cache8_attention_mma_kernel<CT, T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C8Sizes<CT, T, D, NT>::SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(cache8_attention_mma_kernel<CT, T, D, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess && dev < 64) configured[dev] = true;
  return e;
}

template <typename CT, typename T, int D, int NT>
static cudaError_t clusters(int ranks, int* n) {
  cudaError_t e = configure<CT, T, D, NT>();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, 1, 1);
  cfg.blockDim = dim3(32 * C8M_WARPS);
  cfg.dynamicSmemBytes = C8Sizes<CT, T, D, NT>::SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(n, cache8_attention_mma_kernel<CT, T, D, NT>, &cfg);
}

template <typename CT, typename T, int D, int NT>
static cudaError_t launch(const C8Attend& a, int tiles, int ranks, cudaStream_t st) {
  constexpr int smem = C8Sizes<CT, T, D, NT>::SMEM;
  cudaError_t e = configure<CT, T, D, NT>();
  if (e != cudaSuccess) return e;
  C8Attend b = a;
  for (int first = 0; first < tiles; first += 65535) {                  // (the grid's limit)
    b.first_tile = first;
    e = hb_launch_cluster(cache8_attention_mma_kernel<CT, T, D, NT>, dim3(ranks, a.Hkv, tiles - first < 65535 ? tiles - first : 65535),
                          dim3(32 * C8M_WARPS), smem, st, dim3(ranks, 1, 1), b);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// e = what the call gives with DD and NN for the sizes d and n.
#define C8_VARIANTS(d, n, ...)                                                                                       \
  do {                                                                                                               \
    if ((d) == 64) {                                                                                                 \
      constexpr int DD = 64;                                                                                         \
      if ((n) == 1) { constexpr int NN = 1; e = __VA_ARGS__; } else if ((n) == 2) { constexpr int NN = 2; e = __VA_ARGS__; } \
      else if ((n) == 3) { constexpr int NN = 3; e = __VA_ARGS__; } else if ((n) == 4) { constexpr int NN = 4; e = __VA_ARGS__; } \
    } else if ((d) == 128) {                                                                                         \
      constexpr int DD = 128;                                                                                        \
      if ((n) == 1) { constexpr int NN = 1; e = __VA_ARGS__; } else if ((n) == 2) { constexpr int NN = 2; e = __VA_ARGS__; } \
      else if ((n) == 3) { constexpr int NN = 3; e = __VA_ARGS__; } else if ((n) == 4) { constexpr int NN = 4; e = __VA_ARGS__; } \
    }                                                                                                                \
  } while (0)

HB_EXPORT int hb_cache8_attention_mma_supported(int Hkv, int page_size, int D, long n_pages) {
  return Hkv >= 1 && Hkv <= 65535 && page_size >= C8_BLOCK && page_size % C8_BLOCK == 0 && (D == 64 || D == 128) &&
         n_pages * Hkv * (page_size / C8_BLOCK) < (1L << 31);
}

// Clusters of `ranks` blocks that the current device holds at once (their blocks share a part of it, so it need not be its blocks by their number).
HB_EXPORT int hb_cache8_attention_mma_clusters(int dt, int ct, int D, int nt, int ranks) {
  int n = 0;
  cudaError_t e = cudaErrorInvalidValue;
  C8_DISPATCH(ct, "hb_cache8_attention_mma_clusters", HB_DISPATCH_1(dt, "hb_cache8_attention_mma_clusters", {
    C8_VARIANTS(D, nt, (clusters<CT, TA, DD, NN>(ranks, &n)));
  }));
  if (e != cudaSuccess) HB_FAIL("hb_cache8_attention_mma_clusters: %s", cudaGetErrorString(e));
  return n;
}

// tiles: n_tiles int4 on the device (C8Attend) of up to 8 nt pairs; null: n_tiles rows of one token each, whose G heads are cut into tiles of 8 nt.
// kc and vc are 16-byte aligned.
HB_EXPORT int hb_cache8_attention_mma(const void* q, int dt, long ld_q, const void* kc, const void* vc, const float* ks, const float* vs, int ct,
                                      long n_pages, int Hkv, int page_size, int D, const int* bt, long ld_table, int table_rows, int table_width,
                                      const int* pos, const int* tiles, int n_tiles, int nt, int ranks, int G, int window,
                                      float scale, void* out, int beside, cudaStream_t st) {
  if (n_tiles <= 0) return 0;
  if (!hb_cache8_attention_mma_supported(Hkv, page_size, D, n_pages) || G < 1 || G > 32767 || nt < 1 || nt > 4 || ranks < 1 || ranks > C8M_RANKS || (((uintptr_t)kc | (uintptr_t)vc) & 15))
    HB_FAIL("hb_cache8_attention_mma: %d kv heads of %d for %d heads each, pages of %d, %d ranks", Hkv, D, G, page_size, ranks);
  const size_t size = dt == HB_F32 ? 4 : 2;
  const int upp = page_size / C8_BLOCK;
  C8Attend a = {q, ld_q, (const uint8_t*)kc, (const uint8_t*)vc, ks, vs, n_pages, Hkv, upp, upp & (upp - 1) ? -1 : __builtin_ctz(upp), bt, ld_table, table_rows,
                table_width, pos, (const int4*)tiles, 0, (G + 8 * nt - 1) / (8 * nt), G, window, (uint32_t)(((1L << 32) + G - 1) / G), scale * 1.4426950408889634f, out,
                !(((uintptr_t)q | ld_q * size) & (4 * size - 1)), !((uintptr_t)out & (4 * size - 1)), beside};
  const int count = tiles ? n_tiles : n_tiles * a.tiles_row;
  cudaError_t e = cudaErrorInvalidValue;
  C8_DISPATCH(ct, "hb_cache8_attention_mma", HB_DISPATCH_1(dt, "hb_cache8_attention_mma", {
    C8_VARIANTS(D, nt, (launch<CT, TA, DD, NN>(a, count, ranks, st)));
  }));
  if (e != cudaSuccess) HB_FAIL("hb_cache8_attention_mma: %s", cudaGetErrorString(e));
  HB_CHECK_LAUNCH("hb_cache8_attention_mma");
  return 0;
}
