// Decode attention over the 8-bit cache (e4m3 rows with a power of two each, see e4m3.cuh) on tcgen05, the rows as operands
// straight from their pages.
//
// One new token per sequence; scores s_j = q . k_j * scale over the visible positions, softmax, weighted sum of the values
// (models/llm/forward.go:258-278, with rows that take hd + 1 bytes instead of 2 hd).  With k_j = K_j 2^a_j and
// v_j = V_j 2^b_j, K and V being the stored e4m3 numbers, per query head and tile of 128 keys:
//
//   s_j = (K_j . q') * 2^a_j * (scale log2(e) 2^c)      q' = q / 2^c, its largest number in [2^7, 2^8)
//   p_j = 2^(s_j - m),  l = sum_j p_j                   m = the running maximum of s_j, rounded up to a whole number
//   w_j = 2^(s_j + b_j - n + 8),  O' = sum_j w_j V_j    n = the tile's maximum of s_j + b_j, rounded up: w_j <= 2^8
//   O = O 2^(n_before - N) + O' 2^(n - N)               N = the running maximum of n
//   out = O 2^(N - 8 - m) / l
//
// Both products have e4m3 on both sides.  The other operand enters as several e4m3 terms in columns of their own: a query as
// x = x1 + x2 / 16, which holds a bfloat16 number whole down to 2^-22 of the row's largest (each term keeps 4 bits, and what
// the first leaves over is at most 2^-4 of it); a weight as w1 + w2 / 16 (+ w3 / 256 where a block has four heads at most):
// 2^-8 (2^-12) of its size, and of the tile's largest weight 2^-22 (2^-26).  The values' powers are part of the weights, so a
// row of small values may hold all of the softmax's weight without a loss; and because every tile has a reference of its
// own, neither does a long tail of small weights behind a large one.
//
// Bound by the rows, which are read once.  The keys (of the scores) and the numbers of a head (of the output) are the
// MMA's rows and the query heads of a kv head, times their terms, its 16 columns, so no thread touches a row: per tile
// a thread handles one key's scores.  (With mma.sync, whose operands are at least 16 bits wide, converting the rows and the
// scores' arithmetic took 424 instructions per 32 keys and warp: 32 sequences of 256 to 4,096 keys, heads of 128, 35.2 us.)
//   warp 0     TMA: two pages of keys and of values per tile, and their scale bytes, into rings
//   warp 1     tcgen05.mma: scores (keys x 16) one tile ahead, output (numbers x 16); values as the MN-major operand from the
//              page layout [key][number], weights MN-major as the threads write them, 16 bytes a key
//   warps 2-5  a thread per key: scores, maxima over the tile (redux and a barrier), weights; then, a thread per number of a
//              head, the output of the tile before
// Two such blocks share an SM (three with heads of 64), so one's chain of steps runs under the other's.
//
// Work is shared evenly: the tiles of all sequences and kv heads are numbered through, head by head and sequence by sequence,
// and every block takes an equal run of them, as many blocks as are resident at once: all SMs stream until the end, whatever
// the lengths.  What blocks share, at most the first and the last sequence of each, goes through scratch memory, and the block
// that takes a sequence's last ticket adds the parts up in the order of the blocks; nobody waits for another block.
#include <math.h>

#include "common.cuh"
#include "e4m3.cuh"
#include "tcgen05.cuh"

namespace dlgo {

using namespace sm100;

constexpr int DE_THREADS = 192;
constexpr int DE_SOFT = 128;          // of them, warps 2-5
constexpr int DE_TK = 128;            // keys of a tile: two pages
constexpr int DE_GM = 8;              // query heads of a kv head per block at most
constexpr int DE_MIN_TILES = 2;       // a block's least run
constexpr int DE_MAX_B = 512;         // sequences of a launch (their first tiles, positions and slots lie in shared memory)
constexpr int DE_SC = 4;              // tiles whose scale bytes are on their way or in use

template <int HD> constexpr int de_kst = 3;                          // tiles of keys, of values in shared memory
template <int HD> constexpr int de_vst = HD <= 64 ? 3 : 2;
template <int HD> constexpr int de_blocks = HD <= 64 ? 3 : 2;        // blocks on an SM

// Set when a bounded wait ran out: the launch's results are invalid (dlgo_attention_decode_e4m3_error).
__device__ int g_decode_e4m3_error = 0;

struct DecE8 {
  const __nv_bfloat16* q;  // [B][ldq]
  int ldq;
  const uint8_t* kscales;  // [pages][Hkv][64]
  const uint8_t* vscales;
  const int* page_table;   // [slots][max_pages]
  int n_slots, max_pages, n_pages;
  const int* seq_slot;     // [B]
  const int* token_pos;    // [B] position of the new token (its row is in the cache); -1: nothing to see, zeros come out
  __nv_bfloat16* out;      // [B][ldo]
  int ldo, B, Hq, Hkv, n_gchunks, span;
  float scale_log2e;
  const float* sink;       // [Hq] or null: exp(sink) joins the denominator
  float* part_acc;         // [blocks][2][GM][HD]
  float* part_ml;          // [blocks][2][GM][2]
  int* tickets;            // [B][heads], zero between launches
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x for a whole x; below -126: 0
__device__ __forceinline__ float exp2_whole(float x) { return __int_as_float(max((int)fmaxf(x, -127.f) + 127, 0) << 23); }
__device__ __forceinline__ uint32_t bf16_word(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float warp_max_redux(float x) {     // (a NaN does not count)
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// two e4m3 numbers back as fp32
__device__ __forceinline__ float2 e4m3_back(uint32_t pair) {
  const uint32_t h = e4m3_low_half2(pair);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Operand descriptors.  Rows of HD bytes as TMA leaves them: 128-byte swizzle for heads of 128, 64-byte swizzle for heads of 64;
// eight rows are HD * 8 bytes, as the K-major operand (keys, queries) and as the MN-major one (values).
template <int HD> __device__ __forceinline__ uint64_t desc_rows(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(HD * 8 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)(HD == 128 ? 2 : 4) << 61;
}
// The weights, MN-major without a swizzle: 16 columns' bytes a key, keys 16 bytes apart, eight keys 128 bytes.
__device__ __forceinline__ uint64_t desc_weights(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(2048 >> 4) << 32 | (uint64_t)1 << 46;
}
// e4m3 x e4m3 -> fp32, M x N; bits 15 and 16: A and B are MN-major
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N, bool mn) {
  return (1u << 4) | (mn ? 3u << 15 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// A tile of the run: virtual head (kv head and chunk of its query heads), sequence, tile k of its nk.
struct DecPlace {
  int head, b, k, nk;
};

// Shared memory: rings of keys and of values, two buffers of queries and of weights, scale bytes, barriers, ... , sequences
template <int HD> constexpr int de_off_q = (de_kst<HD> + de_vst<HD>) * DE_TK * HD;
template <int HD> constexpr int de_off_p = de_off_q<HD> + 2 * 16 * HD;
template <int HD> constexpr int de_off_sc = de_off_p<HD> + 2 * 2048;
template <int HD> constexpr int de_off_bars = de_off_sc<HD> + DE_SC * 256;
template <int HD> constexpr int de_off_red = de_off_bars<HD> + 256;             // [2][4][2][GM] floats
template <int HD> constexpr int de_off_misc = de_off_red<HD> + 2 * 4 * 2 * DE_GM * 4;    // row scales [2][GM], sums [4][GM], words
template <int HD> constexpr int de_off_seq = de_off_misc<HD> + 6 * DE_GM * 4 + 64;
template <int HD> constexpr size_t de_smem(int B) { return de_off_seq<HD> + (size_t)(4 * B + 1) * 4; }

template <int HD, int GM>
__global__ void __launch_bounds__(DE_THREADS, de_blocks<HD>)
attention_decode_e4m3_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, DecE8 p) {
  constexpr int TERMS = GM <= 4 ? 3 : 2;
  constexpr int KST = de_kst<HD>, VST = de_vst<HD>, STAGE = DE_TK * HD, PAGE_BYTES = E8_PAGE * HD;
  constexpr uint32_t TMEM_COLS = 64, O_COL = 32;      // scores in columns 0 and 16, outputs in 32 and 48
  constexpr int H4 = HD / 4;
  // the swizzled tiles want 1024-byte alignment (checked: a misaligned start ends the kernel with the error word set)
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicExch(&g_decode_e4m3_error, 1);
    return;
  }
  uint8_t* k_s = smem;
  uint8_t* v_s = k_s + KST * STAGE;
  uint8_t* q_s = smem + de_off_q<HD>;                 // [2][16 rows][HD], swizzled as the keys
  uint8_t* p_s = smem + de_off_p<HD>;                 // [2][128 keys][16]
  uint8_t* sc_s = smem + de_off_sc<HD>;               // [DE_SC][keys 128 | values 128]
  uint64_t* bars = (uint64_t*)(smem + de_off_bars<HD>);
  uint64_t* kfull = bars;                // KST
  uint64_t* kempty = bars + 3;           // KST: the scores that read these keys have completed
  uint64_t* vfull = bars + 6;            // VST
  uint64_t* vempty = bars + 9;           // VST: the output that read these values has completed
  uint64_t* sc_full = bars + 12;         // DE_SC
  uint64_t* sc_empty = bars + 16;        // DE_SC
  uint64_t* s_full = bars + 20;          // 2: scores
  uint64_t* s_free = bars + 22;          // 2: ... are in registers
  uint64_t* p_full = bars + 24;          // 2: weights
  uint64_t* o_full = bars + 26;          // 2: the output of a tile (its weights may be overwritten)
  uint64_t* o_free = bars + 28;          // 2: ... is in registers
  uint64_t* q_full = bars + 30;          // 2
  float* red_s = (float*)(smem + de_off_red<HD>);
  float* fs_s = (float*)(smem + de_off_misc<HD>);     // [2][DE_GM] row scales
  float* l_s = fs_s + 2 * DE_GM;                      // [4][DE_GM]
  int* sums = (int*)(l_s + 4 * DE_GM);                // [6]
  int& last = sums[6];
  uint32_t* tmem_slot = (uint32_t*)(sums + 7);
  volatile int* abort_flag = sums + 8;
  int* first = (int*)(smem + de_off_seq<HD>);         // [B + 1] first tile of each sequence
  const int B = p.B, G = p.Hq / p.Hkv, heads = p.Hkv * p.n_gchunks;
  int* pos_s = first + B + 1;                         // [B] last visible position
  int* begin_s = pos_s + B;                           // [B] first visible position
  int* slot_s = begin_s + B;                          // [B]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < 3; ++s) {
      mbar_init(&kfull[s], 1);
      mbar_init(&kempty[s], 1);
      mbar_init(&vfull[s], 1);
      mbar_init(&vempty[s], 1);
    }
    for (int s = 0; s < DE_SC; ++s) {
      mbar_init(&sc_full[s], 1);
      mbar_init(&sc_empty[s], 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 4);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_full[s], 1);
      mbar_init(&o_free[s], 4);
      mbar_init(&q_full[s], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    first[0] = 0;
  }
  // the cut, from the step's own inputs (kept within the table whatever they are)
  for (int b0 = 0, sum = 0; b0 < B; b0 += DE_THREADS) {
    const int i = b0 + tid;
    int n = 0;
    if (i < B) {
      const int pos = min(max(p.token_pos[i], -1), p.max_pages * E8_PAGE - 1), begin = max(first_visible(pos, p.span), 0);
      pos_s[i] = pos;
      begin_s[i] = begin;
      slot_s[i] = min(max(p.seq_slot[i], 0), p.n_slots - 1);
      n = (max(pos, 0) / E8_PAGE - begin / E8_PAGE) / 2 + 1;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += up;
    }
    if (lane == 31) sums[warp] = n;
    __syncthreads();
    for (int k = 0; k < warp; ++k) n += sums[k];
    if (i < B) first[i + 1] = n + sum;
    for (int k = 0; k < DE_THREADS / 32; ++k) sum += sums[k];
    __syncthreads();
  }
  const int P = first[B];
  const long long total = (long long)heads * P;
  const unsigned nb = (unsigned)min((long long)gridDim.x, (total + DE_MIN_TILES - 1) / DE_MIN_TILES);   // (no run is empty)
  if (blockIdx.x >= nb) return;                       // (nothing is on its way yet)
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();       // (now: a successor's block may wait for tensor memory, but never one of these behind it)

  auto block_of = [&](long long tile) { return (int)(((tile + 1) * nb - 1) / total); };
  const long long lo = blockIdx.x * total / nb, hi = (blockIdx.x + 1) * total / nb;
  const int n_tiles = (int)(hi - lo);
  DecPlace start;
  start.head = (int)(lo / P);
  {
    const int y = (int)(lo - (long long)start.head * P);
    int b = 0;
    for (int step = DE_MAX_B / 2; step > 0; step >>= 1)
      if (b + step < B && first[b + step] <= y) b += step;
    start.b = b;
    start.k = y - first[b];
    start.nk = first[b + 1] - first[b];
  }
  auto advance = [&](DecPlace& x) {                   // to the next tile; true: of another sequence or head
    if (++x.k < x.nk) return false;
    x.k = 0;
    if (++x.b == B) {
      x.b = 0;
      ++x.head;
    }
    x.nk = first[x.b + 1] - first[x.b];
    return true;
  };
  auto two_pages = [&](const DecPlace& x) { return begin_s[x.b] / E8_PAGE + 2 * x.k + 1 <= max(pos_s[x.b], 0) / E8_PAGE; };
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      DecPlace at = start;
      bool ok = true;
      for (int it = 0; ok && it < n_tiles; ++it) {
        const int kvh = at.head / p.n_gchunks, pg = begin_s[at.b] / E8_PAGE + 2 * at.k, n = two_pages(at) ? 2 : 1;
        const int* row = p.page_table + (size_t)slot_s[at.b] * p.max_pages + pg;
        int rows[2];                                  // first row of each page's kv head
        for (int j = 0; j < n; ++j) rows[j] = (min(max(row[j], 0), p.n_pages - 1) * p.Hkv + kvh) * E8_PAGE;
        const int ks = it % KST, vs = it % VST, cs = it % DE_SC;
        if (it >= KST) ok = mbar_wait(&kempty[ks], (it / KST - 1) & 1, abort_flag);
        if (!ok) break;
        mbar_expect_tx(&kfull[ks], n * PAGE_BYTES);
        for (int j = 0; j < n; ++j) tma_load_2d(k_s + ks * STAGE + j * PAGE_BYTES, &map_k, &kfull[ks], 0, rows[j]);
        if (it >= DE_SC) ok = mbar_wait(&sc_empty[cs], (it / DE_SC - 1) & 1, abort_flag);
        if (!ok) break;
        mbar_expect_tx(&sc_full[cs], n * 2 * E8_PAGE);
        for (int j = 0; j < n; ++j) {
          bulk_load(sc_s + cs * 256 + j * E8_PAGE, p.kscales + rows[j], E8_PAGE, &sc_full[cs]);
          bulk_load(sc_s + cs * 256 + 128 + j * E8_PAGE, p.vscales + rows[j], E8_PAGE, &sc_full[cs]);
        }
        if (it >= VST) ok = mbar_wait(&vempty[vs], (it / VST - 1) & 1, abort_flag);
        if (!ok) break;
        mbar_expect_tx(&vfull[vs], n * PAGE_BYTES);
        for (int j = 0; j < n; ++j) tma_load_2d(v_s + vs * STAGE + j * PAGE_BYTES, &map_v, &vfull[vs], 0, rows[j]);
        advance(at);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_e4m3(DE_TK, 16, false), idesc_o = idesc_e4m3(HD, 16, true);
      DecPlace ahead = start, at = start;             // the tile whose scores, whose output come next
      int seg = 0;
      bool fresh = true, ok = true;
      auto scores = [&](int it) {
        const int ks = it % KST;
        if (fresh) ok = mbar_wait(&q_full[seg & 1], (seg >> 1) & 1, abort_flag);
        if (ok && it >= 2) ok = mbar_wait(&s_free[it & 1], ((it >> 1) - 1) & 1, abort_flag);
        if (ok) ok = mbar_wait(&kfull[ks], (it / KST) & 1, abort_flag);
        if (!ok) return;
        tc_fence_after_sync();
        const uint64_t a = desc_rows<HD>(smem_u32(k_s + ks * STAGE)), b = desc_rows<HD>(smem_u32(q_s + (seg & 1) * 16 * HD));
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) umma_e4m3(tmem_base + (it & 1) * 16, a + 2 * k, b + 2 * k, idesc_s, k != 0);
        umma_commit(&s_full[it & 1]);
        umma_commit(&kempty[ks]);
        fresh = advance(ahead);
        if (fresh) ++seg;
      };
      scores(0);
      for (int it = 0; ok && it < n_tiles; ++it) {
        if (it + 1 < n_tiles) scores(it + 1);
        const int vs = it % VST;
        if (ok) ok = mbar_wait(&p_full[it & 1], (it >> 1) & 1, abort_flag);
        if (ok && it >= 2) ok = mbar_wait(&o_free[it & 1], ((it >> 1) - 1) & 1, abort_flag);
        if (ok) ok = mbar_wait(&vfull[vs], (it / VST) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t a = desc_rows<HD>(smem_u32(v_s + vs * STAGE)), b = desc_weights(smem_u32(p_s + (it & 1) * 2048));
        const int steps = two_pages(at) ? 4 : 2;      // 32 keys each
        for (int k = 0; k < steps; ++k)
          umma_e4m3(tmem_base + O_COL + (it & 1) * 16, a + k * (32 * HD >> 4), b + k * (32 * 16 >> 4), idesc_o, k != 0);
        umma_commit(&o_full[it & 1]);
        umma_commit(&vempty[vs]);
        advance(at);
      }
    }
  } else {
    // (no way out of this loop: the four warps meet at barriers; once a wait has run out the others are not waited for)
    const int quarter = warp & 3, st = tid - 64;
    const int r = quarter * 32 + lane;                // key of the tile
    const int dim = HD == 128 ? r : quarter * 16 + lane;         // number of the head (heads of 64: a warp's first 16 lanes)
    const bool has_dim = HD == 128 || lane < 16;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) {
      if (ok) ok = mbar_wait(bar, parity & 1, abort_flag);
    };
    // the queries of a sequence and kv head as two e4m3 terms (rows g and GM + g of the operand), and what the scores are
    // scaled by; 16 threads a head
    auto prepare = [&](const DecPlace& x, int buf) {
      const int g0 = x.head % p.n_gchunks * DE_GM, GC = min(GM, G - g0), head0 = x.head / p.n_gchunks * G + g0;
      const int g = st >> 4, part = st & 15;
      constexpr int N = HD / 16;
      float v[N];
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        uint2 u = make_uint2(0u, 0u);
        if (g < GC) u = __ldcg(reinterpret_cast<const uint2*>(p.q + (size_t)x.b * p.ldq + (size_t)(head0 + g) * HD + part * N + k));
        v[k] = __uint_as_float(u.x << 16);
        v[k + 1] = __uint_as_float(u.x & 0xffff0000u);
        v[k + 2] = __uint_as_float(u.y << 16);
        v[k + 3] = __uint_as_float(u.y & 0xffff0000u);
      }
#pragma unroll
      for (int k = 0; k < N; ++k) most = fmaxf(most, fabsf(v[k]));
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const int e = min(max((int)(__float_as_uint(most) >> 23), 8), 254);
      const float down = __uint_as_float((unsigned)(261 - e) << 23);            // 2^(7 - (e - 127))
      if (g < GM) {
        uint32_t hi[N / 4], lo4[N / 4];
#pragma unroll
        for (int k = 0; k < N; k += 4) {
          const float a = v[k] * down, b = v[k + 1] * down, c = v[k + 2] * down, d = v[k + 3] * down;
          hi[k / 4] = e4m3_quad(a, b, c, d);
          const float2 ab = e4m3_back(hi[k / 4]), cd = e4m3_back(hi[k / 4] >> 16);
          lo4[k / 4] = e4m3_quad((a - ab.x) * 16.f, (b - ab.y) * 16.f, (c - cd.x) * 16.f, (d - cd.y) * 16.f);
        }
#pragma unroll
        for (int term = 0; term < 2; ++term) {
          const int row = term * GM + g, chunk = part * N / 16;
          uint8_t* dst = q_s + buf * 16 * HD + row * HD + ((chunk ^ (HD == 128 ? row & 7 : (row >> 1) & 3)) << 4) + part * N % 16;
          const uint32_t* src = term ? lo4 : hi;
          if (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(src[0], src[N / 4 - 1]);
          else *reinterpret_cast<uint32_t*>(dst) = src[0];
        }
        if (part == 0) fs_s[buf * DE_GM + g] = __uint_as_float((unsigned)(e - 7) << 23) * p.scale_log2e;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[buf]);
    };
    DecPlace at = start;
    prepare(at, 0);
    soft_sync();
    int seg = 0;
    bool fresh = true;
    float m[GM], l[GM], N[GM], n_t[GM], o[GM];
    // the output of tile `it`, whose reference is n_t, into o
    auto gather = [&](int it) {
      wait(&o_full[it & 1], it >> 1);
      __syncwarp();
      tc_fence_after_sync();
      float t[16];
      tmem_ld_32x16(lane_addr + O_COL + (it & 1) * 16, t);
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[it & 1]);
#pragma unroll
      for (int g = 0; g < GM; ++g) {
        float x = fmaf(t[GM + g], 0.0625f, t[g]);
        if (TERMS == 3) x = fmaf(t[(TERMS - 1) * GM + g], 0.00390625f, x);
        const float top = fmaxf(N[g], n_t[g]);
        o[g] = fmaf(o[g], exp2_whole(N[g] - top), x * exp2_whole(n_t[g] - top));
        N[g] = top;
      }
    };
    for (int it = 0; it < n_tiles; ++it) {
      const int g0 = at.head % p.n_gchunks * DE_GM, GC = min(GM, G - g0);
      DecPlace next = at;
      const bool ends = advance(next) || it + 1 == n_tiles;
      if (fresh) {
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          m[g] = N[g] = n_t[g] = -1e30f;
          l[g] = o[g] = 0.f;
        }
      }
      if (ends && it + 1 < n_tiles) prepare(next, (seg + 1) & 1);
      wait(&s_full[it & 1], it >> 1);
      __syncwarp();
      tc_fence_after_sync();
      float s[16];
      tmem_ld_32x16(lane_addr + (it & 1) * 16, s);
      wait(&sc_full[it % DE_SC], it / DE_SC);
      __syncwarp();
      const int kb = sc_s[it % DE_SC * 256 + r], vb = sc_s[it % DE_SC * 256 + 128 + r];
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s_free[it & 1]);
        mbar_arrive(&sc_empty[it % DE_SC]);
      }
      const int t = (begin_s[at.b] / E8_PAGE + 2 * at.k) * E8_PAGE + r;
      const bool seen = t >= begin_s[at.b] && t <= pos_s[at.b];
      const float kpow = e4m3_scale(kb), bexp = (float)(vb - 127);
      float* red = red_s + (it & 1) * 4 * 2 * DE_GM;
#pragma unroll
      for (int g = 0; g < GM; ++g) {
        const float x = fmaf(s[GM + g], 0.0625f, s[g]) * (kpow * fs_s[(seg & 1) * DE_GM + g]);
        s[g] = seen ? x : -INFINITY;
        const float a = warp_max_redux(s[g]), b = warp_max_redux(s[g] + bexp);
        if (lane == 0) {
          red[quarter * 2 * DE_GM + g] = a;
          red[quarter * 2 * DE_GM + DE_GM + g] = b;
        }
      }
      soft_sync();
      float n_new[GM];
      uint32_t packed[4];
      {
        float w[GM];
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          const float a = fmaxf(fmaxf(red[g], red[2 * DE_GM + g]), fmaxf(red[4 * DE_GM + g], red[6 * DE_GM + g]));
          const float b = fmaxf(fmaxf(red[DE_GM + g], red[3 * DE_GM + g]), fmaxf(red[5 * DE_GM + g], red[7 * DE_GM + g]));
          const float m_new = fmaxf(m[g], ceilf(a));
          n_new[g] = fmaxf(ceilf(b), -1e30f);
          l[g] = fmaf(l[g], exp2_whole(m[g] - m_new), exp2_fast(s[g] - m_new));
          m[g] = m_new;
          w[g] = exp2_fast(s[g] + (bexp - n_new[g] + 8.f));
        }
        // terms of the weights: byte term * GM + g of the key's 16
        auto term = [&](float f) {
          uint32_t q4[GM / 4];
#pragma unroll
          for (int k = 0; k < GM; k += 4) {
            q4[k / 4] = e4m3_quad(w[k] * f, w[k + 1] * f, w[k + 2] * f, w[k + 3] * f);
            const float2 ab = e4m3_back(q4[k / 4]), cd = e4m3_back(q4[k / 4] >> 16);
            const float back = 1.f / f;
            w[k] = fmaf(-ab.x, back, w[k]);
            w[k + 1] = fmaf(-ab.y, back, w[k + 1]);
            w[k + 2] = fmaf(-cd.x, back, w[k + 2]);
            w[k + 3] = fmaf(-cd.y, back, w[k + 3]);
          }
          return GM == 4 ? make_uint2(q4[0], 0u) : make_uint2(q4[0], q4[GM / 4 - 1]);
        };
        const uint2 a = term(1.f), b = term(16.f);
        if (GM == 4) {
          packed[0] = a.x;
          packed[1] = b.x;
          packed[2] = term(256.f).x;
          packed[3] = 0u;
        } else {
          packed[0] = a.x;
          packed[1] = a.y;
          packed[2] = b.x;
          packed[3] = b.y;
        }
      }
      *reinterpret_cast<uint4*>(p_s + (it & 1) * 2048 + r * 16) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      // value rows that nobody sees may hold anything: zeros, so that 0 times NaN does not come about
      if (!seen && (r < E8_PAGE || two_pages(at))) {
        wait(&vfull[it % VST], it / VST);
        uint8_t* row = v_s + it % VST * STAGE + r * HD;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) *reinterpret_cast<uint4*>(row + k * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[it & 1]);
      if (!fresh) gather(it - 1);
#pragma unroll
      for (int g = 0; g < GM; ++g) n_t[g] = n_new[g];
      fresh = ends;
      if (ends) {
        gather(it);
        // the sequence's result, or this block's part of it
        const long long begin = (long long)at.head * P + first[at.b], end = (long long)at.head * P + first[at.b + 1];
        const bool whole = begin >= lo && end <= hi;
        const int head0 = at.head / p.n_gchunks * G + g0;
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          l[g] = warp_sum(l[g]);
          if (lane == 0) l_s[quarter * DE_GM + g] = l[g];
        }
        soft_sync();
        const size_t part0 = ((size_t)blockIdx.x * 2 + (begin >= lo ? 1 : 0)) * GM;
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          if (g >= GC) continue;
          float ll = (l_s[g] + l_s[DE_GM + g]) + (l_s[2 * DE_GM + g] + l_s[3 * DE_GM + g]);
          // relative to m (in two steps: the values' powers may be far from the weights')
          const float half = floorf(0.5f * (N[g] - 8.f - m[g]));
          const float x = o[g] * exp2_whole(fminf(half, 127.f)) * exp2_whole(fminf(N[g] - 8.f - m[g] - half, 127.f));
          if (whole) {
            float f = 1.f;
            if (p.sink != nullptr) {
              const float sk = p.sink[head0 + g] * 1.4426950408889634f, top = fmaxf(m[g], sk);
              f = exp2_fast(m[g] - top);
              ll = fmaf(ll, f, exp2_fast(sk - top));
            }
            f = ll == 0.f ? 0.f : f / ll;             // (a sequence without a visible key: zeros)
            if (has_dim) p.out[(size_t)at.b * p.ldo + (size_t)(head0 + g) * HD + dim] = __float2bfloat16_rn(x * f);
          } else {
            if (has_dim) p.part_acc[(part0 + g) * HD + dim] = x;
            if (st == 0) *reinterpret_cast<float2*>(p.part_ml + (part0 + g) * 2) = make_float2(m[g], ll);
          }
        }
        if (!whole) {
          soft_sync();
          const int i0 = block_of(begin), parts = block_of(end - 1) - i0 + 1;
          if (st == 0) {
            // releases the block's part, which is behind the barrier; acquires those of the blocks before it for the
            // other threads, behind the next one
            int* ticket = p.tickets + (size_t)at.b * heads + at.head;
            int before;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
            last = before == parts - 1;
            if (before == parts - 1) *ticket = 0;     // for the next launch
          }
          soft_sync();
          if (last) {
            // a thread per four numbers, or 2, 4, 8 threads that share the parts; four parts in flight each
            const int cols = GC * H4;
            int tpc = 1;
            while (tpc < 8 && cols * tpc * 2 <= DE_SOFT) tpc *= 2;
            for (int c0 = 0; c0 < cols; c0 += DE_SOFT / tpc) {
              const int col = c0 + st / tpc;
              const int g = min(col, cols - 1) / H4, d = min(col, cols - 1) % H4 * 4;
              float mm = -1e30f, ll = 0.f;
              float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
              for (int k0 = st % tpc; k0 < parts; k0 += 4 * tpc) {
                float2 ml[4];
                float4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int k = k0 + j * tpc;
                  const size_t x = ((size_t)(i0 + min(k, parts - 1)) * 2 + (k == 0 ? 1 : 0)) * GM + g;
                  ml[j] = k < parts ? __ldcg(reinterpret_cast<const float2*>(p.part_ml) + x) : make_float2(-1e30f, 0.f);
                  v[j] = k < parts ? __ldcg(reinterpret_cast<const float4*>(p.part_acc + x * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                float top = mm;
#pragma unroll
                for (int j = 0; j < 4; ++j) top = fmaxf(top, ml[j].x);
                const float keep = exp2_fast(mm - top);
                mm = top;
                ll *= keep; a.x *= keep; a.y *= keep; a.z *= keep; a.w *= keep;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float w = exp2_fast(ml[j].x - top);
                  ll = fmaf(w, ml[j].y, ll);
                  a.x = fmaf(w, v[j].x, a.x); a.y = fmaf(w, v[j].y, a.y);
                  a.z = fmaf(w, v[j].z, a.z); a.w = fmaf(w, v[j].w, a.w);
                }
              }
              for (int x = tpc >> 1; x > 0; x >>= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, mm, x), top = fmaxf(mm, m2);
                const float k1 = exp2_fast(mm - top), k2 = exp2_fast(m2 - top);
                mm = top;
                ll = ll * k1 + __shfl_xor_sync(0xffffffffu, ll, x) * k2;
                a.x = a.x * k1 + __shfl_xor_sync(0xffffffffu, a.x, x) * k2;
                a.y = a.y * k1 + __shfl_xor_sync(0xffffffffu, a.y, x) * k2;
                a.z = a.z * k1 + __shfl_xor_sync(0xffffffffu, a.z, x) * k2;
                a.w = a.w * k1 + __shfl_xor_sync(0xffffffffu, a.w, x) * k2;
              }
              if (col < cols && st % tpc == 0) {
                float f = 1.f;
                if (p.sink != nullptr) {
                  const float sk = p.sink[head0 + g] * 1.4426950408889634f, top = fmaxf(mm, sk);
                  f = exp2_fast(mm - top);
                  ll = fmaf(ll, f, exp2_fast(sk - top));
                }
                f = ll == 0.f ? 0.f : f / ll;
                *reinterpret_cast<uint2*>(p.out + (size_t)at.b * p.ldo + (size_t)(head0 + g) * HD + d) =
                    make_uint2(bf16_word(a.x * f, a.y * f), bf16_word(a.z * f, a.w * f));
              }
            }
          }
        }
        ++seg;
      }
      at = next;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (tid == 0) atomicExch(&g_decode_e4m3_error, 1);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);       // (what is still on its way arrives)
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

inline int decode_e8_blocks(int hd) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms * (hd <= 64 ? de_blocks<64> : de_blocks<128>);
}

template <int HD, int GM>
int launch_decode_e8(const CUtensorMap& mk, const CUtensorMap& mv, const DecE8& p, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute((const void*)attention_decode_e4m3_kernel<HD, GM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)de_smem<HD>(DE_MAX_B));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute((const void*)attention_decode_e4m3_kernel<HD, GM>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             (int)cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return (int)e;
  launch_kernel(attention_decode_e4m3_kernel<HD, GM>, dim3(decode_e8_blocks(HD)), dim3(DE_THREADS), de_smem<HD>(p.B), stream, mk, mv, p);
  return launch_status();
}

}  // namespace dlgo

using namespace dlgo;

namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)f;
  }
  return fn;
}

// rows of hd bytes, a page of one head (64 rows) at a time
int make_map(CUtensorMap* m, const void* base, long long rows, int hd) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return DLGO_ERR_DRIVER;
  cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)hd};
  cuuint32_t box[2] = {(cuuint32_t)hd, E8_PAGE};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? DLGO_OK : DLGO_ERR_DRIVER;
}

}  // namespace

// Floats of scratch that a launch needs, whatever the number of sequences.
DLGO_EXPORT long long dlgo_attention_decode_e4m3_scratch(int Hq, int Hkv, int hd) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv) return 0;
  return (long long)decode_e8_blocks(hd) * 2 * (Hq / Hkv <= 4 ? 4 : DE_GM) * (hd + 2);
}

// q[B, .] bf16 (row stride ldq, head h at column h * hd), one token per sequence at position token_pos[b] whose key and
// value are in the cache; out[B, .] bf16 (row stride ldo).  `scratch` as above; `tickets` [B * Hkv * ceil(Hq / Hkv / 8)]
// zero, and left zero; `sink` [Hq] fp32 or null.
DLGO_EXPORT int dlgo_attention_decode_e4m3(const void* q, int B, int ldq, const void* kpages, const void* vpages, const void* kscales,
                                           const void* vscales, int n_pages, const int* page_table, int n_slots, int max_pages,
                                           const int* seq_slot, const int* token_pos, void* out, int ldo, int Hq, int Hkv, int hd, int span,
                                           float scale, const float* sink, float* scratch, int* tickets, cudaStream_t stream) {
  if (B <= 0) return DLGO_OK;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || (hd != 64 && hd != 128) || n_pages <= 0 || n_slots <= 0 || max_pages <= 0) return DLGO_ERR_SIZE;
  if ((long long)n_pages * Hkv * E8_PAGE > 0x7fffffffLL || max_pages > 0x7fffffff / E8_PAGE) return DLGO_ERR_SIZE;
  if ((ldq & 3) || (ldo & 3) || ((uintptr_t)q & 7) || ((uintptr_t)out & 7) || ((uintptr_t)kpages & 15) || ((uintptr_t)vpages & 15) ||
      ((uintptr_t)kscales & 15) || ((uintptr_t)vscales & 15) || ((uintptr_t)scratch & 15) || scratch == nullptr || tickets == nullptr)
    return DLGO_ERR_ALIGN;
  CUtensorMap mk, mv;
  int st = make_map(&mk, kpages, (long long)n_pages * Hkv * E8_PAGE, hd);
  if (st == DLGO_OK) st = make_map(&mv, vpages, (long long)n_pages * Hkv * E8_PAGE, hd);
  if (st != DLGO_OK) return st;
  const int G = Hq / Hkv, gm = G <= 4 ? 4 : DE_GM;
  DecE8 p;
  p.ldq = ldq;
  p.kscales = (const uint8_t*)kscales; p.vscales = (const uint8_t*)vscales;
  p.page_table = page_table; p.n_slots = n_slots; p.max_pages = max_pages; p.n_pages = n_pages;
  p.ldo = ldo; p.Hq = Hq; p.Hkv = Hkv;
  p.n_gchunks = (G + DE_GM - 1) / DE_GM;
  p.span = span; p.scale_log2e = scale * 1.4426950408889634f; p.sink = sink;
  p.part_acc = scratch;
  p.part_ml = scratch + (size_t)decode_e8_blocks(hd) * 2 * gm * hd;
  for (int b0 = 0; b0 < B; b0 += DE_MAX_B) {       // (one launch as a rule; they run one after another and share the scratch)
    p.B = B - b0 < DE_MAX_B ? B - b0 : DE_MAX_B;
    p.q = (const __nv_bfloat16*)q + (size_t)b0 * ldq;
    p.out = (__nv_bfloat16*)out + (size_t)b0 * ldo;
    p.seq_slot = seq_slot + b0;
    p.token_pos = token_pos + b0;
    p.tickets = tickets + (size_t)b0 * Hkv * p.n_gchunks;
    if (hd == 64) st = gm == 4 ? launch_decode_e8<64, 4>(mk, mv, p, stream) : launch_decode_e8<64, 8>(mk, mv, p, stream);
    else st = gm == 4 ? launch_decode_e8<128, 4>(mk, mv, p, stream) : launch_decode_e8<128, 8>(mk, mv, p, stream);
    if (st != DLGO_OK) return st;
  }
  return DLGO_OK;
}

// 1 if a bounded wait ran out since the last call (clears the word).
DLGO_EXPORT int dlgo_attention_decode_e4m3_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_decode_e4m3_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_decode_e4m3_error, &zero, sizeof(int));
  return v;
}
