// Decode attention over the 8-bit cache (e4m3 rows with a power of two each, see e4m3.cuh) on tcgen05, the rows as operands
// straight from their pages.
//
// One new token per sequence; scores s_j = q . k_j * scale over the visible positions, softmax, weighted sum of the values
// (models/llm/forward.go:258-278, with rows that take hd + 1 bytes instead of 2 hd).  With k_j = K_j 2^a_j and
// v_j = V_j 2^b_j, K and V being the stored e4m3 numbers, per query head and tile of 128 keys (256 with heads of 64):
//
//   s_j = (K_j . q') * 2^a_j * (scale log2(e) 2^c)      q' = q / 2^c, its largest number in [2^7, 2^8)
//   p_j = 2^(s_j - m),  l = sum_j p_j                   m = the maximum of s_j so far of the keys that one thread sees; the
//                                                       threads' sums meet at the sequence's end
//   w_j = 2^(s_j + b_j - n + 8),  O' = sum_j w_j V_j    n = the tile's maximum of s_j + b_j: w_j <= 2^8
//   O = O 2^(n_before - N) + O' 2^(n - N)               N = the running maximum of n
//   out = O 2^(N - 8 - m) / l
//
// Both products have e4m3 on both sides.  The other operand enters as several e4m3 terms in columns of their own: a query as
// x = x1 + x2 / 16, which holds a bfloat16 number whole down to 2^-22 of the row's largest (each term keeps 4 bits, and what
// the first leaves over is at most 2^-4 of it); a weight as w1 + w2 / 16, 2^-8 of its size, or, where a block has four heads at
// most and columns are left, + w3 / 256, 2^-11 (it passes through float16); and 2^-22 (2^-26) of the tile's largest weight.
// The values' powers are part of the weights, so a row of small values may hold all of the softmax's weight without a loss;
// and because every tile has a reference of its own, neither does a long tail of small weights behind a large one.  s_j + b_j is one
// 32-bit number: a result is off by 2^-24 |s_j| relative to itself (as far as a score's own sum is), and what scores below -1e30 counts
// as not seen.
//
// Bound by the rows, which are read once.  The keys (of the scores) and the numbers of a head (of the output) are the
// MMA's rows and the query heads of a kv head, times their terms, its 16 columns, so no thread touches a row: per tile
// a thread handles one key's scores.  (With mma.sync, whose operands are at least 16 bits wide, converting the rows and the
// scores' arithmetic took 424 instructions per 32 keys and warp: 32 sequences of 256 to 4,096 keys, heads of 128, 35.2 us.)
//   warp 0     TMA, a lane per page: keys, values and scale bytes into rings
//   warps 1, 2 tcgen05.mma: scores (128 keys x 16, once or twice); output (numbers x 16), values as the MN-major operand from
//              the page layout [key][number], weights MN-major as the threads write them, 16 bytes a key.  (One thread for
//              both took 3,200 clocks a tile: it was what the others waited for.)
//   warps 3-6  a thread per key, or per two: scores, maxima over the tile (redux and a barrier), weights; then, a thread per
//              number of a head, the output of the tile before
// Two such blocks share an SM, so one's chain of steps runs under the other's.  The chain is what tiles of 256 keys are for with
// heads of 64: with 128, some 300 instructions and 2,800 clocks a tile, three blocks' chains did not keep up with memory (one
// sequence of 131,072 keys 38 us, 29 with 256).  Tensor memory is allocated before the next launch may begin, 128 of an SM's
// 512 columns a block, so a block of that launch can wait for columns only behind blocks that hold theirs and will end.
//
// Work is shared evenly: the tiles of all sequences and kv heads are numbered through, head by head and sequence by sequence,
// and every block takes an equal run of them, as many blocks as are resident at once: all SMs stream until the end, whatever
// the lengths.  A sequence's first tile counts twice: its queries, the end of the sequence before and the pause between them
// cost about as much as a tile.  What blocks share, at most the first and the last sequence of each, goes through scratch
// memory, and the block that takes a sequence's last ticket adds the parts up in the order of the blocks; nobody waits for
// another block.  With few sequences every block takes tiles of one sequence alone, so that it has one end to come to, not
// two: where a block for each of these parts is there and the longest is no more than two tiles above an equal share (with
// none above, 16 sequences of 64 to 2,048 keys, 24 on 8 heads of 128, 16.6 us, with two 13.4; five are no faster).  Against
// equal runs: these 12.7 us for 16.2, 8 of 300 to 1,700 keys 9.1 for 12.3.  Two tiles stay together either way (8 sequences of 100
// to 160 keys, heads of 128: 6.4 us, cut 7.3); three do not (a whole layer for one sequence of 540 keys, heads of 64: 43.7 us,
// together 45.1).
// The cut and the order of the sums follow from the lengths alone, so a call repeats its bits.
//
// Measured (launches one behind another in a graph, inputs larger than L2 or as large as they are; the copy rate is 6.57 TB/s):
//   32 sequences of 256 to 4,096 keys, 32 query on 8 kv heads of 128   30.8 us, 5.0 TB/s, 76 % of the copy rate
//   64 sequences of 128 to 4,096 keys, 32 on 8 heads of 64             32.3 us, 4.5 TB/s, 69 %
//   one sequence of 131,072 keys, 32 on 8 heads of 128                 45.7 us, 5.9 TB/s, 90 %
//   8 sequences of 300 to 1,700 keys, 32 on 8 heads of 64               8.8 us, and one of 57 keys 4.2 us: latency
// Some 7 to 9 us of a launch are fixed: the cut, the first loads' way, a run's end, its ticket and the join.  The rest of the
// distance is the blocks' uneven progress (10 % either way).  What a launch runs once it fetches anew, so the code is kept short
// where it runs once a sequence: a lane per head at its end, one copy of what takes an output in (34.5 to 33.3 us, 64 sequences).
#include <math.h>

#include "common.cuh"
#include "e4m3.cuh"
#include "tcgen05.cuh"

namespace dlgo {

using namespace sm100;

constexpr int DE_THREADS = 224;
constexpr int DE_SOFT = 128;          // of them, warps 3-6
// halves of a tile, of 128 keys (two pages) each
template <int HD> constexpr int de_halves = HD <= 64 ? 2 : 1;
constexpr int DE_GM = 8;              // query heads of a kv head per block at most
constexpr int DE_MIN_RUN = 2;         // a block's least run (so that none lies within one tile)
constexpr int DE_WHOLE = 2;           // tiles of a sequence that is not cut
constexpr int DE_SLACK = 2;           // tiles beyond an equal share that a block may have where it has one sequence's alone
constexpr int DE_MAX_B = 1024;        // sequences of a launch (their first tiles, positions and slots lie in shared memory)
constexpr int DE_BARS = 40;           // room for barriers
constexpr int DE_SC = 3;              // tiles whose scale bytes are on their way or in use

constexpr int DE_KST = 2, DE_VST = 2; // tiles of keys, of values in shared memory (16 KB each; a third of keys gains nothing)
constexpr int DE_BLOCKS = 2;          // blocks on an SM

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
  int room;                // blocks for each kv head (and chunk of its query heads), at most
  float one_by_room;
  float scale_log2e;
  const float* sink;       // [Hq] or null: exp(sink) joins the denominator
  float* part_acc;         // [blocks][2][GM][HD]  O relative to m
  float* part_ml;          // [blocks][2][GM][2]  m and l
  int* tickets;            // [B][heads], zero between launches
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bf16_word(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float warp_max_redux(float x) {     // (a NaN does not count; volatile: all lanes execute it, wherever its result is used)
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// float16 pairs to e4m3, the first number in the low byte
__device__ __forceinline__ uint32_t e4m3_of_half2(__half2 h) {
  uint16_t q;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(q) : "r"(*reinterpret_cast<const uint32_t*>(&h)));
  return q;
}
__device__ __forceinline__ __half2 half2_of_e4m3(uint32_t pair) {
  const uint32_t h = e4m3_low_half2(pair);
  return *reinterpret_cast<const __half2*>(&h);
}
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

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

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

// A tile of the run: virtual head (kv head and chunk of its query heads), sequence, tile k of its nk, the sequence's pages from
// there on.
struct DecPlace {
  int head, b, k, nk, pages;
};

// Shared memory: rings of keys and of values, two buffers of queries and of weights, scale bytes, barriers, ... , sequences
template <int HD> constexpr int de_off_q = (DE_KST + DE_VST) * de_halves<HD> * 128 * HD;
template <int HD> constexpr int de_off_p = de_off_q<HD> + 2 * 16 * HD;
// What lies behind the rings: scale bytes, barriers, maxima over the tile [2][4][GM] and, each per head, row scales, maxima and
// sums; then the sequences.
constexpr int DE_RED = 2 * 4 * DE_GM * 4, DE_MISC = 10 * DE_GM * 4 + 128;
constexpr int de_seq_bytes(int B) { return (4 * B + 1) * 4; }
template <int HD> constexpr int de_end_p = de_off_p<HD> + 2 * de_halves<HD> * 2048;
template <int HD> constexpr int de_behind = DE_SC * de_halves<HD> * 256 + DE_BARS * 8 + DE_RED + DE_MISC + de_seq_bytes(DE_MAX_B);
// A join holds its parts where the rings were, and behind them in all that DE_BLOCKS blocks leave of an SM's 228 KB (a block takes 1 KB
// beside its own): what lies there is one go less where a sequence has a few parts more than the rings hold (37 parts of heads of
// 128, 35 in the rings alone, 46 with this: one of 131,072 keys 46.3 us for 46.8; nowhere slower).
template <int HD> constexpr int de_spare = (228 * 1024 / DE_BLOCKS - 1024 - de_end_p<HD> - de_behind<HD>) / 1024 * 1024;
static_assert(de_spare<64> >= 0 && de_spare<128> >= 0, "the blocks of an SM fit");
template <int HD> constexpr int de_off_sc = de_end_p<HD> + de_spare<HD>;
template <int HD> constexpr int de_off_bars = de_off_sc<HD> + DE_SC * de_halves<HD> * 256;
template <int HD> constexpr int de_off_red = de_off_bars<HD> + DE_BARS * 8;
template <int HD> constexpr int de_off_misc = de_off_red<HD> + DE_RED;
template <int HD> constexpr int de_off_seq = de_off_misc<HD> + DE_MISC;
template <int HD> constexpr size_t de_smem(int B) { return de_off_seq<HD> + (size_t)de_seq_bytes(B); }

template <int HD, int GM>
__global__ void __launch_bounds__(DE_THREADS, DE_BLOCKS)
attention_decode_e4m3_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, DecE8 p) {
  constexpr int TERMS = GM <= 4 ? 3 : 2;
  constexpr int H = de_halves<HD>, KST = DE_KST, VST = DE_VST, STAGE = H * 128 * HD, PAGE_BYTES = E8_PAGE * HD;
  constexpr uint32_t TMEM_COLS = 128, O_COL = 64;     // scores of two tiles in columns 0 to 63, outputs in 64 and 80
  constexpr int H4 = HD / 4;
  // joining parts: columns of four numbers at a time, bytes of them and their maxima and sums, parts that shared memory holds
  constexpr int JC = GM * H4 < DE_SOFT ? GM * H4 : DE_SOFT, JREC = JC * 16 + GM * 8, JN = de_off_sc<HD> / JREC;
  // the swizzled tiles want 1024-byte alignment (checked: a misaligned start ends the kernel with the error word set)
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicExch(&g_decode_e4m3_error, 1);
    return;
  }
  uint8_t* k_s = smem;
  uint8_t* v_s = k_s + KST * STAGE;
  uint8_t* q_s = smem + de_off_q<HD>;                 // [2][16 rows][HD], swizzled as the keys
  uint8_t* p_s = smem + de_off_p<HD>;                 // [2][H][128 keys][16]
  uint8_t* sc_s = smem + de_off_sc<HD>;               // [DE_SC][H][keys 128 | values 128]
  uint64_t* bars = (uint64_t*)(smem + de_off_bars<HD>);
  uint64_t* kfull = bars;                // KST
  uint64_t* kempty = kfull + KST;        // KST: the scores that read these keys have completed
  uint64_t* vfull = kempty + KST;        // VST
  uint64_t* vempty = vfull + VST;        // VST: the output that read these values has completed
  uint64_t* sc_full = vempty + VST;      // DE_SC
  uint64_t* sc_empty = sc_full + DE_SC;  // DE_SC
  uint64_t* s_full = sc_empty + DE_SC;   // 2: scores
  uint64_t* s_free = s_full + 2;         // 2: ... are in registers
  uint64_t* p_full = s_free + 2;         // 2: weights
  uint64_t* o_full = p_full + 2;         // 2: the output of a tile (its weights may be overwritten)
  uint64_t* o_free = o_full + 2;         // 2: ... is in registers
  uint64_t* q_full = o_free + 2;         // 2
  static_assert(2 * KST + 2 * VST + 2 * DE_SC + 12 <= DE_BARS, "the barriers fit");
  float* red_s = (float*)(smem + de_off_red<HD>);
  float* fs_s = (float*)(smem + de_off_misc<HD>);     // [2][DE_GM] row scales
  float2* ml_s = (float2*)(fs_s + 2 * DE_GM);         // [DE_GM][4 warps] maximum and sum
  int* sums = (int*)(ml_s + 4 * DE_GM);               // [8]
  uint32_t* tmem_slot = (uint32_t*)(sums + 8);
  volatile int* abort_flag = sums + 9;
  int* last_s = sums + 10;                            // [2] this block has a shared sequence's last ticket
  int* shared_s = sums + 16;                          // [2][4] head, sequence, first block, parts of the sequences it shares
  int* plan_s = sums + 24;                            // [2] first block and parts of this block's sequence (0: equal runs)
  int* first = (int*)(smem + de_off_seq<HD>);         // [B + 1] first tile of each sequence
  const int B = p.B, G = p.Hq / p.Hkv, heads = p.Hkv * p.n_gchunks;
  int* pos_s = first + B + 1;                         // [B] last visible position
  int* begin_s = pos_s + B;                           // [B] first visible position
  int* slot_s = begin_s + B;                          // [B]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < KST; ++s) {
      mbar_init(&kfull[s], 1);
      mbar_init(&kempty[s], 1);
    }
    for (int s = 0; s < VST; ++s) {
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
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
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
      n = (max(pos, 0) / E8_PAGE - begin / E8_PAGE) / (2 * H) + 2;         // (its first tile counts twice)
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += up;
    }
    if (lane == 31) sums[warp] = n;
    tc_fence_before_sync();
    __syncthreads();
    for (int k = 0; k < warp; ++k) n += sums[k];
    if (i < B) first[i + 1] = n + sum;
    for (int k = 0; k < DE_THREADS / 32; ++k) sum += sums[k];
    __syncthreads();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();       // (now: a successor's block may wait for tensor memory, but never one of these behind it)
  const int P = first[B];
  const long long total = (long long)heads * P;       // (counting first tiles twice)
  const unsigned nb = (unsigned)min((long long)gridDim.x, total / DE_MIN_RUN);        // (every sequence counts two at least)
  const bool narrow = total < 0xffffffffLL / (nb + 1);                                // (a division of 64 bits takes 100 instructions)
  auto start_of = [&](unsigned i) { return narrow ? (long long)(i * (unsigned)total / nb) : (long long)i * total / nb; };
  auto block_of = [&](long long x) { return (int)(narrow ? ((unsigned)(x + 1) * nb - 1) / (unsigned)total : ((x + 1) * nb - 1) / total); };
  auto enter = [&](DecPlace& x) {                     // what a sequence's tile k follows from the sequence
    x.nk = first[x.b + 1] - first[x.b] - 1;
    x.pages = max(pos_s[x.b], 0) / E8_PAGE - begin_s[x.b] / E8_PAGE + 1 - 2 * H * x.k;
  };
  // the place that the count x falls on: tile k begins at the sequence's count 0 (k = 0) or k + 1
  auto place = [&](long long x) {
    DecPlace at;
    at.head = (int)(narrow ? (unsigned)x / (unsigned)P : x / P);
    const int y = (int)(x - (long long)at.head * P);
    int b = -1;                                       // the last sequence whose first count is no more than y
#pragma unroll 1
    for (int i = lane; i < B; i += 32) b += first[i] <= y;
    b = __reduce_add_sync(0xffffffffu, b + 1) - 1;
    const int u = y - first[b];
    at.b = b;
    at.k = u == 0 ? 0 : max(1, u - 1);
    // a place behind the start of the sequence's last tile, and one within a sequence of DE_WHOLE tiles, is the start of the next
    const int nk = first[b + 1] - first[b] - 1;
    if (at.k >= nk || (at.k > 0 && nk <= DE_WHOLE)) {
      at.k = 0;
      if (++at.b == B) {
        at.b = 0;
        ++at.head;
      }
    }
    enter(at);
    return at;
  };
  int n_tiles = 0, own_parts = 0, own_first = 0;
  DecPlace start = {0, 0, 0, 1, 1};
  // Few sequences: every block takes tiles of one alone, about r at most, with r the least number that leaves a block for each
  // part.  (Every block counts the same, so r's quotients may be off by a rounding.  This runs before every launch's first load:
  // with divisions of whole numbers and unrolled loops it took a microsecond more.)
  if (B <= p.room) {
    const int least = (int)((P - B) * p.one_by_room) + 1;
    int r = least, limit = max(DE_WHOLE, least + DE_SLACK), all;
    float one_by_r;
    auto parts_of = [&](int i) {
      const int n = i < B ? first[i + 1] - first[i] - 1 : 0;
      return n <= DE_WHOLE ? min(n, 1) : min((int)((n - 1) * one_by_r) + 1, n);
    };
    for (; r <= limit; ++r) {
      one_by_r = __fdividef(1.f, r);
      all = 0;
#pragma unroll 1
      for (int i = lane; i < B; i += 32) all += parts_of(i);
      all = __reduce_add_sync(0xffffffffu, all);
      if (all <= p.room) break;
    }
    if (r <= limit) {
      own_parts = -1;                                 // (a block without a part)
      if ((int)blockIdx.x < heads * all) {
        start.head = (int)__fdividef(blockIdx.x + 0.5f, all);
        int y = (int)blockIdx.x - start.head * all;
#pragma unroll 1
        for (int i0 = 0; i0 < B; i0 += 32) {
          const int mine = parts_of(i0 + lane);
          int upto = mine;
#pragma unroll 1
          for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += up;
          }
          const unsigned behind = __ballot_sync(0xffffffffu, upto > y);
          if (behind) {
            const int at = __ffs(behind) - 1;
            own_parts = __shfl_sync(0xffffffffu, mine, at);
            const int j = y - __shfl_sync(0xffffffffu, upto - mine, at);
            own_first = (int)blockIdx.x - j;
            start.b = i0 + at;
            start.nk = first[start.b + 1] - first[start.b] - 1;
            const int each = (int)((unsigned)start.nk / (unsigned)own_parts), more = start.nk - each * own_parts;
            start.k = j * each + min(j, more);
            n_tiles = each + (j < more ? 1 : 0);      // (the first `more` parts have one more)
            enter(start);
            break;
          }
          y -= __shfl_sync(0xffffffffu, upto, 31);
        }
      }
    }
  }
  if (own_parts == 0 && blockIdx.x < nb) {
    DecPlace end;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      end = place(start_of(blockIdx.x + e));
      if (e == 0) start = end;
    }
    // tiles up to a place: those of the heads and sequences before it, and its k
    n_tiles = (end.head - start.head) * (P - B) + (first[end.b] - end.b + end.k) - (first[start.b] - start.b + start.k);
  }
  auto advance = [&](DecPlace& x) {                   // to the next tile; true: of another sequence or head
    x.pages -= 2 * H;
    if (++x.k < x.nk) return false;
    x.k = 0;
    if (++x.b == B) {
      x.b = 0;
      ++x.head;
    }
    enter(x);
    return true;
  };
  auto pages_of = [&](const DecPlace& x) { return min(2 * H, x.pages); };
  if (warp == 0) {
    // Lane j: page j of the tile.  Keys and scale bytes run a tile ahead of values, whose room is free only when the output
    // before is done; page numbers another tile ahead, the first ones before the launch before this has ended.
    DecPlace at = start;
    const int j = lane & (2 * H - 1);
    const bool mine = lane < 2 * H;
    int page = 0, row = 0, n = 0, v_row, v_n;
    auto look_up = [&]() {
      page = p.page_table[(size_t)slot_s[at.b] * p.max_pages + begin_s[at.b] / E8_PAGE + 2 * H * at.k + min(j, pages_of(at) - 1)];
    };
    if (n_tiles > 0) look_up();
    pdl_wait();
    bool ok = true;
    for (int it = 0; it <= n_tiles && n_tiles > 0; ++it) {
      v_row = row;
      v_n = n;
      if (it < n_tiles) {
        n = pages_of(at);
        row = (min(max(page, 0), p.n_pages - 1) * p.Hkv + at.head / p.n_gchunks) * E8_PAGE;   // first of the kv head
        advance(at);
        if (it + 1 < n_tiles) look_up();
        const int cs = it % DE_SC, ks = it % KST;
        if (it >= DE_SC) ok = mbar_wait(&sc_empty[cs], (it / DE_SC - 1) & 1, abort_flag);
        if (ok && it >= KST) ok = mbar_wait(&kempty[ks], (it / KST - 1) & 1, abort_flag);
        if (__any_sync(0xffffffffu, !ok)) break;
        if (lane == 0) {
          mbar_expect_tx(&kfull[ks], n * PAGE_BYTES);
          mbar_expect_tx(&sc_full[cs], n * 2 * E8_PAGE);
        }
        __syncwarp();
        if (mine && j < n) {
          tma_load_2d(k_s + ks * STAGE + j * PAGE_BYTES, &map_k, &kfull[ks], 0, row);
          uint8_t* dst = sc_s + (cs * H + j / 2) * 256 + j % 2 * E8_PAGE;
          bulk_load(dst, p.kscales + row, E8_PAGE, &sc_full[cs]);
          bulk_load(dst + 128, p.vscales + row, E8_PAGE, &sc_full[cs]);
        }
      }
      if (it > 0) {
        const int vi = it - 1, vs = vi % VST;
        if (vi >= VST) ok = mbar_wait(&vempty[vs], (vi / VST - 1) & 1, abort_flag);
        if (__any_sync(0xffffffffu, !ok)) break;
        if (lane == 0) mbar_expect_tx(&vfull[vs], v_n * PAGE_BYTES);
        __syncwarp();
        if (mine && j < v_n) tma_load_2d(v_s + vs * STAGE + j * PAGE_BYTES, &map_v, &vfull[vs], 0, v_row);
      }
    }
  } else if (warp == 1) {
    pdl_wait();
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3(128, 16, false);
      DecPlace at = start;
      int seg = 0;
      bool fresh = true, ok = true;
      for (int it = 0; it < n_tiles; ++it) {
        const int ks = it % KST;
        if (fresh) ok = mbar_wait(&q_full[seg & 1], (seg >> 1) & 1, abort_flag);
        if (ok && it >= 2) ok = mbar_wait(&s_free[it & 1], ((it >> 1) - 1) & 1, abort_flag);
        if (ok) ok = mbar_wait(&kfull[ks], (it / KST) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t a = desc_rows<HD>(smem_u32(k_s + ks * STAGE)), b = desc_rows<HD>(smem_u32(q_s + (seg & 1) * 16 * HD));
        const int n = pages_of(at);
#pragma unroll
        for (int h = 0; h < H; ++h)
          if (2 * h < n) {
#pragma unroll
            for (int k = 0; k < HD / 32; ++k)
              umma_e4m3(tmem_base + (it & 1) * 32 + h * 16, a + h * (128 * HD >> 4) + 2 * k, b + 2 * k, idesc, k != 0);
          }
        umma_commit(&s_full[it & 1]);
        umma_commit(&kempty[ks]);
        fresh = advance(at);
        if (fresh) ++seg;
      }
    }
  } else if (warp == 2) {
    pdl_wait();
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_e4m3(HD, 16, true);
      DecPlace at = start;
      bool ok = true;
      for (int it = 0; it < n_tiles; ++it) {
        const int vs = it % VST;
        if (it >= 2) ok = mbar_wait(&o_free[it & 1], ((it >> 1) - 1) & 1, abort_flag);
        if (ok) ok = mbar_wait(&vfull[vs], (it / VST) & 1, abort_flag);
        if (ok) ok = mbar_wait(&p_full[it & 1], (it >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t a = desc_rows<HD>(smem_u32(v_s + vs * STAGE)), b = desc_weights(smem_u32(p_s + (it & 1) * H * 2048));
        const int n = pages_of(at);
#pragma unroll
        for (int j = 0; j < 2 * H; ++j)
          if (j < n) {                                // a page: twice 32 keys
            umma_e4m3(tmem_base + O_COL + (it & 1) * 16, a + 2 * j * (32 * HD >> 4), b + 2 * j * (32 * 16 >> 4), idesc, j != 0);
            umma_e4m3(tmem_base + O_COL + (it & 1) * 16, a + (2 * j + 1) * (32 * HD >> 4), b + (2 * j + 1) * (32 * 16 >> 4), idesc, true);
          }
        umma_commit(&o_full[it & 1]);
        umma_commit(&vempty[vs]);
        advance(at);
      }
    }
  } else {
    // (no way out of this loop: the four warps meet at barriers; once a wait has run out the others are not waited for)
    pdl_wait();
    const int quarter = warp & 3, st = tid - (DE_THREADS - DE_SOFT);
    const int r = quarter * 32 + lane;                // key of the tile
    const int dim = HD == 128 ? r : quarter * 16 + lane;         // number of the head (heads of 64: a warp's first 16 lanes)
    const bool has_dim = HD == 128 || lane < 16;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) {
      if (ok) ok = mbar_wait(bar, parity & 1, abort_flag);
    };
    // what a head's weighted sum, relative to m, is multiplied with: 1 / l, the sink's share in l
    auto finish = [&](int head, float mm, float ll) {
      float f = 1.f;
      if (p.sink != nullptr) {
        const float sk = p.sink[head] * 1.4426950408889634f, top = fmaxf(mm, sk);
        f = exp2_fast(mm - top);
        ll = fmaf(ll, f, exp2_fast(sk - top));
      }
      return ll == 0.f ? 0.f : __fdividef(f, ll);                // (a sequence without a visible key: zeros)
    };
    // a thread's numbers of the queries of a sequence and kv head, 16 threads a head, asked for when the sequence before begins
    uint2 raw[HD / 64];
    auto fetch = [&](int head, int b) {
      const int g0 = head % p.n_gchunks * DE_GM, g = st >> 4, part = st & 15;
#pragma unroll
      for (int k = 0; k < HD / 64; ++k) {
        raw[k] = make_uint2(0u, 0u);
        if (head < heads && g < min(GM, G - g0))
          raw[k] = __ldcg(reinterpret_cast<const uint2*>(p.q + (size_t)b * p.ldq + (size_t)(head / p.n_gchunks * G + g0 + g) * HD + part * (HD / 16) + 4 * k));
      }
    };
    // those queries as two e4m3 terms (rows g and GM + g of the operand), and what the scores are scaled by
    auto prepare = [&](int buf) {
      const int g = st >> 4, part = st & 15;
      constexpr int N = HD / 16;
      float v[N];
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const uint2 u = raw[k / 4];
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
      // 2^(7 - (e - 127)); NaN for a row with an infinity, whose scores the formula leaves without a value (the terms would hold it
      // as 448)
      const float down = __uint_as_float(most == INFINITY ? 0x7fc00000u : (unsigned)(261 - e) << 23);
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
    if (n_tiles > 0) {
      fetch(at.head, at.b);
      prepare(0);
    }
    if (st < 2) shared_s[4 * st + 3] = 0;
    if (st == 0) {
      plan_s[0] = own_first;
      plan_s[1] = own_parts;
    }
    soft_sync();
    int seg = 0, k_first = 0;
    bool fresh = true;
    float m[GM], l[GM], N[GM], n_t[GM], n_new[GM], o[GM], fs[GM];
    int g0 = 0, GC = 0, head0 = 0, first_key = 0, last_key = 0;       // of the sequence
    int key = 0;                                      // this thread's first; a second is 128 behind it
    // the output of tile `it` (the newest, whose reference is n_new, or the one before it: n_t) into o
    auto gather = [&](int it, bool newest) {
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
        const float n = newest ? n_new[g] : n_t[g], top = fmaxf(N[g], n);
        o[g] = fmaf(o[g], exp2_fast(N[g] - top), x * exp2_fast(n - top));
        N[g] = top;
      }
    };
    for (int it = 0; it < n_tiles; ++it) {
      DecPlace next = at;
      const bool ends = advance(next) || it + 1 == n_tiles;
      if (fresh) {
        g0 = at.head % p.n_gchunks * DE_GM;
        GC = min(GM, G - g0);
        head0 = at.head / p.n_gchunks * G + g0;
        first_key = begin_s[at.b];
        last_key = pos_s[at.b];
        key = (first_key / E8_PAGE + 2 * H * at.k) * E8_PAGE + r;
        k_first = at.k;
        fetch(at.b + 1 < B ? at.head : at.head + 1, at.b + 1 < B ? at.b + 1 : 0);
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          m[g] = N[g] = n_t[g] = -1e30f;
          l[g] = o[g] = 0.f;
          fs[g] = fs_s[(seg & 1) * DE_GM + g];
        }
      }
      if (ends && it + 1 < n_tiles) prepare((seg + 1) & 1);
      wait(&sc_full[it % DE_SC], it / DE_SC);
      int kb[H], vb[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        kb[h] = sc_s[(it % DE_SC * H + h) * 256 + r];
        vb[h] = sc_s[(it % DE_SC * H + h) * 256 + 128 + r];
      }
      wait(&s_full[it & 1], it >> 1);
      __syncwarp();
      tc_fence_after_sync();
      float s[H][GM == 4 ? 8 : 16];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if (GM == 4) tmem_ld_32x8(lane_addr + (it & 1) * 32 + h * 16, s[h]);
        else tmem_ld_32x16(lane_addr + (it & 1) * 32 + h * 16, s[h]);
      }
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s_free[it & 1]);
        mbar_arrive(&sc_empty[it % DE_SC]);
      }
      bool seen[H];
      float bexp[H];
      float* red = red_s + (it & 1) * 4 * DE_GM;
      float most[GM];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        seen[h] = key + 128 * h >= first_key && key + 128 * h <= last_key;
        const float kpow = e4m3_scale(kb[h]);
        bexp[h] = (float)(vb[h] - 127);
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          const float x = fmaf(s[h][GM + g], 0.0625f, s[h][g]) * (kpow * fs[g]);
          s[h][g] = seen[h] ? x : -INFINITY;
        }
      }
#pragma unroll
      for (int g = 0; g < GM; ++g) most[g] = warp_max_redux(fmaxf(s[0][g] + bexp[0], s[H - 1][g] + bexp[H - 1]));
      if (lane == 0) {
#pragma unroll
        for (int g = 0; g < GM; g += 4)
          *reinterpret_cast<float4*>(red + quarter * DE_GM + g) = make_float4(most[g], most[g + 1], most[g + 2], most[g + 3]);
      }
      // (the sums while the others arrive)
#pragma unroll
      for (int g = 0; g < GM; ++g) {
        const float m_new = fmaxf(m[g], fmaxf(s[0][g], s[H - 1][g]));
        l[g] = fmaf(l[g], exp2_fast(m[g] - m_new), exp2_fast(s[0][g] - m_new) + (H == 2 ? exp2_fast(s[H - 1][g] - m_new) : 0.f));
        m[g] = m_new;
      }
      soft_sync();
#pragma unroll
      for (int g = 0; g < GM; g += 4) {
        float4 x = *reinterpret_cast<const float4*>(red + g);
#pragma unroll
        for (int k = 1; k < 4; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(red + k * DE_GM + g);
          x = make_float4(fmaxf(x.x, y.x), fmaxf(x.y, y.y), fmaxf(x.z, y.z), fmaxf(x.w, y.w));
        }
        n_new[g] = fmaxf(x.x, -1e30f);
        n_new[g + 1] = fmaxf(x.y, -1e30f);
        n_new[g + 2] = fmaxf(x.z, -1e30f);
        n_new[g + 3] = fmaxf(x.w, -1e30f);
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        uint32_t terms[TERMS][GM / 4];   // byte term * GM + g of the key's 16
        const float up = bexp[h] + 8.f;
#pragma unroll
        for (int g = 0; g < GM; g += 4) {
          __half2 w01 = __floats2half2_rn(exp2_fast(s[h][g] + up - n_new[g]), exp2_fast(s[h][g + 1] + up - n_new[g + 1]));
          __half2 w23 = __floats2half2_rn(exp2_fast(s[h][g + 2] + up - n_new[g + 2]), exp2_fast(s[h][g + 3] + up - n_new[g + 3]));
#pragma unroll
          for (int k = 0; k < TERMS; ++k) {
            const uint32_t a = e4m3_of_half2(w01), b = e4m3_of_half2(w23);
            terms[k][g / 4] = a | (b << 16);
            if (k + 1 < TERMS) {         // what the term leaves over, exact, times 16
              w01 = __hmul2(__hsub2(w01, half2_of_e4m3(a)), __float2half2_rn(16.f));
              w23 = __hmul2(__hsub2(w23, half2_of_e4m3(b)), __float2half2_rn(16.f));
            }
          }
        }
        *reinterpret_cast<uint4*>(p_s + ((it & 1) * H + h) * 2048 + r * 16) =
            GM == 4 ? make_uint4(terms[0][0], terms[1][0], terms[TERMS - 1][0], 0u)
                    : make_uint4(terms[0][0], terms[0][GM / 4 - 1], terms[1][0], terms[1][GM / 4 - 1]);
      }
      const int n_pages = pages_of(at);
      if (!seen[0] || !seen[H - 1]) {
        // value rows that nobody sees may hold anything: zeros, so that 0 times NaN does not come about
#pragma unroll
        for (int h = 0; h < H; ++h) {
          if (seen[h] || r / E8_PAGE + 2 * h >= n_pages) continue;
          wait(&vfull[it % VST], it / VST);
          uint8_t* row = v_s + it % VST * STAGE + (h * 128 + r) * HD;
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) *reinterpret_cast<uint4*>(row + k * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[it & 1]);
#pragma unroll 1
      for (int t = fresh ? it : it - 1; t < it + ends; ++t) gather(t, t == it);
#pragma unroll
      for (int g = 0; g < GM; ++g) n_t[g] = n_new[g];
      fresh = ends;
      key += 128 * H;
      if (ends) {
        // the sequence's result, or this block's part of it
        const bool whole = k_first == 0 && at.k + 1 == at.nk;
        // the threads' sums: to the warp's maximum, then half of the heads handed over at every step (a lane ends with one
        // head's), then the four warps'
        float mw[GM];
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          mw[g] = warp_max_redux(m[g]);
          l[g] *= exp2_fast(m[g] - mw[g]);
        }
#pragma unroll
        for (int x = 1, n = GM / 2; n > 0; x <<= 1, n >>= 1)
#pragma unroll
          for (int g = 0; g < n; ++g) {
            const float keep = (lane & x) ? l[g + n] : l[g], give = (lane & x) ? l[g] : l[g + n];
            l[g] = keep + __shfl_xor_sync(0xffffffffu, give, x);
            if (lane & x) mw[g] = mw[g + n];
          }
#pragma unroll
        for (int x = GM; x < 32; x <<= 1) l[0] += __shfl_xor_sync(0xffffffffu, l[0], x);
        int mine = 0;                                 // the head whose sum this lane has
#pragma unroll
        for (int x = 1, n = GM / 2; n > 0; x <<= 1, n >>= 1) mine += (lane & x) ? n : 0;
        if (lane < GM) ml_s[mine * 4 + quarter] = make_float2(mw[0], l[0]);
        soft_sync();
        const int side = k_first == 0 ? 1 : 0;        // (a block shares two sequences at most: one that began before, one after)
        const size_t part0 = ((size_t)blockIdx.x * 2 + side) * GM;
        // lane g: head g's maximum and sum over the warps, and its last factor
        const int gl = lane % GM;
        const float2 w0 = ml_s[gl * 4], w1 = ml_s[gl * 4 + 1], w2 = ml_s[gl * 4 + 2], w3 = ml_s[gl * 4 + 3];
        const float mm = fmaxf(fmaxf(w0.x, w1.x), fmaxf(w2.x, w3.x));
        const float ll = fmaf(w0.y, exp2_fast(w0.x - mm), w1.y * exp2_fast(w1.x - mm)) +
                         fmaf(w2.y, exp2_fast(w2.x - mm), w3.y * exp2_fast(w3.x - mm));
        float f = 1.f;
        if (whole) f = finish(head0 + min(gl, GC - 1), mm, ll);
        else if (st < GM) *reinterpret_cast<float2*>(p.part_ml + (part0 + gl) * 2) = make_float2(mm, ll);
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          // relative to m (in two steps: the values' powers may be far from the weights')
          const float half = exp2_fast(0.5f * (N[g] - 8.f - __shfl_sync(0xffffffffu, mm, g)));
          const float x = o[g] * half * half * __shfl_sync(0xffffffffu, f, g);
          if (g >= GC || !has_dim) continue;
          if (whole) p.out[(size_t)at.b * p.ldo + (size_t)(head0 + g) * HD + dim] = __float2bfloat16_rn(x);
          else p.part_acc[(part0 + g) * HD + dim] = x;
        }
        if (!whole && st == 0) {                      // (its ticket when the block's run is over)
          const long long unit = (long long)at.head * P + first[at.b];
          const int i0 = plan_s[1] ? plan_s[0] : block_of(unit);
          shared_s[4 * side] = at.head;
          shared_s[4 * side + 1] = at.b;
          shared_s[4 * side + 2] = i0;
          shared_s[4 * side + 3] = plan_s[1] ? plan_s[1] : block_of(unit + (at.nk == 1 ? 0 : at.nk)) - i0 + 1;
        }
        ++seg;
      }
      at = next;
    }
    soft_sync();
    if (st < 2) {
      // Tickets: both at once, at the run's end (in the run's middle a ticket holds the block up for 1.6 us).  Releases the
      // block's parts, which are behind the barrier; acquires those of the blocks before it for the other threads, behind the next.
      const int parts = shared_s[4 * st + 3];
      bool last = false;
      if (parts > 0) {
        int* ticket = p.tickets + (size_t)shared_s[4 * st + 1] * heads + shared_s[4 * st];
        int was;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(was) : "l"(ticket) : "memory");
        last = was == parts - 1;
        if (last) *ticket = 0;                        // for the next launch
      }
      last_s[st] = last;
    }
    soft_sync();
    for (int side = 0; side < 2; ++side) {
      if (!last_s[side]) continue;                    // (block-uniform)
      const int head = shared_s[4 * side], b = shared_s[4 * side + 1], i0 = shared_s[4 * side + 2], parts = shared_s[4 * side + 3];
      const int first_head = head / p.n_gchunks * G + head % p.n_gchunks * DE_GM;
      // The parts of 128 columns of four numbers at a time (or of all), by way of shared memory, which nothing else uses any more:
      // all of them on their way at once, a thread then adds up one column's.  37 parts take 2.7 us.  (In registers, six in
      // flight, 4.6; with more in flight longer, by the unrolled instructions, which a launch has to fetch anew.)
      const int cols = min(GM, G - head % p.n_gchunks * DE_GM) * H4;
#pragma unroll 1
      for (int c0 = 0; c0 < cols; c0 += JC) {
        const int g = min(c0 + st, cols - 1) / H4;
        float mm = -1e30f, ll = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int k0 = 0; k0 < parts; k0 += JN) {
          const int n = min(JN, parts - k0);
          soft_sync();                                // (those before are read)
          const float* src = p.part_acc + (size_t)(i0 + k0 + st / JC) * 2 * GM * HD + (c0 + st % JC) * 4;
          const uint32_t dst = smem_u32(smem + st % JC * 16);
#pragma unroll 2
          for (int k = st / JC; k < n; k += DE_SOFT / JC) {
            copy16(dst + k * JREC, src + (k0 + k == 0 ? GM * HD : 0));      // (a sequence's first part is the second of its block)
            src += DE_SOFT / JC * 2 * GM * HD;
          }
#pragma unroll 1
          for (int e = st; e < n * (GM / 2); e += DE_SOFT) {
            const int k = e / (GM / 2);
            const size_t x = (size_t)(i0 + k0 + k) * 2 + (k0 + k == 0 ? 1 : 0);
            copy16(smem_u32(smem + JC * 16 + e % (GM / 2) * 16) + k * JREC, p.part_ml + x * GM * 2 + e % (GM / 2) * 4);
          }
          copies_wait();
          soft_sync();
          const uint8_t* ml = smem + JC * 16 + g * 8;
          float top = mm;
#pragma unroll 4
          for (int k = 0; k < n; ++k) top = fmaxf(top, *reinterpret_cast<const float*>(ml + k * JREC));
          const float keep = exp2_fast(mm - top);
          mm = top;
          ll *= keep; a.x *= keep; a.y *= keep; a.z *= keep; a.w *= keep;
          const uint8_t* col = smem + st % JC * 16;
#pragma unroll 4
          for (int k = 0; k < n; ++k) {
            const float2 x = *reinterpret_cast<const float2*>(ml + k * JREC);
            const float4 v = *reinterpret_cast<const float4*>(col + k * JREC);
            const float w = exp2_fast(x.x - top);
            ll = fmaf(w, x.y, ll);
            a.x = fmaf(w, v.x, a.x); a.y = fmaf(w, v.y, a.y);
            a.z = fmaf(w, v.z, a.z); a.w = fmaf(w, v.w, a.w);
          }
        }
        if (st < JC && c0 + st < cols) {
          const float f = finish(first_head + g, mm, ll);
          *reinterpret_cast<uint2*>(p.out + (size_t)b * p.ldo + (size_t)first_head * HD + (c0 + st) * 4) =
              make_uint2(bf16_word(a.x * f, a.y * f), bf16_word(a.z * f, a.w * f));
        }
      }
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

inline int decode_e8_blocks() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms * DE_BLOCKS;
}

template <int HD, int GM>
int launch_decode_e8(const CUtensorMap& mk, const CUtensorMap& mv, const DecE8& p, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute((const void*)attention_decode_e4m3_kernel<HD, GM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)de_smem<HD>(DE_MAX_B));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute((const void*)attention_decode_e4m3_kernel<HD, GM>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             (int)cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return (int)e;
  launch_kernel(attention_decode_e4m3_kernel<HD, GM>, dim3(decode_e8_blocks()), dim3(DE_THREADS), de_smem<HD>(p.B), stream, mk, mv, p);
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
  const int gm = Hq / Hkv <= 4 ? 4 : DE_GM;
  return (long long)decode_e8_blocks() * 2 * gm * (hd + 2);
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
  if ((long long)max_pages * (B < DE_MAX_B ? B : DE_MAX_B) > 0x7fffffffLL) return DLGO_ERR_SIZE;       // (a launch's tiles are counted in 32 bits)
  if (B > 1 && (ldq < 0 || ldo < Hq * hd)) return DLGO_ERR_SIZE;        // (rows of the output that meet would depend on the blocks' order)
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
  p.room = decode_e8_blocks() / (Hkv * p.n_gchunks);
  p.one_by_room = p.room > 0 ? 1.f / p.room : 0.f;
  p.part_acc = scratch;
  p.part_ml = scratch + (size_t)decode_e8_blocks() * 2 * gm * hd;
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

// The same, called with a record (e4m3.cuh).
DLGO_EXPORT int dlgo_attention_decode_e4m3_record(const long long* r) { return call_record(dlgo_attention_decode_e4m3, r); }

// 1 if a bounded wait ran out since the last call (clears the word).
DLGO_EXPORT int dlgo_attention_decode_e4m3_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_decode_e4m3_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_decode_e4m3_error, &zero, sizeof(int));
  return v;
}
