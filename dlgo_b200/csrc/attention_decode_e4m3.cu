// Decode attention over the 8-bit cache (e4m3 rows with a power of two each, see e4m3.cuh) on the tensor cores (warp-level
// mma.sync, m16n8k16, float16 operands, fp32 sums).
//
// One new token per sequence; scores s_j = q . k_j * scale over the visible positions, softmax, weighted sum of the values
// (models/llm/forward.go:258-278, with rows that take hd + 1 bytes instead of 2 hd).  With k_j = K_j 2^a_j and
// v_j = V_j 2^b_j, K and V being the stored e4m3 numbers, which float16 holds exactly:
//
//   s_j = (q / 2^c . K_j) * (scale log2(e) 2^c 2^a_j)         c per query row, so that its largest number lies in [2^14, 2^15)
//   p_j = 2^(s_j - m),   w_j = p_j 2^(b_j - B) 2^f,   l = sum_j p_j,   O = sum_j w_j V_j,   out = O 2^(B - f) / l
//
// The queries lose nothing in float16 but what lies 2^29 below a row's largest number.  The weights of the values carry the
// rows' powers, so they are scaled apart from the softmax (a row of small values may hold all of its weight): B is the
// largest power among the values, 2^f brings the largest weight to 2^10.  Both references, m and N = m + B - f, follow the
// maxima lazily: only when a p_j passes 2^8 or a w_j 2^15 are they set anew (a vote per tile) and the sums rescaled.  A
// weight in float16 has 11 bits down to 2^-24 of the largest, and its last bit at 2^-34.
//
// Bound by the rows, which are read once; next to them by issue slots: a tile of 32 keys takes some 300 instructions, of which
// 1 per two numbers converts e4m3 to float16.  A step has one query row per head, so the keys (of the scores) and the numbers
// of a head (of the output) are the MMA's 16 rows and up to eight query heads of a kv head its 8 columns.  Nothing goes through
// shared memory on the way in: the k index of an MMA may be any permutation of a head's numbers as long as q and k agree, and
// so may the order of the keys and of the output's numbers.  Lane (r = lane / 4, c = lane % 4) loads 16-byte pieces of rows as
// they lie in the pages:
//   scores  numbers [64 v + 16 c, + 16) of keys 4r .. 4r + 3; a 32-bit word is a k-step's share of a key.  Key 4r + 2i + h is row
//           r + 8h of row tile i, so the lane's scores (heads 2c, 2c + 1) belong to four neighbouring keys, whose scale bytes
//           are one word
//   values  numbers [r HD/8, + HD/8) of keys 8c .. 8c + 7; a byte permute pairs two keys' numbers before they are converted.  The
//           weights reach the second MMA's layout by a transposition of 8 x 8 blocks (movmatrix)
//
// Work is shared evenly: the tiles (32 keys) of all sequences, one sequence after another, are numbered through, and each of
// a kv head's blocks takes an equal run of them, as many blocks as are resident at once.  A run may hold several sequences or
// a part of one; parts go through scratch memory, and the block that takes a sequence's last ticket adds them up in the order
// of the blocks; nobody waits for another block.
#include <math.h>

#include "attention_combine.cuh"
#include "common.cuh"
#include "e4m3.cuh"

namespace dlgo {

constexpr int DE_THREADS = 128;
constexpr int DE_WARPS = DE_THREADS / 32;
constexpr int DE_GM = 8;              // query heads of a kv head per block
constexpr int DE_TK = 32;             // keys of a tile
constexpr int DE_SEGS = 4;            // sequences of a round
constexpr int DE_MIN_TILES = 8;       // a block's least run: two tiles a warp
constexpr int DE_MAX_B = 2048;        // sequences of a launch (their first tiles lie in shared memory)

struct DecE8 {
  const __nv_bfloat16* q;  // [B][ldq]
  int ldq;
  const uint8_t* kpages;   // [pages][Hkv][64][HD]
  const uint8_t* vpages;
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
  float* part_acc;         // [heads x blocks][2][GM][HD]
  float* part_ml;          // [heads x blocks][2][GM][2]
  int* tickets;            // [B][heads], zero between launches
};

// Sequence i's position and row of the page table, kept within the table whatever the caller's numbers are.
__device__ __forceinline__ int decode_pos(const DecE8& p, int i) { return min(max(p.token_pos[i], -1), p.max_pages * E8_PAGE - 1); }
__device__ __forceinline__ const int* decode_pages(const DecE8& p, int i) {
  return p.page_table + (size_t)min(max(p.seq_slot[i], 0), p.n_slots - 1) * p.max_pages;
}

// d += A (16 x 16) * B (16 x 8), float16 with fp32 sums
__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 block of 16-bit numbers transposed (lane (r, c) holds row r, columns 2c and 2c + 1)
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_word(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf16_word(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// byte k of four scale bytes as the power of two
__device__ __forceinline__ float byte_power(uint32_t w, int k) {
  return __uint_as_float(k < 3 ? (w << (23 - 8 * k)) & 0x7f800000u : (w >> 1) & 0x7f800000u);
}

template <int HD> struct RowPiece;                 // a lane's HD / 8 numbers of a value row
template <> struct RowPiece<64> { using T = uint2; };
template <> struct RowPiece<128> { using T = uint4; };
__device__ __forceinline__ uint32_t piece_word(const uint2& u, int i) { return i == 0 ? u.x : u.y; }
__device__ __forceinline__ uint32_t piece_word(const uint4& u, int i) { return i == 0 ? u.x : (i == 1 ? u.y : (i == 2 ? u.z : u.w)); }

constexpr float DE_NONE = -3e38f;    // the references before the first key
template <int HD> struct DecState {
  float o[HD / 16][4];     // tile i: numbers r HD/8 + 2i (first two) and + 2i + 1 of heads 2c, 2c + 1
  float m[2], n[2], l[2], f[2];      // of heads 2c, 2c + 1: m, N, this lane's share of l, 2^f
  float unit;              // 2^-B
  int top;                 // B + 127
};

// Tiles first_tile, first_tile + DE_WARPS, ... below n_tiles (tile i: keys [32 i, 32 i + 32) of the sequence whose pages are
// `page_row[]`), keys in [t_begin, t_end) only.  row_scale: of heads 2c, 2c + 1.
template <int HD>
__device__ __forceinline__ void decode_tiles_e8(const DecE8& p, const int* __restrict__ page_row, int kvh, int first_tile, int n_tiles,
                                                int t_begin, int t_end, int lane, const uint32_t (&qb)[HD / 16][2],
                                                const float (&row_scale)[2], DecState<HD>& st) {
  using VP = typename RowPiece<HD>::T;
  constexpr int KP = HD / 64;          // 16-byte pieces of a lane's share of a key row
  const int r = lane >> 2, c = lane & 3;
  for (int tile = first_tile; tile < n_tiles; tile += DE_WARPS) {
    const int t0 = tile * DE_TK;
    const int page = min(readable_page(page_row, t0 / E8_PAGE), p.n_pages - 1);
    const size_t row0 = ((size_t)page * p.Hkv + kvh) * E8_PAGE + (t0 % E8_PAGE);
    const bool full = t0 >= t_begin && t0 + DE_TK <= t_end;      // (warp-uniform)
    // every load of the tile is requested before any arithmetic
    uint4 ku[4][KP];
    const uint8_t* kp = p.kpages + (row0 + 4 * r) * HD + c * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int v = 0; v < KP; ++v) ku[k][v] = *reinterpret_cast<const uint4*>(kp + k * HD + v * 64);
    const uint32_t kb = *reinterpret_cast<const uint32_t*>(p.kscales + row0 + 4 * r);
    const uint32_t vb = *reinterpret_cast<const uint32_t*>(p.vscales + row0 + 4 * r);
    VP vu[8];
    const uint8_t* vp = p.vpages + (row0 + 8 * c) * HD + r * (HD / 8);
    if (full) {
#pragma unroll
      for (int k = 0; k < 8; ++k) vu[k] = *reinterpret_cast<const VP*>(vp + k * HD);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {    // (rows that nobody sees may hold anything, NaN too: zeros in their place)
        const int t = t0 + 8 * c + k;
        vu[k] = VP{};
        if (t >= t_begin && t < t_end) vu[k] = *reinterpret_cast<const VP*>(vp + k * HD);
      }
    }
    float s[2][4];                     // row tile i: keys 4r + 2i (first two) and + 2i + 1, heads 2c, 2c + 1
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const uint32_t w0 = piece_word(ku[2 * i][kk >> 2], kk & 3), w1 = piece_word(ku[2 * i + 1][kk >> 2], kk & 3);
        mma_half(s[i], e4m3_low_half2(w0), e4m3_low_half2(w1), e4m3_high_half2(w0), e4m3_high_half2(w1), qb[kk][0], qb[kk][1]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float power = byte_power(kb, k);
      const int t = t0 + 4 * r + k;
      const bool seen = full || (t >= t_begin && t < t_end);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& x = s[k >> 1][(k & 1) * 2 + e];
        x = seen ? x * (power * row_scale[e]) : -INFINITY;
      }
    }
    float w[2][4];
    auto weights = [&](float (&add)[2], float& most_p, float& most_w) {
      most_p = most_w = 0.f;
      add[0] = add[1] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = t0 + 4 * r + k;
        const float power = (full || (t >= t_begin && t < t_end)) ? byte_power(vb, k) * st.unit : 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float pr = exp2_fast(s[k >> 1][(k & 1) * 2 + e] - st.m[e]);
          float& x = w[k >> 1][(k & 1) * 2 + e];
          add[e] += pr;
          x = pr * power * st.f[e];
          most_p = fmaxf(most_p, pr);
          most_w = fmaxf(most_w, x);
        }
      }
    };
    float add[2], most_p, most_w;
    weights(add, most_p, most_w);
    if (__any_sync(0xffffffffu, most_p > 256.f || most_w > 32768.f)) {
      // the references anew, at least at this tile's maxima
      int high = 8;
      float mx[2] = {DE_NONE, DE_NONE}, nx[2] = {DE_NONE, DE_NONE};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = t0 + 4 * r + k, byte = (int)((vb >> (8 * k)) & 255u);
        if (full || (t >= t_begin && t < t_end)) high = max(high, byte);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = s[k >> 1][(k & 1) * 2 + e];
          mx[e] = fmaxf(mx[e], x);
          nx[e] = fmaxf(nx[e], x + (float)(byte - 127) - 10.f);
        }
      }
      high = max(st.top, __reduce_max_sync(0xffffffffu, min(high, 246)));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], o));
          nx[e] = fmaxf(nx[e], __shfl_xor_sync(0xffffffffu, nx[e], o));
        }
        const float m_new = fmaxf(st.m[e], mx[e]);
        const float n_new = fmaxf(fmaxf(st.n[e], nx[e]), m_new + (float)(high - 127) - 126.f);
        const float keep = exp2_fast(st.n[e] - n_new);
        st.l[e] *= exp2_fast(st.m[e] - m_new);
        st.m[e] = m_new;
        st.n[e] = n_new;
        st.f[e] = exp2_fast(m_new + (float)(high - 127) - n_new);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          st.o[i][e] *= keep;
          st.o[i][2 + e] *= keep;
        }
      }
      st.top = high;
      st.unit = e4m3_inverse(high);
      weights(add, most_p, most_w);
    }
    st.l[0] += add[0];
    st.l[1] += add[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // keys 8c + 2i, 8c + 2i + 4 of head r, and the ones behind them
      const uint32_t b0 = transposed(half2_word(w[i][0], w[i][1])), b1 = transposed(half2_word(w[i][2], w[i][3]));
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {            // word j of the lane's piece: four numbers, two row tiles
        const uint32_t k0 = piece_word(vu[2 * i], j), k1 = piece_word(vu[2 * i + 4], j);
        const uint32_t k2 = piece_word(vu[2 * i + 1], j), k3 = piece_word(vu[2 * i + 5], j);
        const uint32_t p01 = __byte_perm(k0, k1, 0x5140), p23 = __byte_perm(k0, k1, 0x7362);
        const uint32_t q01 = __byte_perm(k2, k3, 0x5140), q23 = __byte_perm(k2, k3, 0x7362);
        mma_half(st.o[2 * j], e4m3_low_half2(p01), e4m3_high_half2(p01), e4m3_low_half2(q01), e4m3_high_half2(q01), b0, b1);
        mma_half(st.o[2 * j + 1], e4m3_low_half2(p23), e4m3_high_half2(p23), e4m3_low_half2(q23), e4m3_high_half2(q23), b0, b1);
      }
    }
  }
}

template <int HD> constexpr size_t decode_e8_smem(int B, int gm) {
  return (size_t)(B + 4) / 4 * 16 + (size_t)DE_SEGS * DE_WARPS * gm * (HD + 4 + 2) * 4;
}

template <int HD>
__global__ void __launch_bounds__(DE_THREADS, HD <= 64 ? 4 : 3) attention_decode_e4m3_kernel(DecE8 p) {
  constexpr int AR = HD + 4;                          // AR: floats from one output row to the next in shared memory
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int last[DE_SEGS], longest;
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int B = p.B, G = p.Hq / p.Hkv;
  const int kvh = blockIdx.y / p.n_gchunks, gc = blockIdx.y - kvh * p.n_gchunks;
  const int GM = min(DE_GM, G), g0 = gc * DE_GM, GC = min(DE_GM, G - g0);
  const int head0 = kvh * G + g0;
  int* first = reinterpret_cast<int*>(smem);                                  // [B + 1] first tile of each sequence
  float* acc_s = reinterpret_cast<float*>(smem + (size_t)(B + 4) / 4 * 16);   // [DE_SEGS][DE_WARPS][GM][AR]
  float* ml_s = acc_s + (size_t)DE_SEGS * DE_WARPS * GM * AR;                 // [DE_SEGS][DE_WARPS][GM][2]

  // the cut, from the step's own inputs
  if (warp == 0) {
    int sum = 0, most = 0;
    if (lane == 0) first[0] = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
      int n = 0;
      if (b0 + lane < B) {
        const int pos = decode_pos(p, b0 + lane);
        n = pos / DE_TK - first_visible(pos, p.span) / DE_TK + 1;
        most = max(most, n);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += up;
      }
      n += sum;
      if (b0 + lane < B) first[b0 + lane + 1] = n;
      sum = __shfl_sync(0xffffffffu, n, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) longest = most;
  }
  __syncthreads();
  const unsigned P = first[B];
  // a block per sequence where none is longer than a block's least run
  const bool whole_only = B <= (int)gridDim.x && longest <= DE_MIN_TILES;
  const unsigned nb = whole_only ? B : min(gridDim.x, max(1u, (P + DE_MIN_TILES - 1) / DE_MIN_TILES));   // (<= P: no run is empty)
  if (blockIdx.x >= nb) return;
  auto start_of = [&](unsigned i) { return whole_only ? first[i] : (int)((unsigned long long)i * P / nb); };
  auto block_of = [&](unsigned tile) { return (int)(((unsigned long long)(tile + 1) * nb - 1) / P); };
  const int lo = start_of(blockIdx.x), hi = start_of(blockIdx.x + 1);
  int b = 0;
  for (int step = 1024; step > 0; step >>= 1)                              // the sequence that holds tile lo
    if (b + step < B && first[b + step] <= lo) b += step;
  static_assert(DE_MAX_B <= 2 * 1024, "the search covers them");
  pdl_wait();

  for (; b < B && first[b] < hi; b += DE_SEGS) {
    int ns = 1;
    while (ns < DE_SEGS && b + ns < B && first[b + ns] < hi) ++ns;
    for (int s = 0; s < ns; ++s) {
      const int begin = max(lo, first[b + s]), end = min(hi, first[b + s + 1]);
      const int pos = decode_pos(p, b + s), t_begin = first_visible(pos, p.span);
      const int rebase = t_begin / DE_TK - first[b + s];        // to the sequence's own tile numbers
      // head r's query in float16, its largest number in [2^14, 2^15)
      uint32_t qb[HD / 16][2];
      float row_scale[2];
      {
        float x[HD / 4];
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 4; k += 8) {
          uint4 u = make_uint4(0u, 0u, 0u, 0u);
          if (r < GC)
            u = __ldcg(reinterpret_cast<const uint4*>(p.q + (size_t)(b + s) * p.ldq + (size_t)(head0 + r) * HD + (k / 16) * 64 + c * 16 + k % 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t word = piece_word(u, e);
            x[k + 2 * e] = __uint_as_float(word << 16);
            x[k + 2 * e + 1] = __uint_as_float(word & 0xffff0000u);
            most = fmaxf(most, fmaxf(fabsf(x[k + 2 * e]), fabsf(x[k + 2 * e + 1])));
          }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max((int)(__float_as_uint(most) >> 23), 16), 254);
        const float down = __uint_as_float((unsigned)(268 - e) << 23);          // 2^(14 - (e - 127))
        const float up = __uint_as_float((unsigned)(e - 14) << 23) * p.scale_log2e;
        row_scale[0] = __shfl_sync(0xffffffffu, up, 8 * c);
        row_scale[1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          qb[kk][0] = half2_word(x[4 * kk] * down, x[4 * kk + 1] * down);
          qb[kk][1] = half2_word(x[4 * kk + 2] * down, x[4 * kk + 3] * down);
        }
      }
      DecState<HD> st;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) st.o[i][0] = st.o[i][1] = st.o[i][2] = st.o[i][3] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        st.m[e] = st.n[e] = DE_NONE;
        st.l[e] = 0.f;
        st.f[e] = 1.f;
      }
      st.unit = 1.f;
      st.top = 8;
      decode_tiles_e8<HD>(p, decode_pages(p, b + s), kvh, begin + rebase + ((warp - (begin - lo)) & (DE_WARPS - 1)), end + rebase, t_begin,
                          pos + 1, lane, qb, row_scale, st);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) st.l[e] += __shfl_xor_sync(0xffffffffu, st.l[e], o);
        const int g = 2 * c + e;
        if (g >= GC) continue;
        // from now on relative to m (in two steps: the values' powers may be far from the weights')
        float* as = acc_s + (((size_t)s * DE_WARPS + warp) * GM + g) * AR + r * (HD / 8);
        const float f = exp2_fast(0.5f * (st.n[e] - st.m[e]));
#pragma unroll
        for (int i = 0; i < HD / 16; i += 2)
          *reinterpret_cast<float4*>(as + 2 * i) = make_float4(st.o[i][e] * f * f, st.o[i][2 + e] * f * f, st.o[i + 1][e] * f * f,
                                                               st.o[i + 1][2 + e] * f * f);
        if (r == 0) {
          float* ml = ml_s + ((s * DE_WARPS + warp) * GM + g) * 2;
          ml[0] = st.m[e];
          ml[1] = st.l[e];
        }
      }
    }
    __syncthreads();
    bool shared_any = false;
    for (int s = 0; s < ns; ++s) shared_any |= first[b + s] < lo || first[b + s + 1] > hi;
    constexpr int H4 = HD / 4;
    auto store4 = [&](int seq, int g, int d, float4 a, float ll, float mm) {
      float f = 1.f;
      if (p.sink != nullptr) {
        const float sk = p.sink[head0 + g] * 1.4426950408889634f, top = fmaxf(mm, sk);
        f = exp2_fast(mm - top);
        ll = fmaf(ll, f, exp2_fast(sk - top));
      }
      f = ll == 0.f ? 0.f : f / ll;               // (a sequence without a visible key: zeros)
      *reinterpret_cast<uint2*>(p.out + (size_t)seq * p.ldo + (size_t)(head0 + g) * HD + d) =
          make_uint2(bf16_word(a.x * f, a.y * f), bf16_word(a.z * f, a.w * f));
    };
    for (int idx = tid; idx < ns * GC * H4; idx += DE_THREADS) {
      const int d = idx % H4 * 4, g = idx / H4 % GC, s = idx / (H4 * GC);
      const float* ml = ml_s + (s * DE_WARPS * GM + g) * 2;
      const float* as = acc_s + ((size_t)s * DE_WARPS * GM + g) * AR + d;
      float mm = -INFINITY, ll = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < DE_WARPS; ++w) mm = fmaxf(mm, ml[w * GM * 2]);
#pragma unroll
      for (int w = 0; w < DE_WARPS; ++w) {
        const float mw = ml[w * GM * 2];
        const float cw = exp2_fast(mw - mm);
        const float4 u = *reinterpret_cast<const float4*>(as + w * GM * AR);
        a.x = fmaf(cw, u.x, a.x); a.y = fmaf(cw, u.y, a.y); a.z = fmaf(cw, u.z, a.z); a.w = fmaf(cw, u.w, a.w);
        ll = fmaf(cw, ml[w * GM * 2 + 1], ll);
      }
      if (first[b + s] >= lo && first[b + s + 1] <= hi) {
        store4(b + s, g, d, a, ll, mm);
      } else {        // a block shares at most two sequences: one that began before its run, one that begins in it
        const size_t at = (((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + (first[b + s] >= lo ? 1 : 0)) * GM + g;
        *reinterpret_cast<float4*>(p.part_acc + at * HD + d) = a;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mm, ll);
      }
    }
    if (shared_any) {
      __syncthreads();
      if (tid < ns) {
        const int seq = b + tid;
        int mine = 0;
        if (first[seq] < lo || first[seq + 1] > hi) {
          const int n = block_of(first[seq + 1] - 1) - block_of(first[seq]) + 1;
          int* ticket = p.tickets + (size_t)seq * gridDim.y + blockIdx.y;
          // releases the block's parts, which are behind the barrier; acquires those of the blocks before it for the whole
          // block, behind the next one
          int before;
          asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
          if (before == n - 1) {
            *ticket = 0;              // for the next launch
            mine = 1;
          }
        }
        last[tid] = mine;
      }
      __syncthreads();
      for (int s = 0; s < ns; ++s) {
        const int seq = b + s;
        if ((first[seq] >= lo && first[seq + 1] <= hi) || !last[s]) continue;           // (block-uniform)
        const int i0 = block_of(first[seq]), n = block_of(first[seq + 1] - 1) - i0 + 1;
        // a thread per four numbers, or 2, 4, 8 threads that share the parts; four parts in flight each
        const int cols = GC * H4;
        int tpc = 1;
        while (tpc < 8 && cols * tpc * 2 <= DE_THREADS) tpc *= 2;
        for (int c0 = 0; c0 < cols; c0 += DE_THREADS / tpc) {
          const int col = c0 + tid / tpc;
          const int g = min(col, cols - 1) / H4, d = min(col, cols - 1) % H4 * 4;
          float mm = -INFINITY, ll = 0.f;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k0 = tid % tpc; k0 < n; k0 += 4 * tpc) {
            float2 ml[4];
            float4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = k0 + j * tpc;
              const size_t at = (((size_t)blockIdx.y * gridDim.x + i0 + min(k, n - 1)) * 2 + (k == 0 ? 1 : 0)) * GM + g;
              ml[j] = k < n ? __ldcg(reinterpret_cast<const float2*>(p.part_ml) + at) : make_float2(-INFINITY, 0.f);
              v[j] = k < n ? __ldcg(reinterpret_cast<const float4*>(p.part_acc + at * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float top = mm;
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, ml[j].x);
            if (top == -INFINITY) continue;
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
          for (int o = tpc >> 1; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, mm, o), top = fmaxf(mm, m2);
            const float k1 = mm == -INFINITY ? 0.f : exp2_fast(mm - top), k2 = m2 == -INFINITY ? 0.f : exp2_fast(m2 - top);
            mm = top;
            ll = ll * k1 + __shfl_xor_sync(0xffffffffu, ll, o) * k2;
            a.x = a.x * k1 + __shfl_xor_sync(0xffffffffu, a.x, o) * k2;
            a.y = a.y * k1 + __shfl_xor_sync(0xffffffffu, a.y, o) * k2;
            a.z = a.z * k1 + __shfl_xor_sync(0xffffffffu, a.z, o) * k2;
            a.w = a.w * k1 + __shfl_xor_sync(0xffffffffu, a.w, o) * k2;
          }
          if (col < cols && tid % tpc == 0) store4(seq, g, d, a, ll, mm);
        }
      }
    }
    __syncthreads();            // the round's shared memory is free again
  }
}

// blocks of a kv head (or chunk of its heads) in a launch: as many as are resident at once
inline int decode_e8_blocks(int hd, int heads) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int n = (hd <= 64 ? 4 : 3) * sms / heads;
  return n < 1 ? 1 : n;
}

template <int HD>
int launch_decode_e8(const DecE8& p, cudaStream_t stream) {
  const int heads = p.Hkv * p.n_gchunks, G = p.Hq / p.Hkv;
  const size_t smem = decode_e8_smem<HD>(p.B, G < DE_GM ? G : DE_GM);
  cudaError_t e = cudaFuncSetAttribute((const void*)attention_decode_e4m3_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  launch_kernel(attention_decode_e4m3_kernel<HD>, dim3(decode_e8_blocks(HD, heads), heads), dim3(DE_THREADS), smem, stream, p);
  return launch_status();
}

}  // namespace dlgo

using namespace dlgo;

// Floats of scratch that a launch needs, whatever the number of sequences.
DLGO_EXPORT long long dlgo_attention_decode_e4m3_scratch(int Hq, int Hkv, int hd) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv) return 0;
  const int G = Hq / Hkv, heads = Hkv * ((G + DE_GM - 1) / DE_GM), gm = G < DE_GM ? G : DE_GM;
  return (long long)heads * decode_e8_blocks(hd, heads) * 2 * gm * (hd + 2);
}

// q[B, .] bf16 (row stride ldq, head h at column h * hd), one token per sequence at position token_pos[b] whose key and
// value are in the cache; out[B, .] bf16 (row stride ldo).  `scratch` as above; `tickets` [B * Hkv * ceil(Hq / Hkv / 8)]
// zero, and left zero; `sink` [Hq] fp32 or null.
DLGO_EXPORT int dlgo_attention_decode_e4m3(const void* q, int B, int ldq, const void* kpages, const void* vpages, const void* kscales,
                                           const void* vscales, int n_pages, const int* page_table, int n_slots, int max_pages,
                                           const int* seq_slot, const int* token_pos, void* out, int ldo, int Hq, int Hkv, int hd, int span, float scale,
                                           const float* sink, float* scratch, int* tickets, cudaStream_t stream) {
  if (B <= 0) return DLGO_OK;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || (hd != 64 && hd != 128) || n_pages <= 0 || n_slots <= 0 || max_pages <= 0) return DLGO_ERR_SIZE;
  if ((ldq & 7) || (ldo & 3) || ((uintptr_t)q & 15) || ((uintptr_t)out & 7) || ((uintptr_t)kpages & 15) || ((uintptr_t)vpages & 15) ||
      ((uintptr_t)kscales & 7) || ((uintptr_t)vscales & 7) || ((uintptr_t)scratch & 15) || scratch == nullptr || tickets == nullptr)
    return DLGO_ERR_ALIGN;
  const int G = Hq / Hkv;
  DecE8 p;
  p.ldq = ldq;
  p.kpages = (const uint8_t*)kpages; p.vpages = (const uint8_t*)vpages;
  p.kscales = (const uint8_t*)kscales; p.vscales = (const uint8_t*)vscales;
  p.page_table = page_table; p.n_slots = n_slots; p.max_pages = max_pages; p.n_pages = n_pages;
  p.ldo = ldo; p.Hq = Hq; p.Hkv = Hkv;
  p.n_gchunks = (G + DE_GM - 1) / DE_GM;
  p.span = span; p.scale_log2e = scale * 1.4426950408889634f; p.sink = sink;
  const int heads = Hkv * p.n_gchunks, gm = G < DE_GM ? G : DE_GM;
  if (heads > 65535) return DLGO_ERR_SIZE;
  p.part_acc = scratch;
  p.part_ml = scratch + (size_t)heads * decode_e8_blocks(hd, heads) * 2 * gm * hd;
  for (int b0 = 0; b0 < B; b0 += DE_MAX_B) {       // (one launch as a rule; they run one after another and share the scratch)
    p.B = B - b0 < DE_MAX_B ? B - b0 : DE_MAX_B;
    p.q = (const __nv_bfloat16*)q + (size_t)b0 * ldq;
    p.out = (__nv_bfloat16*)out + (size_t)b0 * ldo;
    p.seq_slot = seq_slot + b0;
    p.token_pos = token_pos + b0;
    p.tickets = tickets + (size_t)b0 * heads;
    const int st = hd == 64 ? launch_decode_e8<64>(p, stream) : launch_decode_e8<128>(p, stream);
    if (st != DLGO_OK) return st;
  }
  return DLGO_OK;
}
