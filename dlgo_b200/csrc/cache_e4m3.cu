// Writing the 8-bit cache (e4m3 rows with a power of two each, see e4m3.cuh) and reading it back.
//
// The reference stores a position's key and value rows as they are (models/llm/forward.go:246-257, memory/kvcache.go:30-36)
// and reads them back for every later token; here a row takes hd + 1 bytes.
#include <math.h>

#include "common.cuh"
#include "e4m3.cuh"

namespace dlgo {

// Set when a token's position had no page in the table: nothing is written through it, and the host reads the word
// (dlgo_cache_e4m3_error).
__device__ int g_cache_e4m3_error = 0;

struct WriteE8 {
  void* qkv;                 // [T, ld]: query heads, key heads, value heads
  int ld;
  const float* cos_t;        // [positions][rot / 2]
  const float* sin_t;
  const int* token_pos;
  const int* token_seq;
  const int* seq_slot;
  const int* page_table;     // [slots][max_pages]
  int n_seqs, n_slots, max_pages, n_pages, n_positions;
  uint8_t* kpages;           // [n_pages][Hkv][64][hd]
  uint8_t* vpages;
  uint8_t* kscales;          // [n_pages][Hkv][64]
  uint8_t* vscales;
  __nv_bfloat16* q;          // [T][Hq * hd]
  int T, Hq, Hkv, rot, interleaved, write_cache, clear;
};

// Where token t's row goes: the row's number in [n_pages][Hkv][64] for kv head 0, or -1 (nothing is written).  A position
// that the tables of cosines do not have counts as one without a page, and is turned as position 0.
__device__ __forceinline__ long long e8_row(const WriteE8& p, int t, int& pos, bool report) {
  const bool in_tables = pos >= 0 && (p.rot == 0 || pos < p.n_positions);
  int page = -1;
  if (in_tables && p.write_cache) {
    const int seq = p.token_seq[t], slot = seq >= 0 && seq < p.n_seqs ? p.seq_slot[seq] : -1, idx = pos / E8_PAGE;
    if (slot >= 0 && slot < p.n_slots && idx < p.max_pages) page = p.page_table[(size_t)slot * p.max_pages + idx];
  }
  const bool bad = !in_tables || (p.write_cache && (page < 0 || page >= p.n_pages));
  if (bad && report) atomicExch(&g_cache_e4m3_error, 1);
  if (!in_tables) pos = 0;
  if (bad || !p.write_cache) return -1;
  return (long long)page * p.Hkv * E8_PAGE + pos % E8_PAGE;
}

// eight numbers as they lie in memory, and as fp32
template <typename T> struct Eight;
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldcg(reinterpret_cast<const float4*>(p));
    b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void numbers(float (&o)[8]) const {
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
  }
};
template <> struct Eight<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = __ldcg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void numbers(float (&o)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
__device__ __forceinline__ void clear8(float* p) {
  reinterpret_cast<float4*>(p)[0] = make_float4(0.f, 0.f, 0.f, 0.f);
  reinterpret_cast<float4*>(p)[1] = make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void clear8(__nv_bfloat16*) {}

// Heads of 64 or 128 rotated whole in the split-half pairing (i, i + hd/2).  HD/16 lanes take a head, each eight numbers
// of its first half and the eight they pair with: 16-byte accesses, the row's maximum from two or three shuffles, and the
// lane's cosines and sines stay in registers over all heads that it takes of its token.  `per_token` warps share a token's
// heads: all of them for one token or a few, one where tokens alone fill the GPU.
//
// Bound by memory from some thousand tokens on: 16,384 tokens of 32 + 2 * 8 heads of 128 from bfloat16 64.7 us, 89 % of the
// copy rate (378 MB).  Below that it is one chain of loads and a launch: 8 tokens of 32 + 2 * 8 heads of 64 1.4 us, some 1,300
// (from bfloat16) 4.2 us.
constexpr int WE_WARPS = 4;

template <typename T, int HD>
__global__ void __launch_bounds__(WE_WARPS * 32) write_e4m3_kernel(WriteE8 p, int per_token) {
  pdl_launch_dependents();
  constexpr int LANES = HD / 16, HEADS = 32 / LANES;      // lanes of a head, heads of a warp at a time
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * WE_WARPS + (threadIdx.x >> 5);
  const int t = (int)(w / per_token), part = (int)(w % per_token);
  if (t >= p.T) return;                                    // (whole warps)
  const int i = (lane % LANES) * 8;
  const int n_heads = p.Hq + (p.write_cache || p.clear ? 2 * p.Hkv : 0);
  int pos = p.token_pos[t];
  const long long row0 = e8_row(p, t, pos, part == 0 && lane == 0);
  float c[8], s[8];
  {
    const float* ct = p.cos_t + (size_t)pos * (HD / 2) + i;
    const float* st = p.sin_t + (size_t)pos * (HD / 2) + i;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      const float4 a = *reinterpret_cast<const float4*>(ct + k), b = *reinterpret_cast<const float4*>(st + k);
      c[k] = a.x; c[k + 1] = a.y; c[k + 2] = a.z; c[k + 3] = a.w;
      s[k] = b.x; s[k + 1] = b.y; s[k + 2] = b.z; s[k + 3] = b.w;
    }
  }
  pdl_wait();
  T* row = (T*)p.qkv + (size_t)t * p.ld + i;
  const int stride = per_token * HEADS;
  Eight<T> ahead[2] = {};
  const int head_first = part * HEADS + lane / LANES;
  if (head_first < n_heads) {
    ahead[0].load(row + (size_t)head_first * HD);
    ahead[1].load(row + (size_t)head_first * HD + HD / 2);
  }
  for (int h0 = part * HEADS; h0 < n_heads; h0 += stride) {
    const int head = h0 + lane / LANES;
    const bool here = head < n_heads;
    float lo[8], hi[8];
    ahead[0].numbers(lo);
    ahead[1].numbers(hi);
    if (head + stride < n_heads) {                 // the next round's, while this one is worked on
      ahead[0].load(row + (size_t)(head + stride) * HD);
      ahead[1].load(row + (size_t)(head + stride) * HD + HD / 2);
    }
    if (p.clear && here) {
      clear8(row + (size_t)head * HD);
      clear8(row + (size_t)head * HD + HD / 2);
    }
    if (head < p.Hq + p.Hkv) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x0 = lo[k], x1 = hi[k];
        lo[k] = x0 * c[k] - x1 * s[k];
        hi[k] = x0 * s[k] + x1 * c[k];
      }
    }
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = fmaxf(most, fmaxf(fabsf(lo[k]), fabsf(hi[k])));
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (head < p.Hq) {
      __nv_bfloat16* dst = p.q + ((size_t)t * p.Hq + head) * HD + i;
      __nv_bfloat162 a[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = __floats2bfloat162_rn(lo[2 * k], lo[2 * k + 1]);
        b[k] = __floats2bfloat162_rn(hi[2 * k], hi[2 * k + 1]);
      }
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(a);
      *reinterpret_cast<uint4*>(dst + HD / 2) = *reinterpret_cast<uint4*>(b);
    } else if (here && row0 >= 0) {
      const bool is_k = head < p.Hq + p.Hkv;
      const size_t at = (size_t)row0 + (size_t)(head - p.Hq - (is_k ? 0 : p.Hkv)) * E8_PAGE;
      const int byte = e4m3_scale_byte(most);
      const float f = e4m3_inverse(byte);
      uint8_t* dst = (is_k ? p.kpages : p.vpages) + at * HD + i;
      *reinterpret_cast<uint2*>(dst) = make_uint2(e4m3_quad(lo[0] * f, lo[1] * f, lo[2] * f, lo[3] * f),
                                                  e4m3_quad(lo[4] * f, lo[5] * f, lo[6] * f, lo[7] * f));
      *reinterpret_cast<uint2*>(dst + HD / 2) = make_uint2(e4m3_quad(hi[0] * f, hi[1] * f, hi[2] * f, hi[3] * f),
                                                           e4m3_quad(hi[4] * f, hi[5] * f, hi[6] * f, hi[7] * f));
      if (i == 0) (is_k ? p.kscales : p.vscales)[at] = (uint8_t)byte;
    }
  }
}

// Any rotation: the first `rot` numbers of a head in either pairing, or none.  A warp per (token, head), HD / 32 numbers a
// lane; a number's partner is read beside it.  Layers whose whole heads turn in neighbouring pairs take it for every token.
//
// Few tokens cost what they cost above: 8 of 32 + 2 * 8 heads of 64 1.3 us, 64 of 128 2.0 to 2.5.  From some hundred on it is bound by
// its instructions (79 % of the issue slots, 9 % of the memory's rate): a warp's place, its position's page and the cosines are worked
// out for 64 or 128 numbers alone.  From bfloat16, 32 + 2 * 8 heads of 64 in pairs: 1,300 tokens 17.3 us (split in halves, by the kernel
// above: 4.7), 16,384 tokens 209 us, 13 % of the copy rate (35.5); heads of 128 240 us (63.7), half of each head turned 302.
template <typename T, int HD>
__global__ void __launch_bounds__(WE_WARPS * 32) write_e4m3_any_kernel(WriteE8 p) {
  pdl_launch_dependents();
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  const int n_heads = p.Hq + (p.write_cache || p.clear ? 2 * p.Hkv : 0);
  const long long w = (long long)blockIdx.x * WE_WARPS + (threadIdx.x >> 5);
  const int t = (int)(w / n_heads), head = (int)(w % n_heads);
  if (t >= p.T) return;
  int pos = p.token_pos[t];
  const long long row0 = e8_row(p, t, pos, head == 0 && lane == 0);
  pdl_wait();
  T* src = (T*)p.qkv + (size_t)t * p.ld + (size_t)head * HD;
  float x[N];
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int d = lane * N + k;
    x[k] = to_float(src[d]);
    if (head < p.Hq + p.Hkv && d < p.rot) {
      const int half = p.rot / 2;
      const bool second = p.interleaved ? (d & 1) != 0 : d >= half;
      const int pair = p.interleaved ? d >> 1 : d % half;
      const float other = to_float(src[p.interleaved ? d ^ 1 : (second ? d - half : d + half)]);
      const float c = p.cos_t[(size_t)pos * half + pair], s = p.sin_t[(size_t)pos * half + pair];
      x[k] = second ? other * s + x[k] * c : x[k] * c - other * s;
    }
    most = fmaxf(most, fabsf(x[k]));
  }
  if (p.clear) {
    __syncwarp();                      // every lane has read its numbers' partners
#pragma unroll
    for (int k = 0; k < N; ++k) src[lane * N + k] = from_float<T>(0.f);
  }
  if (head < p.Hq) {
#pragma unroll
    for (int k = 0; k < N; ++k) p.q[((size_t)t * p.Hq + head) * HD + lane * N + k] = __float2bfloat16_rn(x[k]);
    return;
  }
  most = warp_max(most);
  if (row0 < 0) return;
  const bool is_k = head < p.Hq + p.Hkv;
  const size_t at = (size_t)row0 + (size_t)(head - p.Hq - (is_k ? 0 : p.Hkv)) * E8_PAGE;
  const int byte = e4m3_scale_byte(most);
  const float f = e4m3_inverse(byte);
  uint8_t* dst = (is_k ? p.kpages : p.vpages) + at * HD + lane * N;
#pragma unroll
  for (int k = 0; k < N; k += 2) *reinterpret_cast<uint16_t*>(dst + k) = (uint16_t)e4m3_pair(x[k] * f, x[k + 1] * f);
  if (lane == 0) (is_k ? p.kscales : p.vscales)[at] = (uint8_t)byte;
}

// ------------------------------------------------------------------ reading back
struct ReadE8 {
  const uint8_t* kpages;
  const uint8_t* vpages;
  const uint8_t* kscales;
  const uint8_t* vscales;
  const int* page_table;
  const int* pages;          // [n][3]: slot, page of the sequence, rows to read (the rest become zeros)
  __nv_bfloat16* keys;       // [n][Hkv][64][HD]
  __nv_bfloat16* values;
  int n_slots, max_pages, n_pages, Hkv;
};

// Bound by memory: a page of one head is HD * 64 bytes in and twice that out.  A block takes the keys or the values of one
// (page, head); a lane reads 8 bytes and writes 16, so that both sides are whole lines, and requests all it needs at once.
// 8 sequences of 16,384 positions, 8 heads of 128: 80.7 us, 93 % of the copy rate (495 MB).  A page of one head takes 1.2 us.
constexpr int RE_THREADS = 128;

template <int HD>
__global__ void __launch_bounds__(RE_THREADS) read_e4m3_kernel(ReadE8 p) {
  pdl_launch_dependents();
  constexpr int N = E8_PAGE * HD / 8 / RE_THREADS;         // pieces of 8 numbers a thread
  const int entry = blockIdx.x, head = blockIdx.y;
  const int slot = p.pages[3 * entry], idx = p.pages[3 * entry + 1], live = p.pages[3 * entry + 2];
  int page = -1;
  if (slot >= 0 && slot < p.n_slots && idx >= 0 && idx < p.max_pages) page = p.page_table[(size_t)slot * p.max_pages + idx];
  const bool have = page >= 0 && page < p.n_pages;
  pdl_wait();
  const size_t row0 = ((size_t)(have ? page : 0) * p.Hkv + head) * E8_PAGE;
  const uint8_t* src = (blockIdx.z ? p.vpages : p.kpages) + row0 * HD;
  const uint8_t* scales = (blockIdx.z ? p.vscales : p.kscales) + row0;
  __nv_bfloat16* dst = (blockIdx.z ? p.values : p.keys) + ((size_t)entry * p.Hkv + head) * E8_PAGE * HD;
  uint2 u[N];
  int byte[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = (k * RE_THREADS + threadIdx.x) * 8, r = at / HD;
    const bool ok = have && r < live;
    u[k] = ok ? *reinterpret_cast<const uint2*>(src + at) : make_uint2(0u, 0u);
    byte[k] = ok ? scales[r] : 0;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = (k * RE_THREADS + threadIdx.x) * 8;
    const float f = e4m3_scale(byte[k]);
    __nv_bfloat162 o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = j < 2 ? u[k].x : u[k].y;
      const uint32_t h = (j & 1) ? e4m3_high_half2(w) : e4m3_low_half2(w);
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
      o[j] = __floats2bfloat162_rn(v.x * f, v.y * f);
    }
    *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<uint4*>(o);
  }
}

}  // namespace dlgo

using namespace dlgo;

namespace {

int sm_count_here() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <typename T, int HD>
int launch_write(const WriteE8& p, cudaStream_t stream) {
  const int n_heads = p.Hq + (p.write_cache || p.clear ? 2 * p.Hkv : 0);
  if (p.rot == HD && !p.interleaved) {
    constexpr int HEADS = 32 / (HD / 16);
    const int rounds = (n_heads + HEADS - 1) / HEADS;
    // as many warps a token as keep 32 of them on every SM
    const long long want = ((long long)sm_count_here() * 32 + p.T - 1) / p.T;
    const int per_token = (int)(want < rounds ? (want < 1 ? 1 : want) : rounds);
    const long long warps = (long long)p.T * per_token;
    launch_kernel(write_e4m3_kernel<T, HD>, dim3((unsigned)((warps + WE_WARPS - 1) / WE_WARPS)), dim3(WE_WARPS * 32), 0, stream, p,
                  per_token);
  } else {
    const long long warps = (long long)p.T * n_heads;
    launch_kernel(write_e4m3_any_kernel<T, HD>, dim3((unsigned)((warps + WE_WARPS - 1) / WE_WARPS)), dim3(WE_WARPS * 32), 0, stream, p);
  }
  return launch_status();
}

}  // namespace

// qkv[T, ld] (query, key, value heads of hd numbers; dtype 0 fp32, 1 bf16): queries rotated at their tokens' positions into
// q[T, Hq * hd] bf16; keys (rotated) and values into the 8-bit pages of those positions, unless write_cache is 0.  clear
// (fp32 only): zeros are left where qkv was read.
DLGO_EXPORT int dlgo_write_e4m3(void* qkv, int dtype, int T, int ld, const float* cos_t, const float* sin_t, int n_positions,
                                const int* token_pos, const int* token_seq, const int* seq_slot, int n_seqs, const int* page_table,
                                int n_slots, int max_pages, void* kpages, void* vpages, void* kscales, void* vscales, int n_pages, void* q, int Hq, int Hkv, int hd,
                                int rot, int interleaved, int write_cache, int clear, cudaStream_t stream) {
  if (T <= 0) return DLGO_OK;
  if (Hq <= 0 || Hkv <= 0 || (hd != 64 && hd != 128) || rot < 0 || rot > hd || rot % 2 || (rot > 0 && n_positions <= 0) ||
      n_pages <= 0 || n_slots <= 0 || max_pages <= 0)
    return DLGO_ERR_SIZE;
  if (ld < (Hq + 2 * Hkv) * hd || (long long)T * (Hq + 2 * Hkv) > 0x7fffffffLL) return DLGO_ERR_SIZE;
  if (dtype != DLGO_F32 && dtype != DLGO_BF16) return DLGO_ERR_DTYPE;
  if (clear && dtype != DLGO_F32) return DLGO_ERR_DTYPE;
  if (((uintptr_t)qkv & 15) || ((uintptr_t)q & 15) || ld % 8 || ((uintptr_t)cos_t & 15) || ((uintptr_t)sin_t & 15) ||
      ((uintptr_t)kpages & 15) || ((uintptr_t)vpages & 15))
    return DLGO_ERR_ALIGN;
  WriteE8 p;
  p.qkv = qkv; p.ld = ld; p.cos_t = cos_t; p.sin_t = sin_t; p.token_pos = token_pos; p.token_seq = token_seq; p.seq_slot = seq_slot;
  p.n_seqs = n_seqs; p.page_table = page_table; p.n_slots = n_slots; p.max_pages = max_pages; p.n_pages = n_pages;
  p.n_positions = n_positions;
  p.kpages = (uint8_t*)kpages; p.vpages = (uint8_t*)vpages; p.kscales = (uint8_t*)kscales; p.vscales = (uint8_t*)vscales;
  p.q = (__nv_bfloat16*)q; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.rot = rot; p.interleaved = interleaved; p.write_cache = write_cache;
  p.clear = clear;
  if (dtype == DLGO_F32) return hd == 64 ? launch_write<float, 64>(p, stream) : launch_write<float, 128>(p, stream);
  return hd == 64 ? launch_write<__nv_bfloat16, 64>(p, stream) : launch_write<__nv_bfloat16, 128>(p, stream);
}

// pages[n][3] = (slot, page of the sequence, rows): keys and values [n][Hkv][64][hd] bf16 of those pages, rows beyond the
// given number (and pages that the table does not have) as zeros.
DLGO_EXPORT int dlgo_read_e4m3(const void* kpages, const void* vpages, const void* kscales, const void* vscales, int n_pages,
                               const int* page_table, int n_slots, int max_pages, const int* pages, int n, void* keys, void* values,
                               int Hkv, int hd, cudaStream_t stream) {
  if (n <= 0) return DLGO_OK;
  if (Hkv <= 0 || Hkv > 65535 || (hd != 64 && hd != 128) || n_pages <= 0 || n_slots <= 0 || max_pages <= 0) return DLGO_ERR_SIZE;
  if (((uintptr_t)kpages & 15) || ((uintptr_t)vpages & 15) || ((uintptr_t)keys & 15) || ((uintptr_t)values & 15)) return DLGO_ERR_ALIGN;
  ReadE8 p;
  p.kpages = (const uint8_t*)kpages; p.vpages = (const uint8_t*)vpages; p.kscales = (const uint8_t*)kscales;
  p.vscales = (const uint8_t*)vscales; p.page_table = page_table; p.pages = pages; p.keys = (__nv_bfloat16*)keys;
  p.values = (__nv_bfloat16*)values; p.n_slots = n_slots; p.max_pages = max_pages; p.n_pages = n_pages; p.Hkv = Hkv;
  if (hd == 64) launch_kernel(read_e4m3_kernel<64>, dim3(n, Hkv, 2), dim3(RE_THREADS), 0, stream, p);
  else launch_kernel(read_e4m3_kernel<128>, dim3(n, Hkv, 2), dim3(RE_THREADS), 0, stream, p);
  return launch_status();
}

// Both, called with a record (e4m3.cuh).
DLGO_EXPORT int dlgo_write_e4m3_record(const long long* r) { return call_record(dlgo_write_e4m3, r); }
DLGO_EXPORT int dlgo_read_e4m3_record(const long long* r) { return call_record(dlgo_read_e4m3, r); }

// 1 if a write was skipped since the last call because its position had no page (clears the word).
DLGO_EXPORT int dlgo_cache_e4m3_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_e4m3_error, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_cache_e4m3_error, &zero, sizeof(int));
  return v;
}
