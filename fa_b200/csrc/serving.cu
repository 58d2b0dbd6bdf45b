// serving.cu -- the light kernels of a serving step: page tables from request
// lengths, rotary positions, and the cache append (rotary included).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "b200fa.h"
#include "host.h"

namespace b200fa {
namespace {

constexpr int64_t kInt32Max = (int64_t(1) << 31) - 1;
constexpr int kSms = 148;  // of a B200: sizes grids only

// ------------------------------------------------------------ page tables
// Latency-bound: a few KB in, 12 bytes per token out.  Every block scans all
// requests (two prefix sums in shared memory, <= 32 KB) instead of waiting for
// another block's scan, so one launch without any grid-wide step does it; the
// token and page loops are then split over the blocks.  8 requests: 4.3 us; 250
// requests and 175,000 token places: 6.3 us.
constexpr int kTableThreads = 256;

struct TableParams {
  const int32_t* ctx;
  const int32_t* add;
  int32_t* table;
  int64_t table_stride;
  const int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int32_t* positions;
  int32_t* cu_q;
  int32_t* kv_lens;
  int32_t* free_left;
  int32_t* status;
  int64_t num_tokens, free_capacity;
  int32_t requests, width, shift;
};

__device__ __forceinline__ int64_t length(int32_t x) { return x > 0 ? x : 0; }

// Last index r of the non-decreasing prefix sums cum[0..n] with cum[r] <= x;
// x < cum[n].
__device__ __forceinline__ int owner(const int32_t* cum, int n, int32_t x) {
  int lo = 0, hi = n;  // cum[lo] <= x < cum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kTableThreads) b200_build_tables_kernel(const TableParams p) {
  extern __shared__ int32_t sm[];
  const int R = p.requests, tid = int(threadIdx.x);
  int32_t* cum_tok = sm;            // [R + 1]
  int32_t* cum_page = sm + R + 1;   // [R + 1]
  __shared__ int64_t warp_tok[kTableThreads / 32], warp_page[kTableThreads / 32];
  const int64_t mask = (int64_t(1) << p.shift) - 1;
  auto pages = [&](int64_t n) { return (n + mask) >> p.shift; };

  // Each thread sums a run of requests; warp and block scans give its offset.
  const int per = (R + kTableThreads - 1) / kTableThreads;
  const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
  int64_t tok = 0, page = 0;
  int wide = 0;
  for (int r = r0; r < r1; ++r) {
    const int64_t c = length(p.ctx[r]), n = length(p.add[r]);
    tok += n;
    page += pages(c + n) - pages(c);
    wide |= pages(c + n) > p.width || c + n > kInt32Max;  // lengths and positions are 32 bits
  }
  int64_t it = tok, ip = page;
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, it, d), b = __shfl_up_sync(0xffffffffu, ip, d);
    if ((tid & 31) >= d) it += a, ip += b;
  }
  if ((tid & 31) == 31) warp_tok[tid >> 5] = it, warp_page[tid >> 5] = ip;
  wide = __syncthreads_or(wide);
  int64_t total_tok = 0, total_page = 0;
  for (int w = 0; w < kTableThreads / 32; ++w) {
    if (w < (tid >> 5)) it += warp_tok[w], ip += warp_page[w];
    total_tok += warp_tok[w];
    total_page += warp_page[w];
  }
  it -= tok;
  ip -= page;
  for (int r = r0; r < r1; ++r) {
    cum_tok[r] = int32_t(min(it, kInt32Max));
    cum_page[r] = int32_t(min(ip, kInt32Max));
    const int64_t c = length(p.ctx[r]), n = length(p.add[r]);
    it += n;
    ip += pages(c + n) - pages(c);
  }
  if (tid == 0) {
    cum_tok[R] = int32_t(min(total_tok, kInt32Max));
    cum_page[R] = int32_t(min(total_page, kInt32Max));
  }
  const int64_t have = min(length(*p.free_count), p.free_capacity);
  const int status = total_tok > p.num_tokens ? 3 : wide ? 2 : total_page > have ? 1 : 0;
  __syncthreads();

  const int64_t first = int64_t(blockIdx.x) * kTableThreads + tid;
  const int64_t step = int64_t(gridDim.x) * kTableThreads;
  const int64_t known = min(total_tok, p.num_tokens);
  for (int64_t t = first; t < p.num_tokens; t += step) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (t < known) {
      const int r = owner(cum_tok, R, int32_t(t));
      const int64_t c = length(p.ctx[r]), at = c + (t - cum_tok[r]);
      pos = int32_t(at);
      if (status == 0) {
        const int64_t held = pages(c), i = at >> p.shift;
        const int32_t pg = i < held ? p.table[r * p.table_stride + i]
                                    : p.free_pages[have - 1 - (cum_page[r] + (i - held))];
        if (pg >= 0) slot = (int64_t(pg) << p.shift) + (at & mask);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
  if (status == 0) {
    for (int64_t i = first; i < total_page; i += step) {
      const int r = owner(cum_page, R, int32_t(i));
      p.table[r * p.table_stride + pages(length(p.ctx[r])) + (i - cum_page[r])] = p.free_pages[have - 1 - i];
    }
  }
  for (int64_t r = first; r <= R; r += step) {
    p.cu_q[r] = cum_tok[r];
    if (r < R) p.kv_lens[r] = int32_t(length(p.ctx[r]) + (status == 0 ? length(p.add[r]) : 0));
  }
  if (first == 0) {
    *p.free_left = int32_t(status == 0 ? have - total_page : length(*p.free_count));
    *p.status = status;
  }
}

// ------------------------------------------------- rotary and cache append
// Bound by memory: every element is read and written once (streaming hints).  A
// block takes a few tokens with all their heads -- and all sequences that share
// their positions -- computes the sines and cosines of its tokens' pairs, once
// each, into shared memory while its first rows are on their way, and then turns
// (or copies) sixteen elements -- eight pairs -- of a row per thread and step,
// the next row's loads ahead of this one's stores.  16000 tokens of 48 heads,
// half of them turned: 69 us, 5.7 TB/s; 2 x 12 x 32768 rows: 79 us, 5.1 TB/s.
// (Angles in the threads' registers, anew for every eight heads: 100 and 102 us;
// more heads at once per thread: slower still, occupancy fell.)
//
// The angle: position times frequency in turns as a 64-bit binary fraction,
// reduced mod 1 by the integer product's wrap-around.  The product is exact, so
// the angle is off by position * 2^-65 turns, the frequency's rounding, where a
// 32-bit product is off by position * 2^-24 radians (0.008 at 131072).
struct Segment {  // a run of heads: rows [batch][n][heads][dim] -> the same, or the cache
  const uint4* src;
  uint4* dst;
  // In units of 16 bytes: 32 bits reach 32 GB, and index times stride is one
  // instruction (the kernel is close to its issue rate).
  int32_t src_b, src_n, src_h;
  int32_t dst_b, dst_n, dst_h;  // scattered: page, token, head
  int32_t heads;
  int32_t rotate, scatter;
};

struct RotaryParams {
  Segment seg[3];
  int32_t segments, heads;   // heads of all segments
  int64_t n, tokens;         // tokens = batch * n
  const void* positions;
  int32_t pos_bits;
  int64_t pos_stride;
  const uint64_t* freq;
  int32_t lanes;             // threads per row: dim / 16
  int32_t rot;
  float magnitude, sign;
  const int64_t* slots;
  int64_t num_slots;
  int32_t shift;
  int32_t tokens_per_block, tokens_first;
  int32_t batched;           // tokens = n, heads = batch * heads: the sequences share their positions
};

constexpr int kMaxTokens = 16;  // of a block

template <typename T>
struct Sixteen {  // 16 elements as 16-byte pieces
  static constexpr int kPer = 16 / int(sizeof(T));   // elements of a piece
  static constexpr int kPieces = 16 / kPer;
  uint4 v[kPieces];
};

template <typename T>
struct Two;
template <>
struct Two<float> { using type = float2; };
template <>
struct Two<__half> { using type = __half2; };
template <>
struct Two<__nv_bfloat16> { using type = __nv_bfloat162; };

__device__ __forceinline__ float2 to_float2(float2 x) { return x; }
__device__ __forceinline__ float2 to_float2(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ float2 to_float2(__nv_bfloat162 x) { return __bfloat1622float2(x); }
__device__ __forceinline__ void from_float2(float2 x, float2& o) { o = x; }
__device__ __forceinline__ void from_float2(float2 x, __half2& o) { o = __float22half2_rn(x); }
__device__ __forceinline__ void from_float2(float2 x, __nv_bfloat162& o) { o = __float22bfloat162_rn(x); }

// kLayout 0: a thread's pairs are elements (8 c + i, rot/2 + 8 c + i); 1:
// (16 c + 2 i, 16 c + 2 i + 1).  Lanes at or behind rot copy elements 16 c ...
template <typename T, int kLayout>
__global__ void __launch_bounds__(256) b200_rotary_kernel(const RotaryParams p) {
  constexpr int kPer = Sixteen<T>::kPer, kPieces = Sixteen<T>::kPieces;
  extern __shared__ __align__(16) float2 angles[];  // [token of the block][pair]: cos, sin; read two pairs at a time
  __shared__ int32_t tok_b[kMaxTokens], tok_n[kMaxTokens];
  __shared__ int64_t tok_slot[kMaxTokens];
  const int32_t token0 = int32_t(blockIdx.x) * p.tokens_per_block;
  const int tokens = min(p.tokens_per_block, int32_t(p.tokens) - token0), pairs = p.rot / 2;
  if (int(threadIdx.x) < tokens) {
    const int32_t token = token0 + int(threadIdx.x), b = token / int32_t(p.n);
    tok_b[threadIdx.x] = b;
    tok_n[threadIdx.x] = token - b * int32_t(p.n);
    tok_slot[threadIdx.x] = p.slots ? p.slots[token] : 0;
  }
  __syncthreads();

  // A thread keeps its place c in the rows and steps over rows, which run over
  // the tokens first where those are closer in memory than the heads.
  const int c = int(threadIdx.x) % p.lanes, step = 256 / p.lanes;
  const bool turn = 16 * c < p.rot, active = int(threadIdx.x) / p.lanes < step;
  // Where the thread's first and second eight elements are, in 16 bytes.
  const int lo = ((turn && kLayout == 0) ? 8 * c : 16 * c) / kPer;
  const int hi = ((turn && kLayout == 0) ? pairs + 8 * c : 16 * c + 8) / kPer;
  const int inners = p.tokens_first ? tokens : p.heads, outers = p.tokens_first ? p.heads : tokens;
  struct Row {
    uint4* dst;  // NULL: none, or skipped
    int t;
    bool turned;
    Sixteen<T> x;
  };
  int inner = int(threadIdx.x) / p.lanes, outer = 0;
  // The row at (inner, outer), loaded; false when there is none.
  auto load = [&](Row& row) -> bool {
    while (inner >= inners && outer < outers) inner -= inners, ++outer;
    if (!active || outer >= outers) return false;
    row.t = p.tokens_first ? inner : outer;
    int hh = p.tokens_first ? outer : inner, k = 0;
    inner += step;
    while (k + 1 < p.segments && hh >= p.seg[k].heads) hh -= p.seg[k++].heads;
    const Segment& s = p.seg[k];
    int b = tok_b[row.t];
    const int n = tok_n[row.t];
    if (p.batched) {  // a token of all sequences: heads run over (sequence, head)
      b = hh / s.heads;
      hh -= b * s.heads;
    }
    row.dst = nullptr;
    uint4* dst = s.dst;
    if (s.scatter) {
      const int64_t slot = tok_slot[row.t];
      if (slot < 0 || slot >= p.num_slots) return true;
      dst += int64_t(int32_t(slot >> p.shift)) * s.dst_b + int64_t(int32_t(slot) & ((1 << p.shift) - 1)) * s.dst_n + int64_t(hh) * s.dst_h;
    } else {
      dst += int64_t(b) * s.dst_b + int64_t(n) * s.dst_n + int64_t(hh) * s.dst_h;
    }
    row.dst = dst;
    row.turned = s.rotate && turn;
    const uint4* src = s.src + int64_t(b) * s.src_b + int64_t(n) * s.src_n + int64_t(hh) * s.src_h;
#pragma unroll
    for (int u = 0; u < kPieces; ++u) row.x.v[u] = __ldcs(src + (u < kPieces / 2 ? lo + u : hi + (u - kPieces / 2)));
    return true;
  };
  Row row;
  bool have = load(row);  // on its way while the angles are computed

  for (int i = int(threadIdx.x); i < tokens * pairs; i += 256) {
    const int t = i / pairs, pair = i - t * pairs;
    int64_t pos = tok_n[t];
    if (p.positions) {
      const int64_t at = tok_b[t] * p.pos_stride + tok_n[t];
      pos = p.pos_bits == 64 ? static_cast<const int64_t*>(p.positions)[at]
                             : int64_t(static_cast<const int32_t*>(p.positions)[at]);
    }
    const uint64_t phase = uint64_t(pos) * p.freq[pair];
    float sn, cs;
    sincospif(2.f * (float(int32_t(phase >> 32)) * 0x1p-32f), &sn, &cs);  // turns in [-1/2, 1/2)
    angles[i] = make_float2(cs * p.magnitude, sn * p.sign * p.magnitude);
  }
  __syncthreads();

  while (have) {
    Row cur = row;
    have = load(row);  // the next row's loads before this one's stores
    if (cur.dst == nullptr) continue;
    if (cur.turned) {
      using T2 = typename Two<T>::type;
      T2* e = reinterpret_cast<T2*>(cur.x.v);
      const float4* a4 = reinterpret_cast<const float4*>(angles + cur.t * pairs + 8 * c);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float4 a = a4[u];  // cos, sin of two pairs
        if constexpr (kLayout == 0) {
          const float2 f = to_float2(e[u]), g = to_float2(e[4 + u]);
          from_float2(make_float2(f.x * a.x - g.x * a.y, f.y * a.z - g.y * a.w), e[u]);
          from_float2(make_float2(g.x * a.x + f.x * a.y, g.y * a.z + f.y * a.w), e[4 + u]);
        } else {
          const float2 f = to_float2(e[2 * u]), g = to_float2(e[2 * u + 1]);
          from_float2(make_float2(f.x * a.x - f.y * a.y, f.y * a.x + f.x * a.y), e[2 * u]);
          from_float2(make_float2(g.x * a.z - g.y * a.w, g.y * a.z + g.x * a.w), e[2 * u + 1]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
      __stcs(cur.dst + (u < kPieces / 2 ? lo + u : hi + (u - kPieces / 2)), cur.x.v[u]);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int element_size(int32_t dtype) { return dtype == B200FA_DTYPE_FP32 ? 4 : 2; }

int check_rotary(const b200fa_rotary_desc* r, int32_t dim) {
  if (dim < 16 || dim > 1024 || dim % 16)
    return fail(B200FA_ERR_HEAD_DIM, "head dim must be a multiple of 16 in [16, 1024], got %d", dim);
  if (!r) return B200FA_OK;
  if (r->struct_size != sizeof(b200fa_rotary_desc)) return fail(B200FA_ERR_ROTARY, "b200fa_rotary_desc.struct_size mismatch");
  if (r->dim != dim || r->rot < 16 || r->rot > dim || r->rot % 16 || r->layout < 0 || r->layout > 1 || !r->freq)
    return fail(B200FA_ERR_ROTARY, "rotary dim %d, rot %d, layout %d: rot is a multiple of 16 up to the head dim %d", r->dim,
                r->rot, r->layout, dim);
  return B200FA_OK;
}

int check_strides(const int64_t* s, int count, int64_t unit, const char* what) {
  for (int i = 0; i < count; ++i)
    if (s[i] < 0 || s[i] % unit || s[i] / unit > kInt32Max)
      return fail(B200FA_ERR_STRIDE, "%s: stride %lld is not a multiple of 16 bytes from 0 to 32 GB", what, (long long)s[i]);
  return B200FA_OK;
}

// Strides (batch, n, heads) or (page, token, head) in elements of 16 / unit bytes.
Segment segment(const void* src, void* dst, const int64_t (&s)[3], const int64_t (&d)[3], int64_t unit, int64_t heads, bool rotate,
                bool scatter) {
  return Segment{static_cast<const uint4*>(src), static_cast<uint4*>(dst), int32_t(s[0] / unit), int32_t(s[1] / unit),
                 int32_t(s[2] / unit), int32_t(d[0] / unit), int32_t(d[1] / unit), int32_t(d[2] / unit), int32_t(heads),
                 int32_t(rotate), int32_t(scatter)};
}

// A written tensor's rows must not share memory.
int check_distinct(const int64_t* s, const int64_t* sizes, int count, const char* what) {
  for (int i = 0; i < count; ++i)
    if (s[i] == 0 && sizes[i] > 1) return fail(B200FA_ERR_STRIDE, "%s is written and must not be expanded", what);
  return B200FA_OK;
}

// Tokens of a block: one where there are few (the shortest chain), else enough
// for about 288 rows, within 16 KiB of angles.
int launch_rotary(RotaryParams& p, const b200fa_rotary_desc* r, int32_t dim, int32_t dtype, void* stream) {
  p.lanes = dim / 16;
  p.rot = r ? r->rot : 0;
  p.freq = r ? r->freq : nullptr;
  p.magnitude = r ? r->magnitude : 1.f;
  p.sign = r && r->inverse ? -1.f : 1.f;
  int64_t per = 1;
  if (p.tokens > 4 * kSms) {
    per = 288 / p.heads;
    const int64_t most = p.rot ? (16 << 10) / (p.rot * 4) : kMaxTokens;
    per = per < 1 ? 1 : per > kMaxTokens ? kMaxTokens : per;
    if (per > most) per = most;
  }
  p.tokens_per_block = int32_t(per);
  const int64_t blocks = (p.tokens + per - 1) / per;
  p.tokens_first = p.seg[0].src_n < p.seg[0].src_h;
  if (p.tokens > kInt32Max - kMaxTokens || p.heads > kInt32Max / 2) return fail(B200FA_ERR_TOO_LARGE, "too many rows for one launch");
  const size_t smem = size_t(per) * size_t(p.rot / 2) * sizeof(float2);
  const int layout = r ? r->layout : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define B200FA_ROTARY(T)                                                          \
  if (layout == 0) b200_rotary_kernel<T, 0><<<unsigned(blocks), 256, smem, st>>>(p); \
  else b200_rotary_kernel<T, 1><<<unsigned(blocks), 256, smem, st>>>(p)
  if (dtype == B200FA_DTYPE_FP16) { B200FA_ROTARY(__half); }
  else if (dtype == B200FA_DTYPE_BF16) { B200FA_ROTARY(__nv_bfloat16); }
  else { B200FA_ROTARY(float); }
#undef B200FA_ROTARY
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200FA_OK : cuda_fail(e, "rotary kernel launch");
}

// Powers of two: a slot's page and offset are a shift and a mask, and a page is
// whole parts of a 128-key block, or whole blocks.
int page_shift(int32_t page_size) {
  if (page_size < 8 || page_size > (1 << 20) || (page_size & (page_size - 1))) return -1;
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace
}  // namespace b200fa

using namespace b200fa;

extern "C" {

int b200fa_build_tables(const int32_t* ctx_lens, const int32_t* new_lens, int32_t requests, int32_t* block_table,
                        int64_t table_stride, int32_t width, const int32_t* free_pages, int64_t free_capacity,
                        const int32_t* free_count, int32_t page_size, int64_t* slots, int32_t* positions,
                        int64_t num_tokens, int32_t* cu_q, int32_t* kv_lens, int32_t* free_left, int32_t* status,
                        void* stream) {
  clear_error();
  if (!ctx_lens || !new_lens || !block_table || !free_count || !cu_q || !kv_lens || !free_left || !status ||
      (free_capacity > 0 && !free_pages) || (num_tokens > 0 && (!slots || !positions)))
    return fail(B200FA_ERR_NULL, "a required pointer is NULL");
  if (requests < 1 || width < 1 || table_stride < width || num_tokens < 0 || free_capacity < 0)
    return fail(B200FA_ERR_SHAPE, "requests %d, width %d, stride %lld, tokens %lld", requests, width,
                (long long)table_stride, (long long)num_tokens);
  if (requests > B200FA_MAX_REQUESTS || num_tokens > kInt32Max)
    return fail(B200FA_ERR_TOO_LARGE, "at most %d requests and 2^31-1 tokens", B200FA_MAX_REQUESTS);
  const int shift = page_shift(page_size);
  if (shift < 0) return fail(B200FA_ERR_PAGE_SIZE, "page size must be a power of two in [8, 2^20], got %d", page_size);
  TableParams p{ctx_lens, new_lens, block_table, table_stride, free_pages, free_count, slots, positions, cu_q, kv_lens,
                free_left, status, num_tokens, free_capacity, requests, width, shift};
  int64_t blocks = (num_tokens + 4 * kTableThreads - 1) / (4 * kTableThreads);
  blocks = blocks < 1 ? 1 : blocks > 2 * kSms ? 2 * kSms : blocks;
  b200_build_tables_kernel<<<unsigned(blocks), kTableThreads, size_t(2 * (requests + 1)) * 4,
                             static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200FA_OK : cuda_fail(e, "page table kernel launch");
}

int b200fa_rotary(const void* x, void* out, int64_t batch, int64_t n, int64_t heads, const int64_t* x_strides,
                  const int64_t* out_strides, const void* positions, int32_t pos_bits, int64_t pos_stride,
                  const b200fa_rotary_desc* rotary, int32_t dtype, void* stream) {
  clear_error();
  if (!x_strides || !out_strides || !rotary) return fail(B200FA_ERR_NULL, "strides and rotary must not be NULL");
  if (dtype < B200FA_DTYPE_FP16 || dtype > B200FA_DTYPE_FP32) return fail(B200FA_ERR_DTYPE, "unknown dtype %d", dtype);
  int rc = check_rotary(rotary, rotary->dim);
  if (rc != B200FA_OK) return rc;
  if (batch < 0 || n < 0 || heads < 0 || batch > kInt32Max || n > kInt32Max || heads > kInt32Max ||
      (positions && pos_bits != 32 && pos_bits != 64) || pos_stride < 0)
    return fail(B200FA_ERR_SHAPE, "invalid rotary geometry");
  if (batch == 0 || n == 0 || heads == 0) return B200FA_OK;
  if (!x || !out) return fail(B200FA_ERR_NULL, "x and out must be device pointers");
  if (!aligned16(x) || !aligned16(out)) return fail(B200FA_ERR_ALIGNMENT, "tensor pointers must be 16-byte aligned");
  const int64_t unit = 16 / element_size(dtype);
  if ((rc = check_strides(x_strides, 3, unit, "x")) != B200FA_OK) return rc;
  if ((rc = check_strides(out_strides, 3, unit, "out")) != B200FA_OK) return rc;
  const int64_t sizes[3] = {batch, n, heads};
  if ((rc = check_distinct(out_strides, sizes, 3, "out")) != B200FA_OK) return rc;
  RotaryParams p{};
  p.seg[0] = segment(x, out, {x_strides[0], x_strides[1], x_strides[2]}, {out_strides[0], out_strides[1], out_strides[2]}, unit,
                     heads, true, false);
  p.segments = 1;
  // Sequences with the same positions share the angles.
  p.batched = (!positions || pos_stride == 0) && batch > 1 && batch * heads <= kInt32Max;
  p.heads = int32_t(p.batched ? batch * heads : heads);
  p.n = n;
  p.tokens = p.batched ? n : batch * n;
  p.positions = positions;
  p.pos_bits = pos_bits;
  p.pos_stride = pos_stride;
  return launch_rotary(p, rotary, rotary->dim, dtype, stream);
}

int b200fa_append(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, const void* k,
                  const int64_t* k_strides, const void* v, const int64_t* v_strides, void* k_pages,
                  const int64_t* k_page_strides, void* v_pages, const int64_t* v_page_strides, int64_t tokens,
                  int32_t heads_q, int32_t heads_kv, int32_t dim, int64_t num_pages, int32_t page_size,
                  const int64_t* slots, const void* positions, int32_t pos_bits, const b200fa_rotary_desc* rotary,
                  int32_t dtype, void* stream) {
  clear_error();
  if (dtype != B200FA_DTYPE_FP16 && dtype != B200FA_DTYPE_BF16) return fail(B200FA_ERR_DTYPE, "unknown dtype %d", dtype);
  int rc = check_rotary(rotary, dim);
  if (rc != B200FA_OK) return rc;
  if (tokens < 0 || tokens > kInt32Max || heads_kv < 1 || (q && heads_q < 1) || num_pages < 1 || num_pages > kInt32Max)
    return fail(B200FA_ERR_SHAPE, "tokens %lld, heads %d and %d, pages %lld", (long long)tokens, heads_q, heads_kv,
                (long long)num_pages);
  const int shift = page_shift(page_size);
  if (shift < 0) return fail(B200FA_ERR_PAGE_SIZE, "page size must be a power of two in [8, 2^20], got %d", page_size);
  if (!k_strides || !v_strides || !k_page_strides || !v_page_strides || (q && (!q_strides || !q_out_strides || !q_out)))
    return fail(B200FA_ERR_NULL, "a required pointer is NULL");
  if (rotary && positions && pos_bits != 32 && pos_bits != 64) return fail(B200FA_ERR_SHAPE, "positions are int32 or int64");
  if (tokens == 0) return B200FA_OK;
  if (!k || !v || !k_pages || !v_pages || !slots || (rotary && !positions))
    return fail(B200FA_ERR_NULL, "k, v, pages, slots and (with rotary) positions must be device pointers");
  if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages))
    return fail(B200FA_ERR_ALIGNMENT, "tensor pointers must be 16-byte aligned");
  if ((q && ((rc = check_strides(q_strides, 2, 8, "q")) || (rc = check_strides(q_out_strides, 2, 8, "q_out")))) ||
      (rc = check_strides(k_strides, 2, 8, "k")) || (rc = check_strides(v_strides, 2, 8, "v")) ||
      (rc = check_strides(k_page_strides, 3, 8, "k_pages")) || (rc = check_strides(v_page_strides, 3, 8, "v_pages")))
    return rc;
  const int64_t rows[2] = {tokens, heads_q}, pages[3] = {num_pages, page_size, heads_kv};
  if ((q && (rc = check_distinct(q_out_strides, rows, 2, "q_out"))) || (rc = check_distinct(k_page_strides, pages, 3, "k_pages")) ||
      (rc = check_distinct(v_page_strides, pages, 3, "v_pages")))
    return rc;
  RotaryParams p{};
  int n = 0;
  const int64_t unit = 8;  // elements of 16 bytes
  p.seg[n++] = segment(k, k_pages, {0, k_strides[0], k_strides[1]}, {k_page_strides[0], k_page_strides[1], k_page_strides[2]}, unit,
                       heads_kv, rotary != nullptr, true);
  p.seg[n++] = segment(v, v_pages, {0, v_strides[0], v_strides[1]}, {v_page_strides[0], v_page_strides[1], v_page_strides[2]}, unit,
                       heads_kv, false, true);
  if (q) p.seg[n++] = segment(q, q_out, {0, q_strides[0], q_strides[1]}, {0, q_out_strides[0], q_out_strides[1]}, unit, heads_q,
                              rotary != nullptr, false);
  p.segments = n;
  p.heads = 2 * heads_kv + (q ? heads_q : 0);
  p.n = tokens;
  p.tokens = tokens;
  p.positions = positions;
  p.pos_bits = pos_bits;
  p.slots = slots;
  p.num_slots = num_pages << shift;
  p.shift = shift;
  return launch_rotary(p, rotary, dim, dtype, stream);
}

}  // extern "C"
