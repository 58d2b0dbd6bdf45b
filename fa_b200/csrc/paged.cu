// paged.cu -- attention over a paged cache (b200fa_paged_fwd): argument
// checks, tensor maps, the choice of kernel, and the kernel that joins the
// parts of items cut by a worker's end.
#include <cmath>
#include <cstddef>
#include <cstring>
#include <mutex>

#include "b200fa.h"
#include "host.h"
#include "paged.h"
#include "paged_short.cuh"

namespace b200fa {

template <bool kBf16, int kM>
__global__ void __launch_bounds__(kShortThreads, 1) b200_paged_short_kernel(const __grid_constant__ PagedParams p) {
  paged_short_body<kBf16, kM>(p);
}

// Joins the parts of the item that begins in worker blockIdx.x's stretch and
// goes on behind it, in worker order.  A warp per row, four columns per lane,
// the outputs of eight parts on their way before their weights are known: the
// time is that of a few trips to L2 (520 bytes per row and part).  Launched so
// that it is resident by the time the attention kernel ends.
template <bool kBf16>
__global__ void __launch_bounds__(256) b200_paged_combine_kernel(const __grid_constant__ PagedParams p) {
  grid_wait();
  const int worker = int(blockIdx.x);
  const PagedRecord rec = *paged_record(p, worker);
  const int lane = int(threadIdx.x & 31), rows = rec.parts > 0 ? rec.tokens * p.group : 0;
  auto part = [&](int i) { return paged_partial(p, i == 0 ? 2 * worker + 1 : 2 * (worker + i)); };
  for (int row = int(blockIdx.y) * 8 + int(threadIdx.x >> 5); row < rows; row += int(gridDim.y) * 8) {
    constexpr int kAhead = 8;
    float4 v[kAhead];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < rec.parts) v[i] = __ldcg(reinterpret_cast<const float4*>(part(i0 + i) + row * 128 + lane * 4));
    };
    fetch(0);
    float top = -1e30f;
    for (int i = lane; i < rec.parts; i += 32) top = fmaxf(top, part(i)[p.part_rows * 128 + row]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    float sum = 0.f, f = 0.f, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < rec.parts; i0 += kAhead) {
      if ((i0 & 31) == 0) {  // weights and sums of 32 parts, one per lane
        f = l = 0.f;
        if (i0 + lane < rec.parts) {
          const float* tail = part(i0 + lane) + p.part_rows * 128;
          f = ex2_approx(tail[row] - top);
          l = tail[p.part_rows + row];
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, (i0 + i) & 31);
        sum += fi * __shfl_sync(0xffffffffu, l, (i0 + i) & 31);
        if (i0 + i < rec.parts) acc.x += fi * v[i].x, acc.y += fi * v[i].y, acc.z += fi * v[i].z, acc.w += fi * v[i].w;
      }
      if (i0 + kAhead < rec.parts) fetch(i0 + kAhead);
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const int t = row / p.group, hd = row - t * p.group;
    uint16_t* dst = static_cast<uint16_t*>(p.o) + int64_t(rec.row0 + t) * p.o_tok +
                    int64_t(rec.h * p.group + hd) * p.o_head + lane * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<kBf16>(acc.x * inv, acc.y * inv), pack2<kBf16>(acc.z * inv, acc.w * inv));
  }
}

namespace {

using PagedKernel = void (*)(PagedParams);

PagedKernel short_kernel(bool bf16, int m) {
  if (bf16)
    return m == 1 ? b200_paged_short_kernel<true, 1> : m == 2 ? b200_paged_short_kernel<true, 2> : b200_paged_short_kernel<true, 4>;
  return m == 1 ? b200_paged_short_kernel<false, 1> : m == 2 ? b200_paged_short_kernel<false, 2> : b200_paged_short_kernel<false, 4>;
}

struct PagedDevice {
  std::once_flag once;
  int sms = 0, pairs = 0;
  cudaError_t err = cudaSuccess;
};
PagedDevice g_paged[64];

int paged_device(const PagedDevice** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64) return fail(B200FA_ERR_OPTIONS, "device ordinal %d out of range", dev);
  PagedDevice& d = g_paged[dev];
  std::call_once(d.once, [&d, dev] {
    cudaError_t e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    for (int bf16 = 0; bf16 < 2; ++bf16)
      for (int m : {1, 2, 4})
        if (e == cudaSuccess)
          e = cudaFuncSetAttribute(short_kernel(bf16, m), cudaFuncAttributeMaxDynamicSharedMemorySize, kShortSmemBytes);
    if (e == cudaSuccess) e = cudaError_t(paged_chunk_setup(&d.pairs));
    if (d.sms > kMaxWorkers) d.sms = kMaxWorkers;
    if (d.pairs > kMaxWorkers) d.pairs = kMaxWorkers;
    d.err = e;
  });
  if (d.err != cudaSuccess) return cuda_fail(d.err, "device setup");
  *out = &d;
  return B200FA_OK;
}

uint64_t partial_bytes(int workers, int rows) { return uint64_t(2) * workers * rows * 130u * 4u; }

uint64_t workspace_bytes(const PagedDevice& d) {
  const uint64_t a = partial_bytes(d.sms, 64), b = partial_bytes(d.pairs, 256);
  return kPagedPartials + (a > b ? a : b);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int kDims>
int encode(CUtensorMap* map, const b200fa_paged_args& a, const void* ptr, const cuuint64_t (&dims)[kDims],
           const cuuint64_t (&strides)[kDims - 1], const cuuint32_t (&box)[kDims], const char* what) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (!fn) return fail(B200FA_ERR_NO_DRIVER, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, a.dtype == B200FA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, kDims,
                        const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B200FA_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled failed for %s (%d)", what, int(r));
  return B200FA_OK;
}

// Byte stride of a dimension; one of a single element has no stride of its own.
cuuint64_t stride_of(int64_t count, int64_t stride) { return cuuint64_t(count > 1 ? stride : 128) * 2; }

// Boxes of 64 columns and up to `rows` tokens of a page ...
int encode_pages(CUtensorMap* map, const b200fa_paged_args& a, const void* ptr, const int64_t* s, int rows, const char* what) {
  return encode<4>(map, a, ptr, {128, cuuint64_t(a.page_size), cuuint64_t(a.heads_kv), cuuint64_t(a.num_pages)},
                   {stride_of(a.page_size, s[1]), stride_of(a.heads_kv, s[2]), stride_of(a.num_pages, s[0])},
                   {64, cuuint32_t(a.page_size < rows ? a.page_size : rows), 1, 1}, what);
}

// ... and of both halves of up to 128 tokens.
int encode_halves(CUtensorMap* map, const b200fa_paged_args& a, const void* ptr, const int64_t* s, const char* what) {
  return encode<5>(map, a, ptr, {64, cuuint64_t(a.page_size), 2, cuuint64_t(a.heads_kv), cuuint64_t(a.num_pages)},
                   {stride_of(a.page_size, s[1]), 128, stride_of(a.heads_kv, s[2]), stride_of(a.num_pages, s[0])},
                   {64, cuuint32_t(a.page_size < kPagedBlock ? a.page_size : kPagedBlock), 2, 1, 1}, what);
}

// Boxes of 64 columns of the group's heads of `tokens` tokens.
int encode_q(CUtensorMap* map, const b200fa_paged_args& a, int32_t group, int32_t tokens) {
  return encode<4>(map, a, a.q, {128, cuuint64_t(group), cuuint64_t(a.heads_kv), cuuint64_t(a.tokens)},
                {stride_of(group, a.q_strides[1]), stride_of(a.heads_kv, a.q_strides[1] * group), stride_of(a.tokens, a.q_strides[0])},
                {64, cuuint32_t(group), 1, cuuint32_t(tokens)}, "q");
}

int check_paged(const b200fa_paged_args& a) {
  if (a.dtype != B200FA_DTYPE_FP16 && a.dtype != B200FA_DTYPE_BF16) return fail(B200FA_ERR_DTYPE, "unknown dtype %d", a.dtype);
  if (a.requests < 0 || a.tokens < 0 || a.width < 1 || a.num_pages < 1 || a.heads_q < 1 || a.heads_kv < 1 || a.max_q < 0)
    return fail(B200FA_ERR_SHAPE, "requests %d, tokens %lld, table width %d, pages %lld, heads %d and %d, max_q %d", a.requests,
                (long long)a.tokens, a.width, (long long)a.num_pages, a.heads_q, a.heads_kv, a.max_q);
  if (a.heads_q % a.heads_kv) return fail(B200FA_ERR_GROUPING, "heads_q (%d) must be a multiple of heads_kv (%d)", a.heads_q, a.heads_kv);
  if (a.heads_q / a.heads_kv > 128) return fail(B200FA_ERR_GROUPING, "at most 128 query heads per key/value head, got %d", a.heads_q / a.heads_kv);
  const int64_t most = (int64_t(1) << 31) - 1;
  if (a.page_size < 8 || a.page_size > (1 << 20) || (a.page_size & (a.page_size - 1)))
    return fail(B200FA_ERR_PAGE_SIZE, "page size must be a power of two in [8, 2^20], got %d", a.page_size);
  if (a.tokens > most || a.num_pages >= most || a.requests > B200FA_MAX_REQUESTS || int64_t(a.width) * a.page_size > most - 1023)  // key indices run up to a block past the last key
    return fail(B200FA_ERR_TOO_LARGE, "tokens and pages must be below 2^31, keys of a table row below 2^31 - 1023, requests at most %d",
                B200FA_MAX_REQUESTS);
  if (a.window < 0 || a.sinks < 0 || (a.sinks > 0 && a.window == 0))
    return fail(B200FA_ERR_OPTIONS, "window %d, sinks %d: both at least 0, sinks only with a window", a.window, a.sinks);
  if (a.flags & ~B200FA_PAGED_TEST_WITHHOLD_V) return fail(B200FA_ERR_OPTIONS, "unknown flags 0x%x", a.flags);
  if (!std::isfinite(a.scale) || !(a.scale > 0.f)) return fail(B200FA_ERR_SCALE, "scale must be finite and positive");
  if (a.requests == 0 || a.tokens == 0) return B200FA_OK;
  if (!a.q || !a.o || !a.k_pages || !a.v_pages || !a.block_table || !a.kv_lens || !a.cu_q)
    return fail(B200FA_ERR_NULL, "a required pointer is NULL");
  if (!aligned16(a.q) || !aligned16(a.o) || !aligned16(a.k_pages) || !aligned16(a.v_pages))
    return fail(B200FA_ERR_ALIGNMENT, "tensor pointers must be 16-byte aligned");
  if (a.table_stride < a.width) return fail(B200FA_ERR_STRIDE, "table stride %lld below its width %d", (long long)a.table_stride, a.width);
  auto bad = [](int64_t s, bool used) { return used && (s < 128 || s % 8 || s >= (int64_t(1) << 39)); };
  const bool toks = a.tokens > 1, heads = a.heads_q > 1;
  if (bad(a.q_strides[0], toks) || bad(a.q_strides[1], heads) || bad(a.o_strides[0], toks) || bad(a.o_strides[1], heads))
    return fail(B200FA_ERR_STRIDE, "q and o: token and head strides must be multiples of 8 elements, at least 128");
  for (const int64_t* s : {a.k_strides, a.v_strides})
    if (bad(s[0], a.num_pages > 1) || bad(s[1], true) || bad(s[2], a.heads_kv > 1))
      return fail(B200FA_ERR_STRIDE, "pages: page, token and head strides must be multiples of 8 elements, at least 128");
  return B200FA_OK;
}

}  // namespace
}  // namespace b200fa

using namespace b200fa;

extern "C" {

int64_t b200fa_paged_workspace_size(void) {
  clear_error();
  const PagedDevice* d = nullptr;
  const int rc = paged_device(&d);
  if (rc != B200FA_OK) return rc > 0 ? -int64_t(1000 + rc) : rc;
  return int64_t(workspace_bytes(*d));
}

int b200fa_paged_fwd(const b200fa_paged_args* args, void* stream) {
  clear_error();
  if (!args) return fail(B200FA_ERR_NULL, "args must not be NULL");
  b200fa_paged_args a = {};
  constexpr uint32_t kArgsV1Bytes = offsetof(b200fa_paged_args, status);  // without the status pointer
  if (args->struct_size != sizeof(a) && args->struct_size != kArgsV1Bytes)
    return fail(B200FA_ERR_OPTIONS, "b200fa_paged_args.struct_size mismatch");
  std::memcpy(&a, args, args->struct_size);
  int rc = check_paged(a);
  if (rc != B200FA_OK) return rc;
  if (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 255u))
    return fail(B200FA_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a.status) | reinterpret_cast<uintptr_t>(a.tables_status)) & 3u)
    return fail(B200FA_ERR_ALIGNMENT, "status and tables_status must be 4-byte aligned");
  if (a.requests == 0 || a.tokens == 0) return B200FA_OK;
  const PagedDevice* d = nullptr;
  if ((rc = paged_device(&d)) != B200FA_OK) return rc;
  if (a.ws_bytes < workspace_bytes(*d))
    return fail(B200FA_ERR_WORKSPACE, "workspace must hold %llu bytes", (unsigned long long)workspace_bytes(*d));

  const int32_t group = a.heads_q / a.heads_kv;
  const int64_t rows = int64_t(a.max_q > 0 ? a.max_q : 1) * group;
  // Up to 64 rows of a request the time is that of its keys' bytes, which the
  // short kernel reads faster; beyond, that of the products.
  const bool chunk = rows > 64;

  PagedParams p;
  std::memset(&p, 0, sizeof(p));
  if (chunk) {  // K: each CTA of a pair loads its half of a block's keys; V: its half of the columns
    if ((rc = encode_pages(&p.tm_k, a, a.k_pages, a.k_strides, kPagedBlock / 2, "k_pages")) != B200FA_OK) return rc;
    if ((rc = encode_pages(&p.tm_v, a, a.v_pages, a.v_strides, kPagedBlock, "v_pages")) != B200FA_OK) return rc;
    if ((rc = encode_pages(&p.tm_v8, a, a.v_pages, a.v_strides, 8, "v_pages")) != B200FA_OK) return rc;
    if ((rc = encode_pages(&p.tm_v1, a, a.v_pages, a.v_strides, 1, "v_pages")) != B200FA_OK) return rc;
  } else {
    if ((rc = encode_halves(&p.tm_k, a, a.k_pages, a.k_strides, "k_pages")) != B200FA_OK) return rc;
    if ((rc = encode_halves(&p.tm_v, a, a.v_pages, a.v_strides, "v_pages")) != B200FA_OK) return rc;
  }
  p.q = a.q;
  p.o = a.o;
  p.q_tok = a.q_strides[0];
  p.q_head = a.q_strides[1];
  p.o_tok = a.o_strides[0];
  p.o_head = a.o_strides[1];
  p.table = a.block_table;
  p.table_stride = a.table_stride;
  p.kv_lens = a.kv_lens;
  p.cu_q = a.cu_q;
  p.requests = a.requests;
  p.width = a.width;
  while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
  p.num_pages = int32_t(a.num_pages);
  p.tokens = int32_t(a.tokens);
  p.heads_kv = a.heads_kv;
  p.group = group;
  p.window = a.window;
  p.sinks = a.sinks;
  p.scale_log2 = float(double(a.scale) * 1.4426950408889634074);
  p.timeout_ns = uint64_t(a.timeout_us ? a.timeout_us : 2000000u) * 1000ull;
  p.flags = a.flags;
  p.tables_status = a.tables_status;
  p.ws = static_cast<uint8_t*>(a.workspace);
  p.status = a.status ? a.status : static_cast<uint32_t*>(a.workspace);
  const bool bf16 = a.dtype == B200FA_DTYPE_BF16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (chunk) {
    p.workers = d->pairs;
    p.tokens_per_tile = 2 * (128 / group);  // half of them per CTA of the pair
    p.part_rows = 256;
    if ((rc = encode_q(&p.tm_q, a, group, p.tokens_per_tile / 2)) != B200FA_OK) return rc;
    e = cudaError_t(paged_chunk_launch(p, bf16, st));
  } else {
    const int m = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    p.workers = d->sms;
    p.tokens_per_tile = 16 * m / group;
    p.part_rows = 16 * m;
    e = launch_early(short_kernel(bf16, m), dim3(unsigned(p.workers)), dim3(kShortThreads), kShortSmemBytes, st, p);
  }
  if (e != cudaSuccess) return cuda_fail(e, "paged attention launch");
  e = launch_early(bf16 ? b200_paged_combine_kernel<true> : b200_paged_combine_kernel<false>,
                   dim3(unsigned(p.workers), unsigned(chunk ? 16 : p.part_rows / 8)), dim3(256), 0, st, p);
  return e == cudaSuccess ? B200FA_OK : cuda_fail(e, "combine kernel launch");
}

}  // extern "C"
