// paged.h -- attention over a paged cache: what its kernels share.  The
// parameters, how the work is cut, and how partial results are joined.
//
// Rows.  The `group` query heads of one key/value head read the same keys, so
// a work item takes them together: `tokens_per_tile` consecutive new tokens
// of a request times the group, row = token * group + head in the tile.
//
// Work.  The key blocks (128 keys) of every item -- request, key/value head,
// tile, in that order -- form one line, and worker w of n takes the stretch
// [total w / n, total (w + 1) / n) of it: every worker has the same number of
// blocks whatever the lengths, a long context is split over many workers when
// there are few rows, and nothing but cu_q and kv_lens (on the device) is
// needed to find one's place.  An item that a worker's end cuts leaves
// partial results, per row the unnormalised output relative to its maximum,
// the maximum (log2 domain) and the sum; worker w keeps at most two: slot 2w
// for an item begun before its stretch, slot 2w + 1 for one that begins in it
// and goes on after it.  The worker an item begins in leaves a record of it,
// from which combine_partials joins the parts in worker order, so the same
// lengths always give the same bits.
//
// Keys.  The row at position p sees keys j <= p, with a window only
// j > p - window or j < sinks; an item visits the blocks that hold a visible
// sink, then those from its first row's window to its last row's position.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace b200fa {

constexpr int kPagedBlock = 128;  // keys per block
constexpr uint32_t kDevPage = 4u;
constexpr uint32_t kPagedHeader = 256;  // status words
constexpr int kMaxWorkers = 512;
constexpr uint32_t kPagedRecord = 32;   // bytes of a worker's record
constexpr uint32_t kPagedPartials = kPagedHeader + kMaxWorkers * kPagedRecord;  // offset of the partial results

struct PagedParams {
  CUtensorMap tm_k, tm_v;   // (128, page_size, heads_kv, num_pages), boxes of 64 columns; short kernel:
                            // (64, page_size, 2, heads_kv, num_pages), boxes of both halves of the head dim
  CUtensorMap tm_v8, tm_v1; // chunk kernel: V in boxes of 64 columns by 8 tokens and by one
  CUtensorMap tm_q;         // chunk kernel: (128, group, heads_kv, tokens), box (64, group, 1, tokens_per_tile / 2)
  const void* q;
  void* o;
  int64_t q_tok, q_head, o_tok, o_head;  // elements
  const int32_t* table;
  int64_t table_stride;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  int32_t requests, width, page_shift, num_pages;
  int32_t tokens, heads_kv, group;
  int32_t tokens_per_tile;
  int32_t window, sinks;
  float scale_log2;
  int32_t workers;
  int32_t part_rows;        // rows of a partial result
  uint64_t timeout_ns;
  uint32_t flags;           // B200FA_PAGED_TEST_WITHHOLD_V
  const int32_t* tables_status;  // other than 0: no row sees a key; may be NULL
  uint8_t* ws;
  uint32_t* status;
};

struct PagedRequest {
  int q0, len;     // its rows of q
  int kv;          // its keys
  __device__ __forceinline__ int tiles(const PagedParams& p) const {
    return (len + p.tokens_per_tile - 1) / p.tokens_per_tile;
  }
};

// Lengths as the kernels use them: rows inside q, keys inside the table, so
// that a malformed length cannot lead outside a tensor.
__device__ __forceinline__ PagedRequest paged_request(const PagedParams& p, int r) {
  int a = p.cu_q[r], b = p.cu_q[r + 1];
  a = a < 0 ? 0 : a > p.tokens ? p.tokens : a;
  b = b < a ? a : b > p.tokens ? p.tokens : b;
  const int64_t most = int64_t(p.width) << p.page_shift;
  int kv = p.kv_lens[r];
  if (p.tables_status != nullptr && *p.tables_status != 0) kv = 0;
  kv = kv < 0 ? 0 : kv > most ? int(most) : kv;
  return PagedRequest{a, b - a, kv};
}

// The key blocks of a tile: block j is key block j for j < sink, else
// j + skip.  At least one, so that a tile whose rows see nothing still
// writes its zeros.  Pages are loaded that hold a key of [first_key, end_key)
// or, below end_key, a sink.
struct PagedBlocks {
  int n, sink, skip;
  int pos0;        // position of the tile's first row (may be negative)
  int first_key;   // first key of the first row's window
  int end_key;     // past the position of the last row
  __device__ __forceinline__ int key_block(int j) const { return j < sink ? j : j + skip; }
  // Whether the key block at `key0` holds keys that no row of the tile sees and
  // that come with its others: between the sinks and the first row's window, or
  // behind the last row.  Of a tile's blocks only the last of the sinks', the
  // first of the window's (block `sink`) and the last can.
  __device__ __forceinline__ bool unseen(const PagedParams& p, int key0) const {
    const int last = key0 + kPagedBlock;
    return last > end_key || (last > p.sinks && key0 < first_key && p.sinks < first_key);
  }
  // Part 0 and 1 of them, [x, y) relative to the block; may be empty.
  __device__ __forceinline__ int2 unseen_keys(const PagedParams& p, int key0, int part) const {
    return part ? make_int2(max(end_key - key0, 0), kPagedBlock)
                : make_int2(max(p.sinks - key0, 0), min(first_key - key0, kPagedBlock));
  }
};

__device__ __forceinline__ PagedBlocks paged_blocks(const PagedParams& p, const PagedRequest& q, int tile) {
  const int t0 = tile * p.tokens_per_tile;
  const int left = q.len - t0;
  const int pos0 = q.kv - q.len + t0;
  const int pos1 = pos0 + (left < p.tokens_per_tile ? left : p.tokens_per_tile) - 1;
  const int end = pos1 >= 0 ? pos1 / kPagedBlock + 1 : 0;
  PagedBlocks b;
  b.pos0 = pos0;
  b.end_key = pos1 >= 0 ? pos1 + 1 : 0;
  b.first_key = 0;
  b.sink = 0;
  int first = 0;
  if (p.window > 0) {
    b.first_key = pos0 > p.window - 1 ? pos0 - (p.window - 1) : 0;
    first = b.first_key / kPagedBlock;
    int s = p.sinks / kPagedBlock + (p.sinks % kPagedBlock != 0);
    if (s > end) s = end;
    b.sink = s < first ? s : first;
  }
  b.n = b.sink + (end > first ? end - first : 0);
  b.skip = first - b.sink;
  if (b.n == 0) b.n = 1, b.sink = 1, b.skip = 0;
  return b;
}

// Sum over i < n of floor((k i + b) / 128), k > 0, b >= 0: the numerators' sum less
// that of their residues mod 128.  With g the largest power of two (up to 128) in
// k, the residues repeat after 128 / g terms, which take every value that is b mod
// g once; what is left of a period is added up term by term (a few, mostly: a
// request's tiles).
__device__ __forceinline__ int64_t block_sum(int64_t n, int k, int64_t b) {
  static_assert(kPagedBlock == 128, "residues mod 128");
  const int log_g = __ffs(k) - 1 < 7 ? __ffs(k) - 1 : 7, g = 1 << log_g, period = 128 >> log_g;
  int64_t residues = (n >> (7 - log_g)) * (int64_t(period) * (int(b) & (g - 1)) + 64 * (period - 1));
  int r = int(b) & 127;
  for (int i = int(n) & (period - 1); i > 0; --i) {
    residues += r;
    r = (r + k) & 127;
  }
  return (k * (n * (n - 1) / 2) + b * n - residues) >> 7;
}

// Key blocks of the request's first `tiles` tiles, for one key/value head: the
// sum of paged_blocks(...).n in closed form, so that a prompt of thousands of
// tiles takes no longer to place than a token.  With c the position of the
// request's first row and k the tokens of a tile, tile t ends in block
// (c + k t + k - 1) / 128 (the last tile of the request: (kv - 1) / 128), and
// skips the blocks between the sinks' and that of c + k t - window + 1.
__device__ __forceinline__ int64_t blocks_before(const PagedParams& p, const PagedRequest& q, int tiles) {
  const int64_t k = p.tokens_per_tile, c = int64_t(q.kv) - q.len;
  if (tiles <= 0) return 0;
  const int64_t last = q.tiles(p) - 1;
  int64_t n = 0, t1 = 0;  // tiles before t1 end before position 0: one masked block each
  if (c + k - 1 < 0) t1 = (-(c + k - 1) + k - 1) / k;
  const int64_t full = tiles < last ? tiles : last;  // tiles that are not the request's last
  if (t1 > full) t1 = full;
  n += t1;
  n += block_sum(full - t1, int(k), c + k * t1 + k - 1) + (full - t1);
  if (tiles > last) n += q.kv > 0 ? (q.kv - 1) / kPagedBlock + 1 : 1;
  if (p.window > 0) {
    const int64_t s = p.sinks / kPagedBlock + (p.sinks % kPagedBlock != 0);
    const int64_t b = c - (p.window - 1) - s * kPagedBlock;  // keys of tile 0 between its window and the sinks' blocks
    int64_t t2 = b < 0 ? (-b + k - 1) / k : 0;
    if (t2 < tiles) n -= block_sum(tiles - t2, int(k), b + k * t2);
  }
  return n;
}

// Key blocks of a request for one key/value head.
__device__ __forceinline__ int64_t head_blocks(const PagedParams& p, const PagedRequest& q) {
  const int tiles = q.tiles(p);
  return tiles == 1 ? paged_blocks(p, q, 0).n : blocks_before(p, q, tiles);
}

// a / b for a >= 0, b > 0: in 32 bits where it fits (a 64-bit division takes
// some hundred cycles, and a worker's start is on every call's path).
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// A worker's place in the line of blocks.
struct PagedStart {
  int r, h, tile, off;   // first item and the block of it to begin with
  int64_t count;         // blocks of the stretch
  int64_t total;         // blocks of all
  int64_t per;           // total / workers
  int workers, rest;     // stretches they are cut into, no more than blocks; total % workers

  // First block of stretch w: floor(total w / workers).
  __device__ __forceinline__ int64_t begin(int w) const { return per * w + int64_t(uint32_t(rest) * uint32_t(w) / uint32_t(workers)); }
  // The stretch that holds block x: the last w with begin(w) <= x.
  __device__ __forceinline__ int owner(int64_t x) const { return int(((x + 1) * workers - 1) / total); }
};
static_assert(kMaxWorkers <= 512, "rest * w stays below 2^32");

// The start of worker `worker`; all threads of the block call it.  `scratch`:
// blockDim.x / 32 shared int64; `start`: shared.
__device__ __forceinline__ void find_start(const PagedParams& p, int worker, int64_t* scratch, PagedStart* start) {
  const int tid = int(threadIdx.x), nt = int(blockDim.x), warps = nt / 32;
  const int per = (p.requests + nt - 1) / nt;
  const int r0 = min(p.requests, tid * per), r1 = min(p.requests, r0 + per);
  int64_t sum = 0;
  for (int r = r0; r < r1; ++r) sum += head_blocks(p, paged_request(p, r)) * p.heads_kv;
  int64_t inc = sum;
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, inc, d);
    if ((tid & 31) >= d) inc += a;
  }
  if ((tid & 31) == 31) scratch[tid >> 5] = inc;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < (tid >> 5)) inc += scratch[w];
    total += scratch[w];
  }
  PagedStart s{0, 0, 0, 0, 0, total, 0, total < p.workers ? int(total) : p.workers, 0};
  int64_t begin = 0;
  if (worker < s.workers) {
    s.per = divide(total, s.workers);
    s.rest = int(total - s.per * s.workers);
    begin = s.begin(worker);
    s.count = s.begin(worker + 1) - begin;
  }
  __syncthreads();  // scratch has been read
  if (s.count == 0) {
    if (tid == 0) *start = s;
    __syncthreads();
    return;
  }
  int64_t at = inc - sum;
  if (at <= begin && begin < inc) {  // one thread
    for (int r = r0; r < r1; ++r) {
      const PagedRequest q = paged_request(p, r);
      const int64_t head = head_blocks(p, q), n = head * p.heads_kv;
      if (begin >= at + n) {
        at += n;
        continue;
      }
      const int64_t x = begin - at, h = divide(x, head);
      s.r = r;
      s.h = int(h);
      s.tile = q.tiles(p) == 1 ? 0 : -1;  // -1: still to be found
      scratch[0] = x - h * head;
      s.off = int(scratch[0]);
      *start = s;
      break;
    }
  }
  __syncthreads();
  if (start->tile == 0) return;
  // The tile: every thread looks at the beginning of one in `step`.
  const PagedRequest q = paged_request(p, start->r);
  const int64_t rest = scratch[0];
  int lo = 0, n = q.tiles(p);
  while (true) {
    const int step = (n + nt - 1) / nt;
    const int t = lo + tid * step;
    __syncthreads();
    if (t < lo + n) {
      const int64_t before = blocks_before(p, q, t);
      if (before <= rest && rest < blocks_before(p, q, min(t + step, lo + n))) {
        start->tile = t;
        start->off = int(rest - before);
      }
    }
    __syncthreads();
    lo = start->tile;
    if (step == 1) break;
    n = min(step, q.tiles(p) - lo);
  }
}

// Walks a worker's items; every role of a kernel walks the same ones.
struct PagedWalk {
  int r, h, tile, off;
  int64_t left;
  PagedRequest req;
  PagedBlocks blocks;
  int take;  // blocks of the current item in this stretch, from block `off` on

  __device__ __forceinline__ PagedWalk(const PagedParams& p, const PagedStart& s)
      : r(s.r), h(s.h), tile(s.tile), off(s.off), left(s.count) {
    if (left > 0) load(p);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void load(const PagedParams& p) {
    req = paged_request(p, r);
    set(p);
  }
  __device__ __forceinline__ void set(const PagedParams& p) {
    blocks = paged_blocks(p, req, tile);
    const int n = blocks.n - off;
    take = n < left ? n : int(left);
  }
  __device__ __forceinline__ bool begins() const { return off == 0; }
  __device__ __forceinline__ bool ends() const { return off + take == blocks.n; }
  __device__ __forceinline__ void next(const PagedParams& p) {
    left -= take;
    off = 0;
    if (left <= 0) return;
    if (++tile == req.tiles(p)) {
      tile = 0;
      if (++h == p.heads_kv) {
        h = 0;
        do req = paged_request(p, ++r);
        while (req.len == 0 && r + 1 < p.requests);
      }
    }
    set(p);
  }
};

// The record of an item that begins in a worker's stretch and ends in another's.
struct PagedRecord {
  int32_t parts;   // stretches the item covers; 0: the worker has no such item
  int32_t row0;    // its first token in q
  int32_t tokens;  // tokens of the tile
  int32_t h;
  int32_t spare[4];
};
static_assert(sizeof(PagedRecord) == kPagedRecord, "record size");

__device__ __forceinline__ PagedRecord* paged_record(const PagedParams& p, int worker) {
  return reinterpret_cast<PagedRecord*>(p.ws + kPagedHeader) + worker;
}

// One thread of a warp with no other role: the worker's record.
__device__ __forceinline__ void write_record(const PagedParams& p, const PagedStart& s, int worker) {
  PagedRecord rec{0, 0, 0, 0, {0, 0, 0, 0}};
  for (PagedWalk w(p, s); w.more(); w.next(p)) {
    if (!w.begins() || w.ends()) continue;
    const int t0 = w.tile * p.tokens_per_tile, left = w.req.len - t0;
    rec.parts = s.owner(s.begin(worker + 1) + (w.blocks.n - (w.off + w.take)) - 1) - worker + 1;
    rec.row0 = w.req.q0 + t0;
    rec.tokens = left < p.tokens_per_tile ? left : p.tokens_per_tile;
    rec.h = w.h;
  }
  *paged_record(p, worker) = rec;
}

// Partial slot s: [rows][128] outputs, then [rows] maxima, then [rows] sums.
__device__ __forceinline__ float* paged_partial(const PagedParams& p, int slot) {
  return reinterpret_cast<float*>(p.ws + kPagedPartials) + size_t(slot) * size_t(p.part_rows) * 130u;
}

__device__ __forceinline__ void paged_status(const PagedParams& p, uint32_t code, uint32_t site) {
  if (atomicCAS(&p.status[0], 0u, code) == 0u) {
    p.status[1] = site;
    p.status[2] = blockIdx.x;
  }
}

// A launch that may begin before the work ahead of it in the stream has ended:
// the kernel waits for that itself (grid_wait) before it touches memory, and
// what can be done before -- barriers, tensor memory, descriptors -- is done.
inline cudaError_t launch_early(void (*kernel)(PagedParams), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                const PagedParams& p) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// The chunk kernel (paged_chunk.cu): workers are CTA pairs.  0 or a CUDA error.
using PagedChunkKernel = void (*)(PagedParams);
int paged_chunk_setup(int* pairs);
int paged_chunk_launch(const PagedParams& p, bool bf16, cudaStream_t stream);

}  // namespace b200fa
