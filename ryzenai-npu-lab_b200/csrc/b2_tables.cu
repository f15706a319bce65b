// Block tables and slot maps built on the GPU (include/b2_tables.h):
//
//   extend_kernel   blocks for new tokens off the end of the free list, in
//                   request order: prefix sums of rows and of needed blocks;
//                   for few rows their slots and positions too
//   slot_kernel     slot and position of every new token's row
//   release_kernel  blocks of finished requests back to the free list
//
// The work is a few bytes per request and eight per row: bound by launch and
// memory latency, so each call is one or two launches and no thread waits for
// another CTA.

#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "b2_decode_attn.h"
#include "b2_internal.h"
#include "b2_tables.h"

namespace {

constexpr int kBlock = 64;
constexpr int kScanThreads = 1024;
constexpr int kSlotThreads = 128;
// Rows that extend_kernel writes itself, one per thread: 64 requests x 1 row 4.7 us,
// with slot_kernel behind 6.1; 1000 x 1: 6.4, 7.4; from there slot_kernel gains
// (1000 x 4: 7.5 us, 10.0 without it).
constexpr int kRowsHere = kScanThreads;
// Rows from which a thread of slot_kernel takes 8 instead of 1: 65 536 rows 4.9 us
// against 3.1, 524 288 6.1 against 6.2, a million 7.2 against 10.4.
constexpr int kRowsWide = 1 << 19;
constexpr int kExtendCtas = 8;           // cluster of extend_kernel for more than kScanThreads requests
constexpr int kFewBlocks = 16;           // blocks that a thread fetches for its own request
constexpr int32_t kMaxTableWidth = (1 << 25) - 1;  // width x 64 tokens stay an int32
constexpr int32_t kMaxPoolBlocks = (1 << 22) - 1;

int fail(int code, const char *msg) { return b2_record_error(code, msg); }

// Exclusive prefix sum of `v` over the CTA; `total` gets the CTA's sum.
__device__ __forceinline__ int64_t scan_exclusive(int64_t v, int64_t *warp_sum, int64_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t incl = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += u;
  }
  __syncthreads();  // warp_sum's last reads are done
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t w = lane < kScanThreads / 32 ? warp_sum[lane] : 0;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, w, off);
    if (lane >= off) w += u;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int64_t before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return incl - v + (warp > 0 ? before : 0);
}

// Largest i in [0, n) with start[i] <= x, or -1.
template <class T>
__device__ __forceinline__ int last_at_or_below(const T *start, int n, T x) {
  int lo = -1, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

struct SlotArgs {
  const int32_t *tables;
  int max_blocks, num_blocks;
  const int32_t *past, *fresh, *granted, *row_start;
  int batch;
  int32_t *slots, *positions;
  int rows, tokens;
  int32_t *err;  // NULL: faults were reported before
};

// Request b of a slot map can be placed: as extend_kernel's `bad`, with its first row.
__device__ __forceinline__ bool request_fits(const SlotArgs &a, int64_t start, int past, int fresh) {
  return past >= 0 && fresh >= 0 && static_cast<int64_t>(past) + fresh <= static_cast<int64_t>(a.max_blocks) * kBlock &&
         (a.row_start ? fresh == 0 || (start >= 0 && start + fresh <= a.rows) : fresh <= a.tokens);
}

// Rows r0 .. r0 + kSlotRows - 1, ascending from request b on (the last one that
// starts at or before r0): eight rows share the search for their request and
// leave as 16-byte stores; one row per thread keeps few rows' loads parallel.
template <bool kPadded, int kSlotRows>
__device__ __forceinline__ void write_rows(const SlotArgs &a, int64_t r0, int b) {
  int slot[kSlotRows], position[kSlotRows];
  int64_t start = 0;
  int past = 0, fresh = 0, flag = 0, held_blk = -1, blk = -1;
  bool granted = false;
  auto request = [&]() {
    const bool in = b >= 0 && b < a.batch;
    start = !in ? 0 : (kPadded ? static_cast<int64_t>(b) * a.tokens : a.row_start[b]);
    past = in ? a.past[b] : 0;
    fresh = in ? a.fresh[b] : 0;
    granted = in && (a.granted ? a.granted[b] > 0 : request_fits(a, start, past, fresh));
    held_blk = -1;
  };
  request();
#pragma unroll
  for (int i = 0; i < kSlotRows; ++i) {
    const int64_t r = r0 + i;
    slot[i] = -1;
    position[i] = 0;
    if (r >= a.rows) continue;
    if (kPadded) {
      if (r - start >= a.tokens) {
        ++b;
        request();
      }
    } else {
      bool moved = false;
      while (b + 1 < a.batch && a.row_start[b + 1] <= r) {
        ++b;
        moved = true;
      }
      if (moved) request();
    }
    const int64_t t = r - start;
    if (b < 0 || b >= a.batch || t >= fresh) continue;
    const int64_t pos = past + t;
    position[i] = static_cast<int>(pos);
    if (!granted) continue;
    if (pos < 0 || pos >= static_cast<int64_t>(a.max_blocks) * kBlock) continue;  // (starts that do not ascend)
    const int logical = static_cast<int>(pos / kBlock);
    if (logical != held_blk) {
      blk = a.tables[static_cast<int64_t>(b) * a.max_blocks + logical];
      held_blk = logical;
    }
    if (blk < 0 || blk >= a.num_blocks) flag |= B2_DEV_BAD_BLOCK;
    else slot[i] = blk * kBlock + static_cast<int>(pos % kBlock);
  }
  if (flag && a.err) atomicOr(a.err, flag);
  const bool wide = kSlotRows >= 4 && r0 + kSlotRows <= a.rows &&
                    ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  if (wide) {
#pragma unroll
    for (int i = 0; i + 3 < kSlotRows; i += 4) {
      *reinterpret_cast<int4 *>(a.slots + r0 + i) = make_int4(slot[i], slot[i + 1], slot[i + 2], slot[i + 3]);
      *reinterpret_cast<int4 *>(a.positions + r0 + i) =
          make_int4(position[i], position[i + 1], position[i + 2], position[i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kSlotRows; ++i)
      if (r0 + i < a.rows) {
        a.slots[r0 + i] = slot[i];
        a.positions[r0 + i] = position[i];
      }
  }
}

// Rows r0 .. of any request.
template <int kSlotRows>
__device__ __forceinline__ void find_and_write_rows(const SlotArgs &a, int64_t r0) {
  if (!a.row_start) write_rows<true, kSlotRows>(a, r0, static_cast<int>(r0 / a.tokens));
  else write_rows<false, kSlotRows>(a, r0, last_at_or_below<int32_t>(a.row_start, a.batch, static_cast<int32_t>(r0)));
}

struct ExtendArgs {
  int32_t *tables;
  int max_blocks;
  const int32_t *held, *free_list;
  int num_blocks;
  const int32_t *free_count, *past, *fresh;
  int batch;
  int32_t *held_out, *count_out, *granted, *row_start;
  int rows, tokens;
  int32_t *err;
  SlotArgs slots;  // rows > 0: to be written here
};

// One CTA walks the requests, kPer per thread and kScanThreads * kPer at a time:
// prefix sums of their rows and needed blocks, then the new table entries of the
// chunk spread over all threads (an entry finds its request by bisection of the
// chunk's sums), so one request of many blocks costs no more than many of one.
// The requests that get blocks are the first ones that need any, so their sums
// of needed blocks are their places on the free list.
//
// Many requests' entries are scattered 4-byte stores, about one per clock of an
// SM (16 000 entries: 11 of 20 us), so a cluster of kCtas CTAs computes the sums
// alike and shares the stores.  held_out and free_count_out may be the inputs: a
// cluster barrier stands between each chunk's loads and its stores.
template <int kPer, int kCtas>
__global__ void __launch_bounds__(kScanThreads) extend_kernel(const ExtendArgs a) {
  __shared__ int64_t warp_sum[kScanThreads / 32];
  __shared__ int32_t first[kScanThreads * kPer];  // exclusive sums of the blocks needed in this chunk
  __shared__ int32_t from[kScanThreads * kPer];   // blocks held before
  __shared__ unsigned long long taken_here;       // blocks given to the chunk's requests
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int cta = static_cast<int>(blockIdx.x);                           // of the cluster
  const bool own = static_cast<int>(threadIdx.x) / (kScanThreads / kCtas) == cta;  // this CTA stores for this thread's requests
  int64_t count = a.free_count[0];
  int flag = 0;
  if (count < 0 || count > a.num_blocks) {
    flag = B2_DEV_BAD_LENGTH;
    count = count < 0 ? 0 : a.num_blocks;
  }
  int64_t rows_before = 0, need_before = 0, taken = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kScanThreads * kPer) {
    const int i0 = static_cast<int>(threadIdx.x) * kPer;
    int past[kPer], fresh[kPer], held[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = b0 + i0 + e;
      past[e] = b < a.batch ? a.past[b] : 0;
      fresh[e] = b < a.batch ? a.fresh[b] : 0;
      held[e] = b < a.batch ? a.held[b] : 0;
    }
    if (threadIdx.x == 0) taken_here = 0;
    if (kCtas > 1) {
      asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    }
    int64_t total = 0, start[kPer], need[kPer], mine = 0;
    if (a.tokens == 0) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) mine += fresh[e] > 0 ? fresh[e] : 0;
      int64_t at = rows_before + scan_exclusive(mine, warp_sum, total);
      rows_before += total;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        start[e] = at;
        at += fresh[e] > 0 ? fresh[e] : 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) start[e] = static_cast<int64_t>(b0 + i0 + e) * a.tokens;
    }
    bool bad[kPer];
    mine = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int64_t upto = static_cast<int64_t>(past[e]) + fresh[e];
      bad[e] = past[e] < 0 || fresh[e] < 0 || held[e] < 0 || held[e] > a.max_blocks ||
               upto > static_cast<int64_t>(a.max_blocks) * kBlock || (a.tokens > 0 && fresh[e] > a.tokens) ||
               (a.tokens == 0 && fresh[e] > 0 && start[e] + fresh[e] > a.rows);
      if (bad[e]) flag |= B2_DEV_BAD_LENGTH;
      const int64_t blocks = (upto + kBlock - 1) / kBlock;
      need[e] = !bad[e] && blocks > held[e] ? blocks - held[e] : 0;
      mine += need[e];
    }
    int64_t pre = scan_exclusive(mine, warp_sum, total);
    int64_t end = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = b0 + i0 + e;
      first[i0 + e] = pre < 0x7fffffff ? static_cast<int32_t>(pre) : 0x7fffffff;  // (no list is that long)
      from[i0 + e] = held[e];
      const bool ok = !bad[e] && (need[e] == 0 || need_before + pre + need[e] <= count);
      pre += need[e];
      if (ok && need[e] > 0) end = pre;
      if (own && b < a.batch) {
        a.held_out[b] = held[e] + (ok ? static_cast<int32_t>(need[e]) : 0);
        a.granted[b] = ok ? fresh[e] : 0;
        a.row_start[b] = static_cast<int32_t>(start[e] < a.rows ? start[e] : a.rows);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const int64_t u = __shfl_xor_sync(0xffffffffu, end, off);
      end = u > end ? u : end;
    }
    if ((threadIdx.x & 31) == 0 && end > 0) atomicMax(&taken_here, static_cast<unsigned long long>(end));
    __syncthreads();
    const int chunk = static_cast<int>(taken_here);
    auto block = [&](int64_t e) {  // the e-th block of the chunk
      const int id = a.free_list[count - 1 - (need_before + e)];
      if (id >= 0 && id < a.num_blocks) return id;
      flag |= B2_DEV_BAD_BLOCK;
      return -1;
    };
    // few blocks per request: its own thread fetches them; else the entries are
    // spread over all threads
    bool few = true;
#pragma unroll
    for (int e = 0; e < kPer; ++e) few = few && need[e] <= kFewBlocks;
    if (__syncthreads_and(few)) {
#pragma unroll
      for (int e = 0; e < kPer && own; ++e) {
        const int at = first[i0 + e];
        int32_t *entry = a.tables + static_cast<int64_t>(b0 + i0 + e) * a.max_blocks + held[e];
#pragma unroll 4
        for (int i = 0; i < static_cast<int>(need[e]) && at + i < chunk; ++i) entry[i] = block(at + i);
      }
    } else
    for (int e = cta * kScanThreads + threadIdx.x; e < chunk; e += kCtas * kScanThreads) {
      const int i = last_at_or_below<int32_t>(first, kScanThreads * kPer, e);
      a.tables[static_cast<int64_t>(b0 + i) * a.max_blocks + from[i] + (e - first[i])] = block(e);
    }
    taken += chunk;
    need_before += total;  // with what was refused: nobody behind a refused request gets a block
    __syncthreads();
  }
  if (flag) atomicOr(a.err, flag);
  __syncthreads();  // every thread has read the old count, and sees the starts, grants and entries
  if (cta == 0 && threadIdx.x == 0) a.count_out[0] = static_cast<int32_t>(count - taken);
  if (kCtas == 1 && a.slots.rows > 0)
    for (int64_t r = threadIdx.x; r < a.slots.rows; r += kScanThreads) find_and_write_rows<1>(a.slots, r);
}

template <int kSlotRows>
__global__ void __launch_bounds__(kSlotThreads) slot_kernel(const SlotArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t thread = static_cast<int64_t>(blockIdx.x) * kSlotThreads + threadIdx.x, r0 = thread * kSlotRows;
  if (a.err) {  // requests that are refused, whether a row shows them or not
    bool bad = false;
    for (int64_t b = thread; b < a.batch; b += static_cast<int64_t>(gridDim.x) * kSlotThreads)
      bad = bad || !request_fits(a, a.row_start ? a.row_start[b] : b * a.tokens, a.past[b], a.fresh[b]);
    if (bad) atomicOr(a.err, B2_DEV_BAD_LENGTH);
  }
  if (r0 < a.rows) find_and_write_rows<kSlotRows>(a, r0);
}

struct ReleaseArgs {
  int32_t *tables;
  int max_blocks;
  int32_t *held, *free_list;
  int num_blocks;
  int32_t *free_count;
  const uint8_t *finished;
  int batch;
  int32_t *err;
};

__global__ void __launch_bounds__(kScanThreads) release_kernel(const ReleaseArgs a) {
  __shared__ int64_t warp_sum[kScanThreads / 32];
  __shared__ int64_t first[kScanThreads];
  const int64_t count = a.free_count[0];
  // first the sum over all requests: nothing is released that does not fit
  int64_t mine = 0, sum = 0;
  bool bad = count < 0;
  for (int b = threadIdx.x; b < a.batch; b += kScanThreads)
    if (a.finished[b]) {
      const int h = a.held[b];
      if (h < 0 || h > a.max_blocks) bad = true;
      else mine += h;
    }
  scan_exclusive(mine, warp_sum, sum);
  bad = __syncthreads_or(bad) || count + sum > a.num_blocks;
  if (bad) {
    if (threadIdx.x == 0) atomicOr(a.err, B2_DEV_BAD_LENGTH);
    return;
  }
  int64_t at = count;
  for (int b0 = 0; b0 < a.batch; b0 += kScanThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    const int64_t n = b < a.batch && a.finished[b] ? a.held[b] : 0;
    int64_t chunk = 0;
    first[threadIdx.x] = scan_exclusive(n, warp_sum, chunk);
    __syncthreads();
    for (int64_t e = threadIdx.x; e < chunk; e += kScanThreads) {
      const int i = last_at_or_below<int64_t>(first, kScanThreads, e);
      int32_t *entry = a.tables + static_cast<int64_t>(b0 + i) * a.max_blocks + (e - first[i]);
      a.free_list[at + e] = *entry;
      *entry = -1;
    }
    if (n > 0) a.held[b] = 0;
    at += chunk;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.free_count[0] = static_cast<int32_t>(at);
}

int launched(cudaError_t e, const char *what) {
  const cudaError_t sticky = cudaGetLastError();
  if (e == cudaSuccess) e = sticky;
  if (e == cudaSuccess) return b2_clear_error();
  char msg[256];
  snprintf(msg, sizeof(msg), "%s launch failed: %s", what, cudaGetErrorString(e));
  return fail(B2_ERR_CUDA, msg);
}

// `dependent`: after extend_kernel, whose launch it overlaps.
int launch_slots(const SlotArgs &a, bool dependent, cudaStream_t st) {
  if (a.rows == 0) return b2_clear_error();
  cudaLaunchConfig_t cfg = {};
  const bool wide = a.rows >= kRowsWide;
  const int per = kSlotThreads * (wide ? 8 : 1);
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(a.rows) + per - 1) / per));
  cfg.blockDim = dim3(kSlotThreads);
  cfg.stream = st;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = dependent ? 1 : 0;
  return launched(wide ? cudaLaunchKernelEx(&cfg, slot_kernel<8>, a) : cudaLaunchKernelEx(&cfg, slot_kernel<1>, a),
                  "slot_kernel");
}

int check_sizes(int32_t max_blocks, int32_t num_blocks, int32_t batch, int32_t rows, int32_t tokens) {
  if (batch < 0 || rows < 0 || tokens < 0) return fail(B2_ERR_ARG, "batch, rows and tokens_per_seq must be >= 0");
  if (max_blocks <= 0 || max_blocks > kMaxTableWidth)
    return fail(B2_ERR_ARG, "max_blocks_per_seq must be in [1, 2^25)");
  if (num_blocks <= 0 || num_blocks > kMaxPoolBlocks) return fail(B2_ERR_ARG, "num_blocks must be in [1, 2^22)");
  if (tokens > 0 && static_cast<int64_t>(batch) * tokens != rows)
    return fail(B2_ERR_ARG, "rows must be batch * tokens_per_seq");
  return B2_OK;
}

}  // namespace

extern "C" int b2_tables_extend(int32_t *block_tables, int32_t max_blocks_per_seq, const int32_t *held,
                                const int32_t *free_list, int32_t num_blocks, const int32_t *free_count,
                                const int32_t *past_lens, const int32_t *new_lens, int32_t batch, int32_t *held_out,
                                int32_t *free_count_out, int32_t *granted, int32_t *row_start, int32_t *slots,
                                int32_t *positions, int32_t rows, int32_t tokens_per_seq, int32_t *dev_err,
                                void *stream) {
  const int rc = check_sizes(max_blocks_per_seq, num_blocks, batch, rows, tokens_per_seq);
  if (rc) return rc;
  if (!free_list || !free_count || !free_count_out || !dev_err ||
      (batch > 0 && (!block_tables || !held || !past_lens || !new_lens || !held_out || !granted || !row_start)) ||
      (rows > 0 && (!slots || !positions)))
    return fail(B2_ERR_ARG, "b2_tables_extend: null pointer argument");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  SlotArgs s{block_tables, max_blocks_per_seq, num_blocks, past_lens, new_lens, granted,
             tokens_per_seq > 0 ? nullptr : row_start, batch, slots, positions, rows, tokens_per_seq, nullptr};
  ExtendArgs a{block_tables, max_blocks_per_seq, held, free_list, num_blocks, free_count, past_lens, new_lens, batch,
               held_out, free_count_out, granted, row_start, rows, tokens_per_seq, dev_err, s};
  // few rows are written by the CTA that has the sums: one launch
  const bool one = batch <= kScanThreads, here = one && rows <= kRowsHere;
  if (!here) a.slots.rows = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(one ? 1 : kExtendCtas);
  cfg.blockDim = dim3(kScanThreads);
  cfg.stream = st;
  cudaLaunchAttribute cluster[1];
  cluster[0].id = cudaLaunchAttributeClusterDimension;
  cluster[0].val.clusterDim.x = kExtendCtas;
  cluster[0].val.clusterDim.y = 1;
  cluster[0].val.clusterDim.z = 1;
  cfg.attrs = cluster;
  cfg.numAttrs = one ? 0 : 1;
  const int lrc = launched(one ? cudaLaunchKernelEx(&cfg, extend_kernel<1, 1>, a)
                               : cudaLaunchKernelEx(&cfg, extend_kernel<4, kExtendCtas>, a),
                           "extend_kernel");
  return lrc || here ? lrc : launch_slots(s, true, st);
}

extern "C" int b2_slot_map(const int32_t *block_tables, int32_t max_blocks_per_seq, int32_t num_blocks,
                           const int32_t *past_lens, const int32_t *new_lens, const int32_t *row_start, int32_t batch,
                           int32_t *slots, int32_t *positions, int32_t rows, int32_t tokens_per_seq, int32_t *dev_err,
                           void *stream) {
  const int rc = check_sizes(max_blocks_per_seq, num_blocks, batch, rows, row_start ? 0 : tokens_per_seq);
  if (rc) return rc;
  if (!row_start && tokens_per_seq <= 0 && rows > 0)
    return fail(B2_ERR_ARG, "b2_slot_map: row_start or tokens_per_seq > 0 is required");
  if (rows == 0) return b2_clear_error();
  if (!slots || !positions || !dev_err || (batch > 0 && (!block_tables || !past_lens || !new_lens)))
    return fail(B2_ERR_ARG, "b2_slot_map: null pointer argument");
  SlotArgs s{block_tables, max_blocks_per_seq, num_blocks, past_lens, new_lens, nullptr, row_start, batch,
             slots, positions, rows, row_start ? 0 : tokens_per_seq, dev_err};
  return launch_slots(s, false, static_cast<cudaStream_t>(stream));
}

extern "C" int b2_tables_release(int32_t *block_tables, int32_t max_blocks_per_seq, int32_t *held, int32_t *free_list,
                                 int32_t num_blocks, int32_t *free_count, const uint8_t *finished, int32_t batch,
                                 int32_t *dev_err, void *stream) {
  const int rc = check_sizes(max_blocks_per_seq, num_blocks, batch, 0, 0);
  if (rc) return rc;
  if (batch == 0) return b2_clear_error();
  if (!block_tables || !held || !free_list || !free_count || !finished || !dev_err)
    return fail(B2_ERR_ARG, "b2_tables_release: null pointer argument");
  ReleaseArgs a{block_tables, max_blocks_per_seq, held, free_list, num_blocks, free_count, finished, batch, dev_err};
  release_kernel<<<1, kScanThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launched(cudaSuccess, "release_kernel");
}
