// The 8-bit paged KV cache (include/b2_kv8.h): e4m3 codes with a power-of-two
// scale for each block of 64 tokens and KV head.
//
//   kv8_append_kernel  q/k norm + RoPE and the quantised append of new tokens
//   kv8_step_kernel    a whole decode step: append and split attention
//   kv8_prefill_kernel causal attention of a prompt chunk over the cache (tcgen05)
//   kv8_merge_kernel   merge of a prompt tile's keys split over CTAs

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "b2_decode_attn.h"
#include "b2_device.cuh"
#include "b2_internal.h"
#include "b2_kv8.h"

namespace {

constexpr int kHq = 16;
constexpr int kHkv = 8;
constexpr int kBlock = 64;
constexpr int kQkvWidth = (kHq + 2 * kHkv) * kDim;  // 2048
constexpr int kTile = kBlock * kDim;                // codes (bytes) of one (block, head): 4 KiB
constexpr int kMaxStepTokens = 4;
constexpr int32_t kMaxTableWidth = (1 << 25) - 1;  // width x 64 tokens stay an int32
constexpr int32_t kMaxPoolBlocks = (1 << 22) - 1;
constexpr float kBf16Max = 3.3895313892515355e38f;
constexpr int kMinScaleExp = -100;

int fail(int code, const char *msg) { return b2_record_error(code, msg); }
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int launched(cudaError_t e, const char *what) {
  const cudaError_t sticky = cudaGetLastError();
  if (e == cudaSuccess) e = sticky;
  if (e == cudaSuccess) return b2_clear_error();
  char msg[256];
  snprintf(msg, sizeof(msg), "%s launch failed: %s", what, cudaGetErrorString(e));
  return fail(B2_ERR_CUDA, msg);
}

// ------------------------------------------------------------------ codes and scales

// Two floats as e4m3 codes (lo in the low byte), nearest even, limited to +-448.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// |x| limited to the largest finite bf16; NaN stays NaN (fmaxf then drops it).
__device__ __forceinline__ float limited_abs(float x) {
  const float a = fabsf(x);
  return a > kBf16Max ? kBf16Max : a;
}

__device__ __forceinline__ float limited(float x) {
  return x > kBf16Max ? kBf16Max : (x < -kBf16Max ? -kBf16Max : x);
}

// The smallest 2^e >= 2^kMinScaleExp with amax <= 448 * 2^e: 448 = 1.75 * 2^8,
// so e is amax's exponent - 8, one more when its mantissa is over 1.75.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < kMinScaleExp ? kMinScaleExp : e;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// 16 codes moved to another scale (ratio = old / new <= 1), those with index
// < keep; the others stay.
__device__ __forceinline__ uint4 rescale16(uint4 w, float ratio, int keep) {
  uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 lo = from_e4m3x2(u[i]), hi = from_e4m3x2(u[i] >> 16);
    const uint32_t y = e4m3x2(lo.x * ratio, lo.y * ratio) | (e4m3x2(hi.x * ratio, hi.y * ratio) << 16);
    const int n = keep - 4 * i;
    const uint32_t mask = n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
    u[i] = (y & mask) | (u[i] & ~mask);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
  return x;
}

// ------------------------------------------------------------------ append

struct AppendArgs {
  const uint16_t *qkv;
  int64_t row_stride;
  int rows;
  const int32_t *slots, *positions;
  const int32_t *past_lens, *chunk_lens;
  int tokens;
  const int32_t *block_tables;
  int max_blocks;
  const uint16_t *gamma_q, *gamma_k;
  float eps;
  const uint16_t *cos, *sin;
  int rope_rows;
  uint8_t *k_pool, *v_pool;
  float *k_scale, *v_scale;
  int num_blocks;
  uint16_t *q_out;
  int mode;
  int32_t *err;
};

constexpr int kMaxWindow = 32;   // rows whose runs start in one CTA: 8 or 32, at most a warp's lanes
constexpr int kNoSlot = -1;
constexpr int kAppendWarps = 4;  // K and V of two heads
constexpr int kAppendThreads = kAppendWarps * 32;

// A run's rows of one head, K or V, per warp, and the places of the rows around.
struct AppendShared {
  uint16_t rows[kAppendWarps][kBlock][kDim];
  int slot[1 + kMaxWindow + kBlock + 1], place[1 + kMaxWindow + kBlock + 1];  // entry i: row row0 - 1 + i
};

// Slot and RoPE position of a row; kNoSlot for a row to skip.
__device__ __forceinline__ int row_place(const AppendArgs &a, int row, int &position, int &flag) {
  position = 0;
  if (a.slots) {
    const int s = a.slots[row];
    if (s < 0) return kNoSlot;
    if (s >= a.num_blocks * kBlock) {
      flag |= B2_DEV_BAD_BLOCK;
      return kNoSlot;
    }
    if (a.positions) position = a.positions[row];
    return s;
  }
  const int b = row / a.tokens, t = row - b * a.tokens;
  const int chunk = a.chunk_lens ? a.chunk_lens[b] : a.tokens;
  const int64_t past = a.past_lens[b], pos = past + t;
  if (chunk == 0) return kNoSlot;
  // lengths that do not fit refuse the sequence whole, as the attention does: its cached tokens stay as they are
  if (past < 0 || chunk < 0 || chunk > a.tokens || past + chunk > static_cast<int64_t>(a.max_blocks) * kBlock) {
    flag |= B2_DEV_BAD_LENGTH;
    return kNoSlot;
  }
  if (t >= chunk) return kNoSlot;
  position = static_cast<int>(pos);
  if (!(a.mode & B2_STORE_KV)) return 0;
  const int blk = a.block_tables[static_cast<int64_t>(b) * a.max_blocks + pos / kBlock];
  if (blk < 0 || blk >= a.num_blocks) {
    flag |= B2_DEV_BAD_BLOCK;
    return kNoSlot;
  }
  return blk * kBlock + static_cast<int>(pos % kBlock);
}

// One warp: the nearest row up to r with a slot lies in block `blk`.
__device__ __forceinline__ bool block_in_front(const AppendArgs &a, int r, int blk) {
  const int lane = threadIdx.x & 31;
  for (; r >= 0; r -= 32) {
    const int s = r - lane >= 0 ? a.slots[r - lane] : kNoSlot;
    const uint32_t there = __ballot_sync(0xffffffffu, s >= 0 && s < a.num_blocks * kBlock);
    if (there) return __shfl_sync(0xffffffffu, s, __ffs(there) - 1) / kBlock == blk;
  }
  return false;
}

// One CTA per window of rows and pair of heads, warp = (KV head, K or V).  A run
// is a sequence of adjacent rows that go to adjacent slots of one block; the
// warps of the window that holds its first row quantise the whole run, each for
// its head, so a block's scale is found and its codes are written by one warp
// alone, with no atomics.  A run's loads are copies to shared memory, all in
// flight together (up to 16 per lane; 8 lanes own one 64-wide head vector) and
// without registers, from where norm and RoPE, the maximum and the codes are
// taken.  Codes leave in 16-byte pieces: a lane takes 16 dims of a K row, or 16
// tokens of two V dims, for which shared memory is the transpose.
//
// Bound by latency: a run's loads, its codes, its stores (64 x 128 tokens 14 us,
// 8 of them the loads; 21 tokens 4.4 us).  A warp takes the runs of its window in
// turn, so many short runs want kWindow 8 (256 sequences x 4 tokens 7.5 us, with
// 32 17.9; 128 x 16: 7.5, 9.1), while CTAs that hold no run's start only cost in
// long prompts (one of 1024 tokens 7.2 us, with 32 5.0; 32 x 32: 7.8, 6.1; 64 x
// 128 10 % slower, with 64 15-25 %).  Where the rows' runs are not known (slots),
// up to 1024 rows take 8.
template <int kWindow>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const AppendArgs a) {
  extern __shared__ uint8_t smem_raw[];
  AppendShared &sh = *reinterpret_cast<AppendShared *>(smem_raw);
  const int row0 = static_cast<int>(blockIdx.x) * kWindow;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane & 7, grp = lane >> 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int i = threadIdx.x; i < 1 + kWindow + kBlock; i += kAppendThreads) {
    const int64_t r = static_cast<int64_t>(row0) - 1 + i;
    int position = 0, flag = 0;
    sh.slot[i] = r >= 0 && r < a.rows ? row_place(a, static_cast<int>(r), position, flag) : kNoSlot;
    sh.place[i] = position;
    if (i >= 1 && i <= kWindow && blockIdx.y == 0) {
      if (sh.slot[i] >= 0 && (a.mode & B2_ROPE_QK) && (position < 0 || position >= a.rope_rows))
        flag |= B2_DEV_BAD_POSITION;
      if (flag) atomicOr(a.err, flag);
    }
  }
  __syncthreads();
  const bool norm = (a.mode & B2_NORM_QK) != 0, rope = (a.mode & B2_ROPE_QK) != 0;
  // norm and RoPE of four head vectors (one per 8 lanes) of the rows at entries i
  auto turn = [&](float x[8], int i, const uint16_t *gamma) {
    const int pos = sh.place[i];
    const bool on = rope && pos >= 0 && pos < a.rope_rows;
    norm_rope8(x, j, norm, on, gamma, a.eps, on ? a.cos + static_cast<int64_t>(pos) * kDim : nullptr,
               on ? a.sin + static_cast<int64_t>(pos) * kDim : nullptr);
  };

  if (a.q_out) {
    // four query heads of a row per pass, the passes of the window's rows over the warps
    for (int p = static_cast<int>(blockIdx.y) * kAppendWarps + warp; p < kWindow * (kHq / 4);
         p += static_cast<int>(gridDim.y) * kAppendWarps) {
      const int i = 1 + p / (kHq / 4), vec = 4 * (p % (kHq / 4)) + grp;
      if (sh.slot[i] < 0) continue;
      const int64_t r = row0 - 1 + i;
      float x[8];
      unpack8(__ldg(reinterpret_cast<const uint4 *>(a.qkv + r * a.row_stride + vec * kDim + j * 8)), x);
      if (norm || rope) turn(x, i, a.gamma_q);
      *reinterpret_cast<uint4 *>(a.q_out + (r * kHq + vec) * kDim + j * 8) = pack8(x);
    }
  }
  if (!(a.mode & B2_STORE_KV)) return;

  const int h = static_cast<int>(blockIdx.y) * (kAppendWarps / 2) + (warp >> 1);
  const bool is_v = warp & 1;
  uint16_t(*rows)[kDim] = sh.rows[warp];
  // rows of the window that start a run: valid, and not the slot behind the row before in the same block
  const int here = lane < kWindow ? sh.slot[1 + lane] : kNoSlot, before = lane < kWindow ? sh.slot[lane] : kNoSlot;
  uint32_t starts = __ballot_sync(0xffffffffu, here >= 0 && (before < 0 || before + 1 != here || here % kBlock == 0));
  for (; starts; starts &= starts - 1) {
    const int i0 = __ffs(starts), s0 = sh.slot[i0], front = sh.slot[i0 - 1];
    const int blk = s0 / kBlock, r0 = s0 % kBlock;
    // rows of this block in front of the run belong to another warp, which writes its scale: refused
    if (front >= 0 ? front / kBlock == blk : a.slots && r0 > 0 && block_in_front(a, row0 + i0 - 3, blk)) {
      if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.err, B2_DEV_BAD_SLOT);
      continue;
    }
    // rows that follow: 1 + lane, 33 + lane behind the first
    const uint32_t m0 = __ballot_sync(0xffffffffu, r0 + 1 + lane < kBlock && sh.slot[i0 + 1 + lane] == s0 + 1 + lane);
    const uint32_t m1 = __ballot_sync(0xffffffffu, r0 + 33 + lane < kBlock && sh.slot[i0 + 33 + lane] == s0 + 33 + lane);
    const int n = 1 + (m0 != 0xffffffffu ? __ffs(~m0) - 1 : 32 + __ffs(~m1) - 1);  // lane 31 of m1 would be row 64
    const uint16_t *src = a.qkv + (static_cast<int64_t>(row0) - 1 + i0 + grp) * a.row_stride +
                          (kHq + (is_v ? kHkv : 0) + h) * kDim + j * 8;
    const uint32_t dst = smem_u32(&rows[grp][8 * j]);
    for (int i = 0; i < n; i += 4)
      if (i + grp < n)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * kDim * 2), "l"(src + i * a.row_stride)
                     : "memory");
    const int64_t id = static_cast<int64_t>(blk) * kHkv + h;
    float *sp = (is_v ? a.v_scale : a.k_scale) + id;
    uint8_t *codes = (is_v ? a.v_pool : a.k_pool) + id * kTile;
    const float old = r0 > 0 ? *sp : 0.f;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    const bool turned = !is_v && (norm || rope);
    float amax = 0.f;
#pragma unroll 4
    for (int i = 0; i < n; i += 4) {
      const bool live = i + grp < n;
      float x[8];
      unpack8(live ? *reinterpret_cast<const uint4 *>(&rows[i + grp][8 * j]) : make_uint4(0u, 0u, 0u, 0u), x);
      if (turned) {
        turn(x, live ? i0 + i + grp : 0, a.gamma_k);
        if (live) *reinterpret_cast<uint4 *>(&rows[i + grp][8 * j]) = pack8(x);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, live ? limited_abs(x[e]) : 0.f);
    }
    amax = warp_max(amax);
    const float s = fmaxf(scale_for(amax), old), inv = 1.0f / s;
    const bool finite = amax < kBf16Max;  // no value to limit
    const bool raise = r0 > 0 && s > old;  // the rows in front of the run move to the larger scale
    const float ratio = raise ? old / s : 1.f;
    __syncwarp();
    if (lane == 0) *sp = s;
    auto code = [&](uint32_t two) -> uint32_t {  // two bf16 as two codes
      float x = __uint_as_float(two << 16), y = __uint_as_float(two & 0xffff0000u);
      if (!finite) {
        x = limited(x);
        y = limited(y);
      }
      return e4m3x2(x * inv, y * inv);
    };
    if (!is_v) {
      // 4 lanes per row, 16 dims each
      if (raise)
        for (int c = lane; c < r0 * 4; c += 32) {
          uint4 *p = reinterpret_cast<uint4 *>(codes) + c;
          *p = rescale16(*p, ratio, 16);
        }
      for (int c = lane; c < n * 4; c += 32) {
        const uint4 *p = reinterpret_cast<const uint4 *>(&rows[c >> 2][16 * (c & 3)]);
        const uint4 x = p[0], y = p[1];
        reinterpret_cast<uint4 *>(codes)[r0 * 4 + c] =
            make_uint4(code(x.x) | (code(x.y) << 16), code(x.z) | (code(x.w) << 16), code(y.x) | (code(y.y) << 16),
                       code(y.z) | (code(y.w) << 16));
      }
    } else {
      // dims 2 lane, 2 lane + 1; pieces of 16 tokens that hold rows of the run (or rows that move)
      const int first = raise ? 0 : r0 / 16, last = (r0 + n - 1) / 16;
      for (int q = first; q <= last; ++q) {
        uint4 *p0 = reinterpret_cast<uint4 *>(codes + 2 * lane * kBlock) + q, *p1 = p0 + kBlock / 16;
        const int lo = r0 - 16 * q, hi = r0 + n - 16 * q;  // rows of the run in this piece: [lo, hi)
        uint32_t u[4], v[4];
        if (lo <= 0 && hi >= 16) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            uint32_t c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = code(*reinterpret_cast<const uint32_t *>(&rows[i + e - lo][2 * lane]));
            const uint32_t x = __byte_perm(c[0], c[1], 0x5410), y = __byte_perm(c[2], c[3], 0x5410);
            u[i >> 2] = __byte_perm(x, y, 0x6420);
            v[i >> 2] = __byte_perm(x, y, 0x7531);
          }
          *p0 = make_uint4(u[0], u[1], u[2], u[3]);
          *p1 = make_uint4(v[0], v[1], v[2], v[3]);
          continue;
        }
        uint4 x = *p0, y = *p1;
        if (raise && lo > 0) {
          x = rescale16(x, ratio, lo);
          y = rescale16(y, ratio, lo);
        }
        u[0] = x.x; u[1] = x.y; u[2] = x.z; u[3] = x.w;
        v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (i < lo || i >= hi) continue;
          const uint32_t c = code(*reinterpret_cast<const uint32_t *>(&rows[i - lo][2 * lane]));
          const uint32_t keep = ~(0xffu << (8 * (i & 3)));
          u[i >> 2] = (u[i >> 2] & keep) | ((c & 0xffu) << (8 * (i & 3)));
          v[i >> 2] = (v[i >> 2] & keep) | ((c >> 8) << (8 * (i & 3)));
        }
        *p0 = make_uint4(u[0], u[1], u[2], u[3]);
        *p1 = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncwarp();  // the rows may be overwritten by the next run's
  }
}

// ------------------------------------------------------------------ decode step

// The step streams the cache once: 64-token tiles of one (sequence, KV head),
// 4 KiB of K and 4 KiB of V codes and their two scales.  All tiles of the batch
// in the order (sequence, head, block) are cut into equal ranges, one per warp,
// so every warp streams the same number of tiles whatever the lengths are.  A
// warp is its own pipeline: lane 0 copies the tiles of the warp's range
// (cp.async.bulk on an mbarrier per stage) kStages ahead, the warp multiplies
// them on the tensor cores and hands the stage back to itself, with no barrier
// between warps until the end.
//
//   S[64 x 8]   = K[64 x 64] . Q^T       columns: (new token, head of the pair)
//   O^T[64 x 8] += V^T[64 x 64] . P^T    V is stored dim-major, so both A operands
//                                        are rows of 16-byte pieces
// The products are mma.sync m16n8k16 in f16, which holds every e4m3 code
// exactly.  (mma.sync m16n8k32 on the codes themselves runs at 0.4 of that rate
// per element here and needs Q and P in two parts: 60.5 us against 57.4 us for
// 64 sequences of 128-8192 tokens.)  Vector v (2 * new token + head) is column
// 2 v, or 2 (v - 4) + 1: a lane then holds the scores of one vector, of two only
// with 3 or 4 new tokens.
//
// Which tokens and dims the rows and k slots of a fragment stand for is free as
// long as both operands agree: a lane's 16 k slots of four mma steps are 16
// adjacent bytes of a row, so an operand of 16 rows is two 16-byte loads per
// lane, free of bank conflicts without a swizzle.
//
// Scales: a vector's scores are c * (q factor * k scale), the query scaled to
// 2^14 so that f16 keeps all bf16 bits of values down to 2^-28 of its largest.
// The sum of p runs against the reference m (log2 units), moved only when a
// score exceeds m + kSlack (a vote, no shuffles, in all other tiles).  The
// products p * v scale are rounded to f16 against a reference of their own, mo:
// g = v scale * 2^(m - mo) is 2^kTopLog2 where the largest product so far is, and
// up to kMaxGain needs no look at the tile (p * g <= 2^15); above, the tile's
// true maximum decides whether mo moves.  f16 gives p 11 bits (bf16 would give 8)
// down to 2^-22 of the largest product; what is below 2^-33 of it is lost, so a
// tail of 2^17 tokens loses at most 2^-16 of the largest product.  The room above
// (2^7 of it) is shared by scores that rise and v scales that grow: less of it
// means more looks, and in a prompt more passes over the output.
//
// Ends: a segment (sequence, head) inside one warp's range is written by that
// warp.  Others leave partial states in shared memory, merged by the CTA after
// its last tile; what crosses CTAs goes through the workspace, and the last
// CTA to arrive merges it in CTA order (the result does not depend on who is
// last).  At most two segments of a CTA are open, so the workspace has two
// slots and one counter per CTA whatever the batch.
template <int kT>
constexpr int step_warps() { return kT <= 2 ? 12 : 10; }
template <int kT>
constexpr int step_stages() { return 2; }
constexpr int kMaxSeqs = 1024;   // sequences per launch (lengths and sums in shared memory)
constexpr int kSegmentCost = 2;  // tiles that the start and end of a segment weigh as
constexpr int kMaxCtas = 256;
constexpr uint64_t kDrainNs = 2000000000ull;
constexpr float kSlack = 5.0f;          // log2 units that a score may exceed m by
constexpr float kTopLog2 = 8.0f;        // the largest product when mo moves
constexpr float kMaxGainLog2 = 10.0f;   // g without a look at the tile's maximum
constexpr float kMaxGain = 1024.0f;
static_assert(kSlack + kMaxGainLog2 <= 15.0f && kTopLog2 <= kMaxGainLog2, "products of a weight stay in f16's range");
constexpr float kMinGainLog2 = 60.0f;   // below 2^-60 the products' sum may underflow
constexpr float kUnset = -1.0e30f;

// log2 of a scale; exact for powers of two
__device__ __forceinline__ float log2_scale(float s) {
  const uint32_t u = __float_as_uint(s);
  const float e = static_cast<float>(static_cast<int>(u >> 23) - 127);
  return (u & 0x007fffffu) == 0 ? e : e + __log2f(__uint_as_float((u & 0x007fffffu) | 0x3f800000u));
}

template <int kT>
struct __align__(128) StepShared {
  static constexpr int kWarps = step_warps<kT>(), kStages = step_stages<kT>();
  static constexpr int kSets = (kT + 1) / 2;  // vectors of a lane
  static constexpr int kVecs = 4 * kSets;     // vectors: 2 * new token + head of the pair
  struct State {  // output in units of 2^mo, and (m, l, mo, -), of every vector
    float o[kVecs][kDim];
    float4 ref[kVecs];
  };
  uint8_t codes[kWarps][kStages][2 * kTile];
  union {
    uint16_t q[kVecs][kDim];         // f16, scaled
    uint16_t out[kVecs][kDim];       // bf16, on the way to memory
  } row[kWarps];
  State head[kWarps];                // a segment that began before the warp's range
  float factor[kWarps][kVecs];
  uint64_t full[kWarps][kStages];
  int tile[kWarps][kStages];         // block * 8 + head, -1: no such block
  int open[kWarps][2];               // segments of the warp's partial states (head[], codes[][0]), -1: none
  int warp_sum[kWarps];
  int pos[kMaxSeqs + 1];             // where a sequence's work starts
  int past[kMaxSeqs];
  uint8_t fresh[kMaxSeqs];           // new tokens
};

static_assert(sizeof(StepShared<2>) + 128 <= 232448 && sizeof(StepShared<kMaxStepTokens>) + 128 <= 232448,
              "shared memory of a CTA");
static_assert(2 * step_warps<2>() <= 32 && 2 * step_warps<kMaxStepTokens>() <= 32, "open states fit a bit mask");

struct StepArgs {
  const uint16_t *qkv;
  int64_t row_stride;
  int rows;
  const int32_t *row_start;
  int tokens;
  const int32_t *chunk_lens;
  const uint16_t *gamma_q, *gamma_k;
  float eps;
  const uint16_t *cos, *sin;
  int rope_rows;
  const int32_t *past_lens, *block_tables;
  int max_blocks;
  uint8_t *k_pool, *v_pool;
  float *k_scale, *v_scale;
  int num_blocks, batch;
  float scale_log2;
  int mode;
  uint16_t *out;
  int32_t *counters;  // [kMaxCtas][kMaxStepTokens], zero between calls
  float *slots;       // [kMaxCtas][2] states
  int32_t *err;
  uint64_t wait_ns;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void mma_f16(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Four codes as two f16 pairs.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// The product of a 64 x 64 operand of codes with 64 x 8 columns: r[i] are this
// lane's 16 bytes of rows g and g + 8 of m-tile i.  The four m-tiles take turns,
// so four independent products are in flight.
__device__ __forceinline__ void mma_codes(float c[4][4], const uint4 r[4][2], const uint32_t b[4][2]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = k == 0 ? r[i][0].x : k == 1 ? r[i][0].y : k == 2 ? r[i][0].z : r[i][0].w;
      const uint32_t w = k == 0 ? r[i][1].x : k == 1 ? r[i][1].y : k == 2 ? r[i][1].z : r[i][1].w;
      uint32_t a0, a1, a2, a3;
      codes_f16(u, a0, a2);
      codes_f16(w, a1, a3);
      mma_f16(c[i], a0, a1, a2, a3, b[k][0], b[k][1]);
    }
  }
}

// The (m, l, mo) of a partial state, written one by one: as one store it took four registers in a row for the whole
// loop (prompt: 28 bytes of spills more, 289 us against 281 for 64 x 128 tokens).
__device__ __forceinline__ void write_ref(float4 *ref, float m, float l, float mo) {
  ref->x = m;
  ref->y = l;
  ref->z = mo;
}

// Sum of partial states of one new token: 16 lanes per head of the pair, 4 dims
// each.  States come in groups of 16, lane i of the 16 holding state i's (m, l,
// mo).  Outputs keep the reference of their products, which the last division
// takes with it: in units of 2^m a sum of values near fp32's largest leaves it.
struct StateSum {
  float m = kUnset, l = 0.f, mo = kUnset;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float c = 0.f;  // factor of this lane's state of the group
  __device__ __forceinline__ void group(float4 ref) {
    float top = ref.x, top_o = ref.z;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      top_o = fmaxf(top_o, __shfl_xor_sync(0xffffffffu, top_o, off));
    }
    const float n = fmaxf(m, top), no = fmaxf(mo, top_o), again = ex2(mo - no);
    float s = ref.y * ex2(ref.x - n);
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    l = fmaf(l, ex2(m - n), s);
    m = n;
    mo = no;
    c = ex2(ref.z - no);
    o.x *= again;
    o.y *= again;
    o.z *= again;
    o.w *= again;
  }
  __device__ __forceinline__ void add(int i, float4 x, int lane) {
    const float f = __shfl_sync(0xffffffffu, c, (lane & 16) + i);
    o.x = fmaf(x.x, f, o.x);
    o.y = fmaf(x.y, f, o.y);
    o.z = fmaf(x.z, f, o.z);
    o.w = fmaf(x.w, f, o.w);
  }
  // the two context rows
  __device__ __forceinline__ void write(uint16_t *out, int lane) const {
    const float inv = ex2(mo - m) / l;
    *reinterpret_cast<uint2 *>(out + (lane >> 4) * kDim + 4 * (lane & 15)) =
        make_uint2(pack_bf16x2_rn(o.x * inv, o.y * inv), pack_bf16x2_rn(o.z * inv, o.w * inv));
  }
};

__device__ __forceinline__ void fence_gpu() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

template <int kT>
__global__ void __launch_bounds__(step_warps<kT>() * 32, 1) kv8_step_kernel(const StepArgs a) {
  using Shared = StepShared<kT>;
  using State = typename Shared::State;
  constexpr int kWarps = Shared::kWarps, kStages = Shared::kStages, kStepThreads = kWarps * 32;
  extern __shared__ uint8_t smem_raw[];
  Shared &sh = *reinterpret_cast<Shared *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;    // mma: row (column) group, thread in group
  const int j = lane & 7, grp = lane >> 3;  // head vectors: 8 values, vector of four
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&sh.full[warp][s]), 1);
    mbar_fence_init();
    sh.open[warp][0] = sh.open[warp][1] = -1;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // the row of a sequence's first new token
  auto row_of = [&](int sb) -> int64_t {
    return a.row_start ? __ldcg(a.row_start + sb) : static_cast<int64_t>(sb) * a.tokens;
  };
  // The batch's work as a line: sequence b has the positions [pos[b], pos[b + 1]),
  // its 8 heads' segments in turn, a segment its tiles and kSegmentCost more
  // positions that stand for the cost of its start and end.
  int running = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kStepThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int n = 0;
    if (b < a.batch) {
      const int past = __ldcg(a.past_lens + b), ntok = a.chunk_lens ? __ldcg(a.chunk_lens + b) : a.tokens;
      const int64_t first = row_of(b);
      const bool fits = ntok == 0 || (past >= 0 && ntok > 0 && ntok <= a.tokens &&
                                      static_cast<int64_t>(past) + ntok <= static_cast<int64_t>(a.max_blocks) * kBlock &&
                                      first >= 0 && first + ntok <= a.rows);
      if (!fits && blockIdx.x == 0) atomicOr(a.err, B2_DEV_BAD_LENGTH);
      if (fits && ntok > 0) n = ((past + ntok + kBlock - 1) / kBlock + kSegmentCost) * kHkv;
      sh.past[b] = past;
      sh.fresh[b] = static_cast<uint8_t>(n > 0 ? ntok : 0);
    }
    int incl = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
    }
    if (lane == 31) sh.warp_sum[warp] = incl;
    __syncthreads();
    int before = running;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int v = sh.warp_sum[w];
      if (w < warp) before += v;
      running += v;
    }
    if (b < a.batch) sh.pos[b + 1] = before + incl;
    if (threadIdx.x == 0 && b0 == 0) sh.pos[0] = 0;
    __syncthreads();
  }
  const int weight = running;
  // as many CTAs as there are positions for their warps
  const int ctas = min(static_cast<int>(gridDim.x), (weight + kWarps - 1) / kWarps);
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  // this warp's positions [w0, w1): lane 0 and 1 divide
  const int unit = static_cast<int>(blockIdx.x) * kWarps + warp;
  const int edge = static_cast<int>(static_cast<uint64_t>(unit + (lane & 1)) * static_cast<uint32_t>(weight) /
                                    static_cast<uint32_t>(ctas * kWarps));
  const int w0 = __shfl_sync(0xffffffffu, edge, 0), w1 = __shfl_sync(0xffffffffu, edge, 1);

  // sequence, head, block of position w; a block past the segment's last stands for its cost
  auto place = [&](int w, int &sb, int &head, int &block, int &blocks) {
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh.pos[mid] <= w) lo = mid; else hi = mid;
    }
    const int start = sh.pos[lo], per = (sh.pos[lo + 1] - start) / kHkv;
    sb = lo;
    head = (w - start) / per;
    block = w - start - head * per;
    blocks = per - kSegmentCost;
  };
  constexpr int kNoTile = -2;  // a position without a tile; -1: a tile without a valid block
  int b = 0, h = 0, blk = 0, nblk = 0;
  auto look = [&](int w, bool keep) {
    int sb = 0, head = 0, block = 0, blocks = 0, id = kNoTile;
    if (w < w1) {
      place(w, sb, head, block, blocks);
      if (block < blocks) {
        const int e = __ldcg(a.block_tables + static_cast<int64_t>(sb) * a.max_blocks + block);
        id = e < 0 || e >= a.num_blocks ? -1 : e * kHkv + head;
      }
    }
    if (keep) {  // the warp starts at lane 0's position
      b = __shfl_sync(0xffffffffu, sb, 0);
      h = __shfl_sync(0xffffffffu, head, 0);
      blk = __shfl_sync(0xffffffffu, block, 0);
      nblk = __shfl_sync(0xffffffffu, blocks, 0);
    }
    return id;
  };

  const uint64_t policy = evict_first_policy();
  // tiles of 32 positions: one per lane, those not issued yet in `left`
  int base = w0, entry = look(w0 + lane, true), entry_next = kNoTile, issued = 0;
  uint32_t left = __ballot_sync(0xffffffffu, entry != kNoTile);
  // the segment after (b, h): its sequence
  auto following = [&](int sb) {
    do ++sb; while (sb < a.batch && sh.pos[sb + 1] == sh.pos[sb]);
    return sb;
  };
  if (blk >= nblk && ++h == kHkv) {  // starts behind a segment's last tile
    h = 0;
    b = following(b);
  }
  // head vectors of the segment's new tokens, bf16: q (lanes 0-15), k (16-23) and
  // v (24-31), and those of the next segment on their way
  uint4 fresh[kT], fresh_next[kT];
  auto fetch = [&](int sb, int head) {
    const int vec = grp < 2 ? 2 * head + grp : (grp == 2 ? kHq + head : kHq + kHkv + head);
    const uint16_t *p = a.qkv + row_of(sb) * a.row_stride + vec * kDim + j * 8;
#pragma unroll
    for (int i = 0; i < kT; ++i)
      if (i < sh.fresh[sb]) fresh_next[i] = __ldcg(reinterpret_cast<const uint4 *>(p + i * a.row_stride));
  };
  if (blk >= nblk) blk = 0;
  if (b < a.batch && w0 < w1) {
    nblk = (sh.pos[b + 1] - sh.pos[b]) / kHkv - kSegmentCost;
    fetch(b, h);  // ahead of the tiles, behind which it would queue
  }
  bool looked = false;  // entry_next is the next 32 positions
  float2 scales[kStages];  // k and v scale of the tiles in flight, the next one's first
  auto issue = [&]() {
    while (left == 0) {
      if (base + 32 >= w1) return;
      base += 32;
      entry = looked ? entry_next : look(base + lane, false);
      looked = false;
      left = __ballot_sync(0xffffffffu, entry != kNoTile);
    }
    const int id = __shfl_sync(0xffffffffu, entry, __ffs(left) - 1);
    left &= left - 1;
    if (lane == 0) {
      const int s = issued % kStages;
      const int from = id < 0 ? 0 : id;  // a tile that exists; its result is flagged as bad
      if (id < 0) atomicOr(a.err, B2_DEV_BAD_BLOCK);
      sh.tile[warp][s] = id;
      const uint32_t bar = smem_u32(&sh.full[warp][s]), dst = smem_u32(sh.codes[warp][s]);
      mbar_expect_tx(bar, 2 * kTile);
      bulk_load(dst, a.k_pool + static_cast<int64_t>(from) * kTile, kTile, bar, policy);
      bulk_load(dst + kTile, a.v_pool + static_cast<int64_t>(from) * kTile, kTile, bar, policy);
    }
    // (as 16-byte copies of their own the scales doubled the copies, which one
    // thread issues at about 100 ns each)
    scales[kStages - 1] = make_float2(__ldcg(a.k_scale + max(id, 0)), __ldcg(a.v_scale + max(id, 0)));
    ++issued;
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) scales[i] = scales[i + 1];
    issue();
  }

  // state of the current segment: vector t + 4 u of set u in the lanes of thread t
  constexpr int kSets = Shared::kSets;
  uint32_t bq[4][2];
  float o[4][4], m[kSets], mo[kSets], l[kSets], factor[kSets];
  bool begin = true, from_start = false;  // the next tile is the segment's first in this warp, .. of all
  int past = 0, ntok = 0;
  bool ok = true;
  from_start = blk == 0;
  for (int k = 0; k < issued; ++k) {
    const int s = k % kStages;
    if (begin) {
      // queries of the segment: norm + RoPE, then f16 columns in shared memory
      past = sh.past[b];
      ntok = sh.fresh[b];
#pragma unroll
      for (int i = 0; i < kT; ++i) fresh[i] = fresh_next[i];
      if (sh.pos[b] + (h + 1) * (nblk + kSegmentCost) < w1)  // another segment follows: its rows are here by then
        fetch(h + 1 < kHkv ? b : following(b), (h + 1) % kHkv);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        if (i >= ntok) break;
        float y[8];
        unpack8(fresh[i], y);
        if (a.mode & (B2_NORM_QK | B2_ROPE_QK)) {
          const int pos = past + i;
          const bool turn_ok = pos < a.rope_rows;
          if ((a.mode & B2_ROPE_QK) && !turn_ok && lane == 0) atomicOr(a.err, B2_DEV_BAD_POSITION);
          const bool turn = grp < 3 && (a.mode & B2_ROPE_QK) && turn_ok;
          norm_rope8(y, j, grp < 3 && (a.mode & B2_NORM_QK), turn, grp < 2 ? a.gamma_q : a.gamma_k, a.eps,
                     turn ? a.cos + static_cast<int64_t>(pos) * kDim : nullptr,
                     turn ? a.sin + static_cast<int64_t>(pos) * kDim : nullptr);
          fresh[i] = pack8(y);
        }
        float big = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(y[e]));
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
        if (grp < 2) {
          // the query with its largest value in [2^14, 2^15)
          int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
          e = e < -100 ? -100 : e;
          const float up = __uint_as_float(static_cast<uint32_t>(141 - e) << 23);
          const int v = 2 * i + grp;
          *reinterpret_cast<uint4 *>(&sh.row[warp].q[v][8 * j]) =
              make_uint4(pack_f16x2(y[0] * up, y[1] * up), pack_f16x2(y[2] * up, y[3] * up),
                         pack_f16x2(y[4] * up, y[5] * up), pack_f16x2(y[6] * up, y[7] * up));
          if (j == 0) sh.factor[warp][v] = __uint_as_float(static_cast<uint32_t>(113 + e) << 23) * a.scale_log2;
        }
      }
      __syncwarp();
      // column g holds vector g / 2 (g even) or 4 + g / 2
      const int qv = (g >> 1) + 4 * (g & 1);
      uint4 q0 = make_uint4(0u, 0u, 0u, 0u), q1 = q0;
      if (qv < 2 * ntok) {
        const uint4 *p = reinterpret_cast<const uint4 *>(&sh.row[warp].q[qv][16 * t]);
        q0 = p[0];
        q1 = p[1];
      }
      bq[0][0] = q0.x; bq[0][1] = q0.y; bq[1][0] = q0.z; bq[1][1] = q0.w;
      bq[2][0] = q1.x; bq[2][1] = q1.y; bq[3][0] = q1.z; bq[3][1] = q1.w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll
      for (int u = 0; u < kSets; ++u) {
        factor[u] = 4 * u + t < 2 * ntok ? sh.factor[warp][4 * u + t] : 0.f;
        m[u] = mo[u] = kUnset;
        l[u] = 0.f;
      }
      begin = false;
    }
    if (!mbar_wait(smem_u32(&sh.full[warp][s]), (k / kStages) & 1, a.wait_ns)) ok = false;
    if (__any_sync(0xffffffffu, !ok)) {
      ok = false;
      if (lane == 0) atomicOr(a.err, B2_DEV_TIMEOUT);
      break;
    }
    uint8_t *kc = sh.codes[warp][s], *vc = kc + kTile;
    float ks = scales[0].x, vs = scales[0].y;
    const int key0 = blk * kBlock;

    if ((a.mode & B2_STORE_KV) && key0 + kBlock > past && sh.tile[warp][s] >= 0) {
      // append: rows [lo, hi) of this tile are new tokens first ..
      const int lo = max(past - key0, 0), hi = min(past + ntok - key0, kBlock), first = key0 + lo - past;
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        if (i < first || i >= first + hi - lo) continue;
        float y[8];
        unpack8(fresh[i], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, limited_abs(y[e]));
      }
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
      const float want = scale_for(big);
      const float ks_new = fmaxf(__shfl_sync(0xffffffffu, want, 16), lo > 0 ? ks : 0.f);
      const float vs_new = fmaxf(__shfl_sync(0xffffffffu, want, 24), lo > 0 ? vs : 0.f);
      const int64_t id = sh.tile[warp][s];
      uint8_t *kg = a.k_pool + id * kTile, *vg = a.v_pool + id * kTile;
      if (lo > 0 && ks_new > ks) {
        const float ratio = ks / ks_new;
        for (int c = lane; c < lo * 4; c += 32) {
          uint4 *p = reinterpret_cast<uint4 *>(kc) + c;
          const uint4 w = rescale16(*p, ratio, 16);
          *p = w;
          reinterpret_cast<uint4 *>(kg)[c] = w;
        }
      }
      if (lo > 0 && vs_new > vs) {
        const float ratio = vs / vs_new;
        const int per = (lo + 15) / 16;
        for (int c = lane; c < kDim * per; c += 32) {
          const int d = c / per, q = d * (kBlock / 16) + (c - d * per);
          uint4 *p = reinterpret_cast<uint4 *>(vc) + q;
          const uint4 w = rescale16(*p, ratio, lo - 16 * (c - d * per));
          *p = w;
          reinterpret_cast<uint4 *>(vg)[q] = w;
        }
      }
      __syncwarp();
      if (grp >= 2) {
        const float inv = 1.0f / (grp == 2 ? ks_new : vs_new);
#pragma unroll
        for (int i = 0; i < kT; ++i) {
          if (i < first || i >= first + hi - lo) continue;
          const int at = lo + i - first;
          float y[8];
          unpack8(fresh[i], y);
          uint32_t c[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = e4m3x2(limited(y[2 * e]) * inv, limited(y[2 * e + 1]) * inv);
          if (grp == 2) {
            const uint2 w = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
            *reinterpret_cast<uint2 *>(kc + at * kDim + 8 * j) = w;
            *reinterpret_cast<uint2 *>(kg + at * kDim + 8 * j) = w;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint8_t w = static_cast<uint8_t>(c[e >> 1] >> (8 * (e & 1)));
              vc[(8 * j + e) * kBlock + at] = w;
              vg[(8 * j + e) * kBlock + at] = w;
            }
          }
        }
        if (j == 0) (grp == 2 ? a.k_scale : a.v_scale)[id] = grp == 2 ? ks_new : vs_new;
      }
      ks = ks_new;
      vs = vs_new;
      // these stores come before the stage's next copy
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }

    // S = K . Q^T: row g of m-tile i is token 16 (g / 2) + 4 i + g % 2, row g + 8
    // the one two behind it (8 lanes of a load read two adjacent rows)
    const int tok0 = 16 * (g >> 1) + (g & 1), tok1 = tok0 + 2;
    float c[4][4];
    uint4 r[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i][0] = *reinterpret_cast<const uint4 *>(kc + (tok0 + 4 * i) * kDim + 16 * t);
      r[i][1] = *reinterpret_cast<const uint4 *>(kc + (tok1 + 4 * i) * kDim + 16 * t);
#pragma unroll
      for (int e = 0; e < 4; ++e) c[i][e] = 0.f;
    }
    mma_codes(c, r, bq);
    const bool tail = key0 + kBlock > past + 1;  // some token does not see the whole tile
    const uint32_t vbits = __float_as_uint(vs);  // mantissa and exponent of the v scale apart
    const float vmant = __uint_as_float((vbits & 0x007fffffu) | 0x3f800000u);
    const float vexp = static_cast<float>(static_cast<int>(vbits >> 23) - 127);
    float p[kSets][4][2];  // p * g of rows g and g + 8
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      const bool used = 4 * u + t < 2 * ntok;
      // scores in log2 units of rows g (x) and g + 8 (y)
      const float w = factor[u] * ks;
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = c[i][u] * w;
        y[i] = c[i][2 + u] * w;
      }
      if (tail) {
        const int lim = past + ((4 * u + t) >> 1) + 1 - key0;  // the vector's token sees rows < lim
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (tok0 + 4 * i >= lim) x[i] = -INFINITY;
          if (tok1 + 4 * i >= lim) y[i] = -INFINITY;
        }
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], y[0]), fmaxf(x[1], y[1])), fmaxf(fmaxf(x[2], y[2]), fmaxf(x[3], y[3])));
      if (__any_sync(0xffffffffu, used && top > m[u] + kSlack)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float n = fmaxf(m[u], top);
        l[u] *= ex2(m[u] - n);
        m[u] = n;
      }
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = ex2(x[i] - m[u]);
        y[i] = ex2(y[i] - m[u]);
        sum += x[i] + y[i];
      }
      l[u] += sum;
      float gain = vmant * ex2(m[u] - mo[u] + vexp);
      if (__any_sync(0xffffffffu, used && gain > kMaxGain)) {
        float big = fmaxf(fmaxf(fmaxf(x[0], y[0]), fmaxf(x[1], y[1])), fmaxf(fmaxf(x[2], y[2]), fmaxf(x[3], y[3])));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
        // the largest product so far at 2^kTopLog2 (p as small as 2^-126 may have one: g stays in fp32 all the same);
        // where every p is 0, g may have left it
        const float n = big > 0.f ? fmaxf(mo[u], m[u] + vexp + fmaxf(__log2f(big * vmant) - kTopLog2, -120.f)) : mo[u];
        const float again = ex2(mo[u] - n);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i][u] *= again;
          o[i][2 + u] *= again;
        }
        mo[u] = n;
        gain = big > 0.f ? vmant * ex2(m[u] - n + vexp) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[u][i][0] = x[i] * gain;
        p[u][i][1] = y[i] * gain;
      }
    }
    uint32_t bp[4][2];  // P^T: tokens 16 t + 4 i + {0, 1} and + {2, 3} of column g
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        bp[i][e] = transpose8x8(pack_f16x2(p[0][i][e], kSets > 1 ? p[kSets - 1][i][e] : 0.f));
    if (tail && ntok > 1) {
      // a new token's NaN (no other code is not finite) must not meet p = 0 of the tokens in front of it: it goes
      // to the outputs of those that see it, and the product takes a 0
      bool moved = false, look = !(a.mode & B2_STORE_KV);  // (their v is in registers, or in the cache alone)
      if (!look) {
        uint32_t nans = 0;  // top bit of a bf16 that is a NaN
#pragma unroll
        for (int i = 1; i < kT; ++i) {
          if (i >= ntok) break;
          for (const uint32_t w : {fresh[i].x, fresh[i].y, fresh[i].z, fresh[i].w}) nans |= (w & 0x7fff7fffu) + 0x007f007fu;
        }
        look = __any_sync(0xffffffffu, grp == 3 && (nans & 0x80008000u));
      }
      for (int at = max(past + 1 - key0, 0); look && at < min(past + ntok - key0, kBlock); ++at) {
        uint8_t *c0 = vc + lane * kBlock + at, *c1 = c0 + 32 * kBlock;  // dims lane, 32 + lane
        const uint32_t n0 = __ballot_sync(0xffffffffu, (*c0 & 0x7f) == 0x7f);
        const uint32_t n1 = __ballot_sync(0xffffffffu, (*c1 & 0x7f) == 0x7f);
        if ((n0 | n1) == 0) continue;
        moved = true;
        if (n0 >> lane & 1) *c0 = 0;
        if (n1 >> lane & 1) *c1 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // dim 16 i + 8 (e / 2) + g, vector 4 (e % 2) + t
            const uint32_t bits = i < 2 ? n0 : n1;
            if ((bits >> (16 * (i & 1) + 8 * (e >> 1) + g) & 1) && (4 * (e & 1) + t) >> 1 >= key0 + at - past)
              o[i][e] = __int_as_float(0x7fffffff);
          }
      }
      if (moved) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next copy
        __syncwarp();
      }
    }
    // O^T += V^T . P^T: rows g and g + 8 of m-tile i are dims 16 i + g and 16 i + 8 + g
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *row = vc + (16 * i + g) * kBlock + 16 * t;
      r[i][0] = *reinterpret_cast<const uint4 *>(row);
      r[i][1] = *reinterpret_cast<const uint4 *>(row + 8 * kBlock);
    }
    if (tail) {
      // codes of rows past the sequence must not meet p = 0
      const int n = past + ntok - key0 - 16 * t;
      auto mask = [&](int i) { return n >= 4 * i + 4 ? ~0u : (n <= 4 * i ? 0u : (1u << (8 * (n - 4 * i))) - 1u); };
      const uint4 keep = make_uint4(mask(0), mask(1), mask(2), mask(3));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          r[i][e].x &= keep.x;
          r[i][e].y &= keep.y;
          r[i][e].z &= keep.z;
          r[i][e].w &= keep.w;
        }
    }
    mma_codes(o, r, bp);
    __syncwarp();
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) scales[i] = scales[i + 1];
    issue();  // the stage is read: its next tile
    if (!looked && base + 32 < w1) {
      entry_next = look(base + 32 + lane, false);
      looked = true;
    }

    const bool last = blk + 1 == nblk;  // of the segment
    if (last || k + 1 == issued) {
#pragma unroll
      for (int u = 0; u < kSets; ++u)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[u] += __shfl_xor_sync(0xffffffffu, l[u], off);
      if (last && from_start) {
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
          const int v = 4 * u + t;
          if (v >= 2 * ntok) continue;
          const float f = ex2(mo[u] - m[u]) / l[u];  // dims 16 i + g, 16 i + 8 + g
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sh.row[warp].out[v][16 * i + g] = static_cast<uint16_t>(bf16_bits(o[i][u] * f));
            sh.row[warp].out[v][16 * i + 8 + g] = static_cast<uint16_t>(bf16_bits(o[i][2 + u] * f));
          }
        }
        __syncwarp();
        for (int c8 = lane; c8 < 2 * ntok * 8; c8 += 32) {
          const int v = c8 >> 3;
          *reinterpret_cast<uint4 *>(a.out + ((row_of(b) + (v >> 1)) * kHq + 2 * h + (v & 1)) * kDim +
                                     8 * (c8 & 7)) = *reinterpret_cast<const uint4 *>(&sh.row[warp].out[v][8 * (c8 & 7)]);
        }
        __syncwarp();
      } else {
        // open: began before this range (head), or goes on behind it (in the ring, idle by then)
        const int which = from_start ? 1 : 0;
        State *st = which ? reinterpret_cast<State *>(sh.codes[warp][0]) : &sh.head[warp];
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
          const int v = 4 * u + t;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            st->o[v][16 * i + g] = o[i][u];
            st->o[v][16 * i + 8 + g] = o[i][2 + u];
          }
          if (g == 0) write_ref(&st->ref[v], m[u], l[u], mo[u]);
        }
        if (lane == 0) sh.open[warp][which] = b * kHkv + h;
      }
      if (last) {
        begin = from_start = true;
        blk = -1;
        if (++h == kHkv) {
          h = 0;
          b = following(b);
          if (b < a.batch) nblk = (sh.pos[b + 1] - sh.pos[b]) / kHkv - kSegmentCost;
        }
      }
    }
    ++blk;
  }
  if (!ok) {
    // leave no copy in flight behind
    for (int s = 0; s < kStages && s < issued; ++s) {
      const int k = s + kStages * ((issued - 1 - s) / kStages);
      if (!mbar_wait(smem_u32(&sh.full[warp][s]), (k / kStages) & 1, kDrainNs) && lane == 0) atomicOr(a.err, B2_DEV_TIMEOUT);
    }
  }
  __syncthreads();

  // The CTA's partial states in tile order, one per lane; those of one segment
  // are merged by one warp per new token.
  const int mine = lane < 2 * kWarps ? sh.open[lane >> 1][lane & 1] : -1;
  const uint32_t same = __match_any_sync(0xffffffffu, mine);
  uint32_t todo = __ballot_sync(0xffffffffu, mine >= 0 && (same & ((1u << lane) - 1u)) == 0);
  for (int task = 0; todo; todo &= todo - 1) {
    const int seg = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
    const uint32_t members = __shfl_sync(0xffffffffu, same, __ffs(todo) - 1);
    const int sb = seg / kHkv, hh = seg - sb * kHkv, stok = sh.fresh[sb];
    for (int v = 0; v < stok; ++v, ++task) {
      if (task % kWarps != warp) continue;
      const int per = (sh.pos[sb + 1] - sh.pos[sb]) / kHkv;
      // the CTAs of the segment's first and last tile: the last ones that start
      // at or before them (CTA c starts at position c * weight / ctas)
      const int at = sh.pos[sb] + hh * per + ((lane & 1) ? per - kSegmentCost : 1);
      const int cta_of = static_cast<int>((static_cast<uint64_t>(at) * static_cast<uint32_t>(ctas) - 1) /
                                          static_cast<uint32_t>(weight));
      const int cf = __shfl_sync(0xffffffffu, cta_of, 0), cl = __shfl_sync(0xffffffffu, cta_of, 1);
      const int vec = 2 * v + (lane >> 4), d = 4 * (lane & 15);
      StateSum sum;
#pragma unroll
      for (int e0 = 0; e0 < 2 * kWarps; e0 += 16) {
        if ((members >> e0 & 0xffffu) == 0) continue;
        auto state = [&](int e) -> const State * {
          return (e & 1) ? reinterpret_cast<const State *>(sh.codes[e >> 1][0]) : &sh.head[e >> 1];
        };
        const int e = e0 + (lane & 15);
        float4 ref = make_float4(kUnset, 0.f, kUnset, 0.f);
        if (e < 2 * kWarps && (members >> e & 1)) ref = state(e)->ref[vec];
        sum.group(ref);
        for (uint32_t rest = members >> e0 & 0xffffu; rest; rest &= rest - 1) {
          const int i = __ffs(rest) - 1;
          sum.add(i, *reinterpret_cast<const float4 *>(&state(e0 + i)->o[vec][d]), lane);
        }
      }
      uint16_t *dst = a.out + ((row_of(sb) + v) * kHq + 2 * hh) * kDim;
      if (cf == cl) {
        sum.write(dst, lane);
        continue;
      }
      // the segment's first CTA leaves its state in slot 1, the others in slot 0
      State *slots = reinterpret_cast<State *>(a.slots);
      const int cta = static_cast<int>(blockIdx.x);
      State *slot = slots + 2 * cta + (cta == cf ? 1 : 0);
      *reinterpret_cast<float4 *>(&slot->o[vec][d]) = sum.o;
      if (d == 0) write_ref(&slot->ref[vec], sum.m, sum.l, sum.mo);
      __syncwarp();
      int32_t *counter = a.counters + cf * kMaxStepTokens + v;
      int arrived = 0;
      if (lane == 0) {
        fence_gpu();
        arrived = atomicAdd(counter, 1) == cl - cf;
        if (arrived) fence_gpu();
      }
      if (!__shfl_sync(0xffffffffu, arrived, 0)) continue;
      __syncwarp();
      StateSum whole;
      for (int c0 = cf; c0 <= cl; c0 += 16) {
        // sixteen states' loads in flight together
        const int c = c0 + (lane & 15);
        float4 ref = make_float4(kUnset, 0.f, kUnset, 0.f);
        if (c <= cl) ref = __ldcg(&(slots + 2 * c + (c == cf ? 1 : 0))->ref[vec]);
        float4 x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int q = min(c0 + e, cl);
          x[e] = __ldcg(reinterpret_cast<const float4 *>(&(slots + 2 * q + (q == cf ? 1 : 0))->o[vec][d]));
        }
        whole.group(ref);
#pragma unroll
        for (int e = 0; e < 16; ++e) whole.add(e, x[e], lane);  // factor 0 past the last state
      }
      whole.write(dst, lane);
      if (lane == 0) *counter = 0;
    }
  }
}

template <int kT>
bool step_ready() {
  static std::atomic<bool> done[128];  // the attribute is per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return false;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kv8_step_kernel<kT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(StepShared<kT>)) + 128) != cudaSuccess)
      return false;
    done[dev] = true;
  }
  return true;
}

int sm_count() {
  static std::atomic<int> count[128];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return 148;
  if (!count[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    count[dev] = n;
  }
  return count[dev];
}

constexpr int64_t kCounterBytes = kMaxCtas * kMaxStepTokens * 4;
constexpr int64_t kStepBytes =
    kCounterBytes + 2 * kMaxCtas * static_cast<int64_t>(sizeof(StepShared<kMaxStepTokens>::State));

template <int kT>
int launch_step(StepArgs a, cudaStream_t st) {
  if (!step_ready<kT>()) return fail(B2_ERR_CUDA, "cannot set the step kernel's shared memory size");
  // launches of at most kMaxSeqs sequences whose tiles an int32 counts
  const int64_t most = ((int64_t(1) << 28) - 1) / (a.max_blocks + kSegmentCost);
  const int per = static_cast<int>(most < kMaxSeqs ? (most < 1 ? 1 : most) : kMaxSeqs);
  const int batch = a.batch;
  constexpr int kWarps = step_warps<kT>();
  for (int b0 = 0; b0 < batch; b0 += per) {
    a.batch = batch - b0 < per ? batch - b0 : per;
    const int64_t tiles = static_cast<int64_t>(a.batch) * a.max_blocks * kHkv;
    int64_t ctas = (tiles + kWarps - 1) / kWarps;
    if (ctas > sm_count()) ctas = sm_count();
    if (ctas > kMaxCtas) ctas = kMaxCtas;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = sizeof(StepShared<kT>) + 128;
    cfg.stream = st;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const int rc = launched(cudaLaunchKernelEx(&cfg, kv8_step_kernel<kT>, a), "kv8_step_kernel");
    if (rc) return rc;
    if (a.row_start) {
      a.row_start += a.batch;
    } else {
      const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens;
      a.qkv += rows * a.row_stride;
      a.out += rows * kHq * kDim;
      a.rows -= static_cast<int>(rows);
    }
    a.past_lens += a.batch;
    if (a.chunk_lens) a.chunk_lens += a.batch;
    a.block_tables += static_cast<int64_t>(a.batch) * a.max_blocks;
  }
  return b2_clear_error();
}

// ------------------------------------------------------------------ prompt chunks

// Attention of a chunk of new tokens per sequence, appended before, on the
// tcgen05 tensor cores.  One CTA per (64-token query tile, KV head, sequence)
// holds 128 query rows (64 tokens x the pair of heads) and walks the
// sequence's 64-token blocks:
//   S_j[128 x 64]  = Q[128 x 64] . K_j^T     into tensor memory, f16 operands
//   O[128 x 64]   += P_j[128 x 64] . V_j     P_j as the A operand from tensor memory
// Warp roles: warps 0-3 the online softmax (thread = query row = TMEM lane),
// warp 4 issues the products, warps 5 and 6 bring K and V: each copies its 4 KiB
// tiles of codes ahead (cp.async.bulk), converts them to f16 (exact) and stores
// them as 128-byte-swizzled operands.  V is stored dim-major, so both B operands
// are K-major.  S and P are double-buffered, as the operands' rings are, so
// conversion, products and softmax of different blocks overlap.
//
// 64 sequences, 128 new tokens over 128-8064 cached: 286 us with the append (14),
// against 84 us of products at the matrix rate and 50 us of bytes.  Profiled:
// exponentials 50 % of their pipe, matrix pipe 24 %, DRAM 13 %, issue 49 %: what
// bounds it is the chain of a block (S, 64 scores to registers, maximum, 64
// exponentials, P to tensor memory), about 1.1 us, of which two CTAs per SM run
// side by side.  Three CTAs per SM with half the stages (344 us against 331 then),
// four with single buffers (441) and more registers for the softmax warps
// (setmaxnreg, 340) were slower, and so were two sets of softmax warps on
// alternate blocks, with 80 registers and P in the place of S (328 against 286:
// each waits for its products).  The rest is a CTA's start, a row of dependent
// loads under load, about 5 us: reading a tile's lengths a second time after the
// search for it cost 21 us in all, starting K and V only behind the query 5.
//
// A launch of more CTAs than start at once runs its query tiles longest first;
// as they come: 376 us against 324 at that step.
//
// The scales never touch the operands: a row's scores are S * (q factor * k
// scale), and P is p * g with g = v scale * 2^(m - mo), the references m (of
// the sum) and mo (of the output, moved when the block's largest product
// exceeds it by kMaxGain) as in the decode step; only moving mo needs the
// output rescaled in tensor memory.
//
// Few long sequences leave most SMs idle: then the blocks of a tile are split
// over several CTAs, whose states go through the workspace to kv8_merge_kernel,
// launched behind as a programmatic dependent.
constexpr int kPfStages = 3;                 // f16 operand stages of K and of V
constexpr int kPfRaw = 4;                    // stages of codes
constexpr int kPfThreads = 7 * 32;
constexpr int kPfTmemCols = 256;             // S at columns 0 and 64, O at 128, P at 192 and 224
constexpr int kPfOperand = kBlock * kDim * 2;
constexpr int kPfMaxSplit = 32;
constexpr int kPfSortMax = 128;              // sequences whose tiles are started longest first
constexpr int kPfMaxParts = 320;             // CTAs of a split launch
constexpr uint32_t kPfIdesc = (1u << 4) | (8u << 17) | (8u << 24);  // f32 <- f16, M 128, N 64, both K-major

struct __align__(16) PrefillTail {
  uint64_t raw[2][kPfRaw];       // codes landed (K, V)
  uint64_t full[2][kPfStages];   // operand written by its converter warp
  uint64_t empty[2][kPfStages];  // operand read by its product (commit)
  uint64_t sbar[2];              // S_j computed, and every product issued before it done (commit)
  uint64_t sfree[2];             // S_j read by the softmax threads
  uint64_t pready[2];            // P_j written by the softmax threads
  uint64_t pvbar;                // P_j . V_j accumulated (commit per block)
  uint64_t obar;                 // every product done (one commit)
  uint32_t tmem;
  int abort;
  int nan_any, nan_key[kDim];    // first key with a NaN of V that not all rows of the tile see, per dim
};
constexpr int kPfSmem = 1024 + 2 * kPfOperand + 2 * kPfStages * kPfOperand + 2 * kPfRaw * kTile + (int)sizeof(PrefillTail);

struct PrefillState {  // a query tile's rows over one CTA's blocks: output in units of 2^mo, and (m, l, mo, -)
  float o[2 * kBlock][kDim];
  float4 ref[2 * kBlock];
};

struct PrefillArgs {
  const uint16_t *q;
  int64_t q_stride;
  int rows;
  const int32_t *row_start, *past_lens, *chunk_lens;
  int tokens;
  const int32_t *block_tables;
  int max_blocks;
  const uint8_t *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  int num_blocks;
  float scale_log2;
  uint16_t *out;
  int batch, tiles;      // tiles: of the longest chunk
  bool sorted;           // jobs by their blocks, not by sequence
  int nsplit;
  PrefillState *parts;   // [query tile][nsplit]
  int32_t *err;
  uint64_t wait_ns;
};

// Query tile t0 of sequence b: its first row, tokens, blocks, and the blocks of
// one of its parts.  False: nothing there (or lengths that do not fit, flagged).
struct PrefillTile {
  int past, rows, blocks, per, parts;
  int64_t row;
};
__device__ __forceinline__ bool prefill_fits(const PrefillArgs &a, int past, int chunk, int64_t row) {
  return past >= 0 && chunk >= 0 && chunk <= a.tokens &&
         static_cast<int64_t>(past) + chunk <= static_cast<int64_t>(a.max_blocks) * kBlock &&
         row >= 0 && row + chunk <= a.rows;
}
__device__ __forceinline__ void prefill_blocks(const PrefillArgs &a, int past, int chunk, int64_t row, int t0,
                                               PrefillTile &t) {
  t.past = past;
  t.row = row + t0;
  t.rows = min(kBlock, chunk - t0);
  t.blocks = (past + t0 + t.rows - 1) / kBlock + 1;
  t.per = (t.blocks + a.nsplit - 1) / a.nsplit;
  t.parts = (t.blocks + t.per - 1) / t.per;
}
__device__ __forceinline__ bool prefill_tile(const PrefillArgs &a, int b, int t0, bool report, PrefillTile &t) {
  const int chunk = a.chunk_lens ? a.chunk_lens[b] : a.tokens;
  const int past = a.past_lens[b];
  const int64_t row = a.row_start ? static_cast<int64_t>(a.row_start[b]) : static_cast<int64_t>(b) * a.tokens;
  if (chunk == 0) return false;
  if (!prefill_fits(a, past, chunk, row)) {
    if (report) atomicOr(a.err, B2_DEV_BAD_LENGTH);
    return false;
  }
  if (t0 >= chunk) return false;
  prefill_blocks(a, past, chunk, row, t0, t);
  return true;
}

struct PrefillJob {
  int b, tile, past, chunk;  // b < 0: none
  int64_t row;
};
// One warp: the job-th query tile of the batch, the one with the most blocks
// first (equal ones by sequence).
// Tile t of a sequence with p cached blocks (the last one included) has p + t + 1
// blocks, its last tile those of the whole length, so the tiles with more than
// x blocks are counted without a loop over them, and x is found by search.
template <int kGroups>  // of 32 sequences
__device__ void prefill_job(const PrefillArgs &a, int job, PrefillJob &chosen) {
  const int lane = threadIdx.x & 31;
  int past[kGroups], chunk[kGroups];
  int64_t row[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int b = i * 32 + lane;
    const bool there = b < a.batch;
    past[i] = there ? a.past_lens[b] : 0;
    chunk[i] = there ? (a.chunk_lens ? a.chunk_lens[b] : a.tokens) : 0;
    row[i] = !a.row_start ? static_cast<int64_t>(b) * a.tokens : there ? a.row_start[b] : 0;
  }
  int held[kGroups], full[kGroups], all[kGroups];  // blocks cached, tiles before the last, blocks of the last
  int top = 0, n = 0;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    held[i] = full[i] = all[i] = 0;
    if (chunk[i] == 0) continue;
    if (!prefill_fits(a, past[i], chunk[i], row[i])) {
      if (job == 0) atomicOr(a.err, B2_DEV_BAD_LENGTH);
      continue;
    }
    held[i] = (past[i] + kBlock - 1) / kBlock;
    full[i] = (chunk[i] + kBlock - 1) / kBlock - 1;
    all[i] = (past[i] + chunk[i] - 1) / kBlock + 1;
    top = max(top, all[i]);
    n += full[i] + 1;
  }
  if (static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(n))) <= job) {
    if (lane == 0) chosen.b = -1;
    return;
  }
  auto above = [&](int i, int x) { return full[i] - min(max(x - held[i], 0), full[i]) + (all[i] > x ? 1 : 0); };
  auto count = [&](int x) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) c += above(i, x);
    return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(c)));
  };
  // the smallest x with at most `job` tiles above it: the job's blocks
  int lo = 0, hi = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(top)));
  while (hi - lo > 1) {  // above lo: more than `job` tiles, above hi: not
    const int d = (hi - lo + 3) >> 2, x1 = lo + d, x2 = min(x1 + d, hi), x3 = min(x2 + d, hi);
    const bool p1 = count(x1) <= job, p2 = count(x2) <= job, p3 = count(x3) <= job;
    lo = p1 ? lo : (p2 ? x1 : (p3 ? x2 : x3));
    hi = p1 ? x1 : (p2 ? x2 : (p3 ? x3 : hi));
  }
  int skip = job - count(hi);  // of the tiles with hi blocks, which one
  const unsigned below = (1u << lane) - 1u;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int mine = above(i, hi - 1) - above(i, hi);  // 0, 1 or 2
    const unsigned one = __ballot_sync(0xffffffffu, mine >= 1), two = __ballot_sync(0xffffffffu, mine == 2);
    const int before = __popc(one & below) + __popc(two & below);
    if (skip >= before && skip < before + mine) {
      // the last tile first, then the one before it
      chosen.b = i * 32 + lane;
      chosen.tile = skip == before && all[i] == hi ? full[i] : hi - 1 - held[i];
      chosen.past = past[i];
      chosen.chunk = chunk[i];
      chosen.row = row[i];
    }
    skip -= __popc(one) + __popc(two);
  }
}

// V's NaN at a key that only later rows of the query tile see (keys [first, end), counted from the V tile's first)
// must not meet p = 0 of the others: the product takes a 0, and the rows that see the key get the NaN at the end.
// One warp, on the codes in shared memory; two of 65 blocks for 64 x 128 tokens, 283 us with it and 279 without.
// (Within the conversion 3 us more, as were a conversion loop of its own for such blocks and a look between two runs of
// the loop; unrolled, its cold instructions cost a call of one tile 0.15 us.)
__device__ __forceinline__ void hide_late_nans(uint8_t *tile, PrefillTail *tail, int key0, int first, int end) {
  const int lane = threadIdx.x & 31;
  const int at = 16 * (lane & 3);  // the lane's first key of the tile
  auto from = [](int k, int i) { return k >= 4 * i + 4 ? 0u : (k <= 4 * i ? 0x80808080u : 0x80808080u << (8 * (k - 4 * i))); };
  auto late = [&](int i) { return from(first - at, i) & ~from(end - at, i); };
  auto nans = [](uint32_t x) { return (x & 0x7f7f7f7fu) + 0x01010101u; };  // top bit of each NaN's byte
  const uint4 *piece = reinterpret_cast<const uint4 *>(tile) + lane;       // 32 i + lane: 16 tokens of dim 8 i + lane / 4
  const uint32_t late0 = late(0), late1 = late(1), late2 = late(2), late3 = late(3);
  uint32_t any = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const uint4 x = piece[32 * i];
    any |= (nans(x.x) & late0) | (nans(x.y) & late1) | (nans(x.z) & late2) | (nans(x.w) & late3);
  }
  if (!__any_sync(0xffffffffu, any != 0)) return;
#pragma unroll 1
  for (int i = 0; i < 32; ++i) {  // word i % 4 of piece i / 4
    uint32_t *word = reinterpret_cast<uint32_t *>(tile) + (32 * (i >> 2) + lane) * 4 + (i & 3);
    const uint32_t z = nans(*word) & late(i & 3);
    if (z == 0) continue;
    atomicMin(&tail->nan_key[8 * (i >> 2) + (lane >> 2)], key0 + at + 4 * (i & 3) + ((__ffs(z) - 1) >> 3));
    tail->nan_any = 1;
    *word &= ~((z >> 7) * 0xffu);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next copy
  __syncwarp();
}

__device__ __forceinline__ float fmax3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

__global__ void __launch_bounds__(kPfThreads, 2) kv8_prefill_kernel(const PrefillArgs a) {
  // grid: job (a query tile, in the order they start), its parts, its heads
  const int h = static_cast<int>(blockIdx.x) % kHkv, part = static_cast<int>(blockIdx.x) / kHkv;
  const int job = part / a.nsplit, split = part - job * a.nsplit;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sq = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = sq + 2 * kPfOperand;                   // K stages, then V stages
  uint8_t *raw = ring + 2 * kPfStages * kPfOperand;      // codes of K, then of V
  PrefillTail *tail = reinterpret_cast<PrefillTail *>(raw + 2 * kPfRaw * kTile);

  if (tid == 4 * 32) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
      for (int s = 0; s < kPfRaw; ++s) mbar_init(smem_u32(&tail->raw[w][s]), 1);
#pragma unroll
      for (int s = 0; s < kPfStages; ++s) {
        mbar_init(smem_u32(&tail->full[w][s]), 32);
        mbar_init(smem_u32(&tail->empty[w][s]), 1);
      }
      mbar_init(smem_u32(&tail->sbar[w]), 1);
      mbar_init(smem_u32(&tail->sfree[w]), 128);
      mbar_init(smem_u32(&tail->pready[w]), 128);
    }
    mbar_init(smem_u32(&tail->pvbar), 1);
    mbar_init(smem_u32(&tail->obar), 1);
    tail->abort = 0;
    mbar_fence_init();
  }
  // the last tiles of a sequence see the most keys: they start first
  int b = job / a.tiles, tile = a.tiles - 1 - (job - b * a.tiles);
  PrefillTile pt;
  if (a.sorted) {
    __shared__ PrefillJob chosen;
    if (warp == 0) {
      if (a.batch <= 32) prefill_job<1>(a, job, chosen);
      else if (a.batch <= 64) prefill_job<2>(a, job, chosen);
      else prefill_job<kPfSortMax / 32>(a, job, chosen);
    }
    __syncthreads();
    b = chosen.b;
    tile = chosen.tile;
    if (b < 0) return;
    prefill_blocks(a, chosen.past, chosen.chunk, chosen.row, tile * kBlock, pt);
  } else {
    __syncthreads();
    if (!prefill_tile(a, b, tile * kBlock, tid == 0, pt)) return;
  }
  if (split >= pt.parts) return;
  const int t0 = tile * kBlock;
  const int past = pt.past, rows_t = pt.rows, last_key = past + t0 + rows_t - 1;
  const int64_t row0 = pt.row;
  // this CTA's blocks [j0, j0 + nblk)
  const int j0 = split * pt.per, nblk = min(pt.per, pt.blocks - j0);

  // The warps of K and V start at once; the others meet when the query is in
  // shared memory and the tensor memory allocated.
  auto meet = [&]() -> uint32_t {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tmem_fence_before();
    asm volatile("bar.sync 1, 160;" ::: "memory");
    tmem_fence_after();
    return tail->tmem;
  };
  if (warp >= 5) {
    // ---------------- K (warp 5) and V (warp 6): codes in, f16 operands out
    const int which = warp - 5;
    const uint8_t *pool = which ? a.v_pool : a.k_pool;
    uint8_t *codes = raw + which * kPfRaw * kTile, *operand = ring + which * kPfStages * kPfOperand;
    const int32_t *table = a.block_tables + static_cast<int64_t>(b) * a.max_blocks + j0;
    const uint64_t policy = evict_first_policy();
    int entry = lane < nblk ? table[lane] : 0, entry_next = 32 + lane < nblk ? table[32 + lane] : 0;
    int issued = 0;
    auto issue = [&]() {
      if (issued >= nblk) return;
      if (issued > 0 && (issued & 31) == 0) {
        entry = entry_next;
        entry_next = issued + 32 + lane < nblk ? table[issued + 32 + lane] : 0;
      }
      int blk = __shfl_sync(0xffffffffu, entry, issued & 31);
      if (blk < 0 || blk >= a.num_blocks) {
        if (lane == 0 && which == 0) atomicOr(a.err, B2_DEV_BAD_BLOCK);
        blk = 0;  // read a valid tile instead; the result is flagged as bad
      }
      const int64_t id = static_cast<int64_t>(blk) * kHkv + h;
      const int s = issued % kPfRaw;
      if (lane == 0) {
        const uint32_t bar = smem_u32(&tail->raw[which][s]);
        mbar_expect_tx(bar, kTile);
        bulk_load(smem_u32(codes + s * kTile), pool + id * kTile, kTile, bar, policy);
      }
      ++issued;
    };
    for (int s = 0; s < kPfRaw; ++s) issue();
    if (which) {
      tail->nan_key[lane] = tail->nan_key[32 + lane] = 0x7fffffff;
      if (lane == 0) tail->nan_any = 0;
      __syncwarp();
    }
    const int whole = which ? (past + t0 + 1) / kBlock - j0 : nblk;  // V's blocks from here on hold keys that not all rows see
    for (int j = 0; j < nblk; ++j) {
      const int s = j % kPfStages, rs = j % kPfRaw;
      bool got = mbar_wait(smem_u32(&tail->raw[which][rs]), (j / kPfRaw) & 1, a.wait_ns);
      if (j >= whole)
        hide_late_nans(codes + rs * kTile, tail, (j0 + j) * kBlock, past + t0 + 1 - (j0 + j) * kBlock,
                       last_key + 1 - (j0 + j) * kBlock);
      uint4 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint4 *>(codes + rs * kTile + (32 * i + lane) * 16);
      __syncwarp();
      issue();
      if (j >= kPfStages) got = got && mbar_wait(smem_u32(&tail->empty[which][s]), ((j / kPfStages) - 1) & 1, a.wait_ns);
      if (__any_sync(0xffffffffu, !got || tail->abort)) {
        if (lane == 0 && !tail->abort) atomicOr(a.err, B2_DEV_TIMEOUT);
        tail->abort = 1;
        break;
      }
      if (j >= whole && (j0 + j) * kBlock + kBlock - 1 > last_key) {
        // tokens past the tile's last key may hold anything (even NaN): p = 0 must not meet them
        const int n = last_key + 1 - (j0 + j) * kBlock - 16 * (lane & 3);
        auto mask = [&](int i) { return n >= 4 * i + 4 ? ~0u : (n <= 4 * i ? 0u : (1u << (8 * (n - 4 * i))) - 1u); };
        const uint4 keep = make_uint4(mask(0), mask(1), mask(2), mask(3));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i].x &= keep.x;
          w[i].y &= keep.y;
          w[i].z &= keep.z;
          w[i].w &= keep.w;
        }
      }
      // piece c = 32 i + lane is 16 codes of row c / 4 (token or dim): two 16-byte pieces of f16
      uint8_t *dst = operand + s * kPfOperand;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = 8 * i + (lane >> 2), c = 2 * (lane & 3);
        uint4 lo, hi;
        codes_f16(w[i].x, lo.x, lo.y);
        codes_f16(w[i].y, lo.z, lo.w);
        codes_f16(w[i].z, hi.x, hi.y);
        codes_f16(w[i].w, hi.z, hi.w);
        *reinterpret_cast<uint4 *>(dst + row * 128 + ((c ^ (row & 7)) << 4)) = lo;
        *reinterpret_cast<uint4 *>(dst + row * 128 + (((c + 1) ^ (row & 7)) << 4)) = hi;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(smem_u32(&tail->full[which][s]));
    }
    // leave no copy in flight behind
    for (int s = 0; s < kPfRaw && s < issued; ++s) {
      const int k = s + kPfRaw * ((issued - 1 - s) / kPfRaw);
      if (!mbar_wait(smem_u32(&tail->raw[which][s]), (k / kPfRaw) & 1, kDrainNs) && lane == 0) atomicOr(a.err, B2_DEV_TIMEOUT);
    }
    if (which) asm volatile("bar.sync 2, 160;" ::: "memory");  // nan_key is complete
  } else if (warp == 4) {
    // ---------------- products: S_0, S_1, then per block P_j . V_j and S_{j+2}
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem)),
                 "n"(kPfTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    const uint32_t tmem = meet();
    if (lane == 0) {
      auto issue_s = [&](int j) -> bool {
        const int s = j % kPfStages;
        if (!mbar_wait(smem_u32(&tail->full[0][s]), (j / kPfStages) & 1, a.wait_ns)) return false;
        if (j >= 2 && !mbar_wait(smem_u32(&tail->sfree[j & 1]), ((j >> 1) - 1) & 1, a.wait_ns)) return false;
        tmem_fence_after();
        const uint32_t kt = smem_u32(ring + s * kPfOperand);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_f16(tmem + 64 * (j & 1), umma_desc(smem_u32(sq) + 32 * ks, 16), umma_desc(kt + 32 * ks, 16), kPfIdesc, ks > 0);
        umma_commit(smem_u32(&tail->sbar[j & 1]));
        umma_commit(smem_u32(&tail->empty[0][s]));
        return true;
      };
      bool ok = issue_s(0) && (nblk < 2 || issue_s(1));
      for (int j = 0; ok && j < nblk; ++j) {
        const int s = j % kPfStages;
        if (!mbar_wait(smem_u32(&tail->pready[j & 1]), (j >> 1) & 1, a.wait_ns) || tail->abort ||
            !mbar_wait(smem_u32(&tail->full[1][s]), (j / kPfStages) & 1, a.wait_ns)) {
          ok = false;
          break;
        }
        tmem_fence_after();
        const uint32_t vt = smem_u32(ring + (kPfStages + s) * kPfOperand);
        const uint32_t pt = tmem + 192 + 32 * (j & 1);  // 16 tokens per step = 8 columns
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_f16_ta(tmem + 128, pt + 8 * ks, umma_desc(vt + 32 * ks, 16), kPfIdesc, (j > 0 || ks > 0) ? 1u : 0u);
        umma_commit(smem_u32(&tail->pvbar));
        umma_commit(smem_u32(&tail->empty[1][s]));
        if (j + 2 < nblk) ok = issue_s(j + 2);
      }
      if (!ok) {
        if (!tail->abort) atomicOr(a.err, B2_DEV_TIMEOUT);
        tail->abort = 1;
      }
      // one commit behind the last product: its phase says that all are done
      umma_commit(smem_u32(&tail->obar));
      if (!mbar_wait(smem_u32(&tail->obar), 0, kDrainNs)) atomicOr(a.err, B2_DEV_TIMEOUT);
    }
  } else {
    // ---------------- softmax: thread = query row = TMEM lane
    const int hl = tid >> 6, t = tid & 63;
    const bool row_ok = t < rows_t;
    const int qpos = past + t0 + t;
    float m = kUnset, mo = kUnset, l = 0.f;
    bool ok = true;
    // decided for the whole warp: the tensor memory accesses are warp-collective
    auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.wait_ns));
    };
    // a warp whose rows are all past the chunk keeps step with the barriers only
    const bool active = __any_sync(0xffffffffu, row_ok);
    // scales of 32 blocks, one per lane; the next 32 on their way
    const int32_t *table = a.block_tables + static_cast<int64_t>(b) * a.max_blocks + j0;
    auto pool_tile = [&](int j) -> int64_t {
      const int blk = j < nblk ? table[j] : 0;
      return static_cast<int64_t>(blk < 0 || blk >= a.num_blocks ? 0 : blk) * kHkv + h;
    };
    int64_t id = pool_tile(lane);
    float2 scale = make_float2(__ldcg(a.k_scale + id), __ldcg(a.v_scale + id)), scale_next = scale;
    // query rows: row r = (head of the pair) * 64 + token, its largest value at 2^14 in f16
    float factor = 0.f;
    {
      const uint4 *src = reinterpret_cast<const uint4 *>(a.q + (row0 + t) * a.q_stride + (2 * h + hl) * kDim);
      uint4 w[8];
      float big = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        w[c] = t < rows_t ? src[c] : make_uint4(0u, 0u, 0u, 0u);
        float y[8];
        unpack8(w[c], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(y[e]));
      }
      int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
      e = e < -100 ? -100 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(141 - e) << 23);
      factor = __uint_as_float(static_cast<uint32_t>(113 + e) << 23) * a.scale_log2;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float y[8];
        unpack8(w[c], y);
        *reinterpret_cast<uint4 *>(sq + tid * 128 + ((c ^ (tid & 7)) << 4)) =
            make_uint4(pack_f16x2(y[0] * up, y[1] * up), pack_f16x2(y[2] * up, y[3] * up),
                       pack_f16x2(y[4] * up, y[5] * up), pack_f16x2(y[6] * up, y[7] * up));
      }
    }
    const uint32_t trow = meet() + (static_cast<uint32_t>(32 * warp) << 16);
    for (int j = 0; j < nblk; ++j) {
      if (!warp_wait(smem_u32(&tail->sbar[j & 1]), (j >> 1) & 1)) {
        ok = false;
        break;
      }
      if (!active) {
        mbar_arrive(smem_u32(&tail->sfree[j & 1]));
        mbar_arrive(smem_u32(&tail->pready[j & 1]));
        continue;
      }
      tmem_fence_after();
      if (j > 0 && (j & 31) == 0) scale = scale_next;
      if ((j & 31) == 8) id = pool_tile((j & ~31) + 32 + lane);
      if ((j & 31) == 16) scale_next = make_float2(__ldcg(a.k_scale + id), __ldcg(a.v_scale + id));
      const float ks = __shfl_sync(0xffffffffu, scale.x, j & 31), vs = __shfl_sync(0xffffffffu, scale.y, j & 31);
      float sc[64];
      tmem_ld64(trow + 64 * (j & 1), sc);
      tmem_fence_before();
      mbar_arrive(smem_u32(&tail->sfree[j & 1]));  // S_j is in registers
      const int key0 = (j0 + j) * kBlock;
      const int lim = row_ok ? qpos - key0 : -1;  // tokens c <= lim are visible
      if (__any_sync(0xffffffffu, lim < kBlock - 1)) {
#pragma unroll
        for (int c = 0; c < 64; ++c) sc[c] = c <= lim ? sc[c] : -INFINITY;
      }
      float bm[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bm[e] = fmaxf(sc[e], sc[e + 4]);
#pragma unroll
      for (int c = 8; c < 64; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) bm[e] = fmax3(bm[e], sc[c + e], sc[c + 4 + e]);
      const float w = fmaxf(factor * ks, 1.2e-38f);  // not 0, which would make NaN of a masked score
      const float top = fmaxf(fmax3(bm[0], bm[1], bm[2]), bm[3]) * w;
      if (top > m + kSlack) {
        l *= ex2(m - top);
        m = top;
      }
      const float lv = log2_scale(vs);
      float again = 1.f;
      if (m - mo + lv > kMaxGainLog2) {
        // the largest product so far at 2^kTopLog2
        const float n = fmaxf(mo, top + lv - kTopLog2);
        again = ex2(mo - n);
        mo = n;
      }
      if (__any_sync(0xffffffffu, again != 1.f && j > 0)) {
        if (!warp_wait(smem_u32(&tail->pvbar), (j - 1) & 1)) {
          ok = false;
          break;
        }
        tmem_fence_after();
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t r[16];
          tmem_ld16_nowait(trow + 128 + c, r);
          tmem_wait_ld();
          float o16[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o16[e] = __uint_as_float(r[e]) * again;
          tmem_st16(trow + 128 + c, o16);
        }
        tmem_wait_st();
      }
      const float off = lv - mo;  // p * g = 2^(score - m) * 2^(m - mo) * scale, in one exponent
      float ps[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) ps[e] = 0.f;
      uint32_t pk[32];  // P_j of this row as f16 pairs
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        float x0, x1;
        ffma2(x0, x1, sc[c], sc[c + 1], w, w, off, off);
        x0 = ex2(x0);
        x1 = ex2(x1);
        const int e = c & 7;
        fadd2(ps[e], ps[e + 1], ps[e], ps[e + 1], x0, x1);
        pk[c >> 1] = pack_f16x2(x0, x1);
      }
      float sum = ((ps[0] + ps[1]) + (ps[2] + ps[3])) + ((ps[4] + ps[5]) + (ps[6] + ps[7]));
      const float low = mo - lv - m;  // -log2 of the gain
      if (__any_sync(0xffffffffu, low > kMinGainLog2)) {
        // a scale so far below the others' that its products underflow: the sum on its own
        if (low > kMinGainLog2) {
          sum = 0.f;
#pragma unroll
          for (int c = 0; c < 64; ++c) sum += ex2(fmaf(sc[c], w, -m));
          l += sum;
        } else {
          l = fmaf(sum, ex2(low), l);
        }
      } else {
        l = fmaf(sum, ex2(low), l);
      }
      // into buffer j % 2: P_{j-2} . V_{j-2}, which read it, was issued before S_j, so it is done
      tmem_st32(trow + 192 + 32 * (j & 1), pk);
      tmem_wait_st();
      tmem_fence_before();
      mbar_arrive(smem_u32(&tail->pready[j & 1]));
    }
    asm volatile("bar.sync 2, 160;" ::: "memory");  // the V warp's nan_key
    if (!ok) {
      if (!tail->abort) atomicOr(a.err, B2_DEV_TIMEOUT);
      tail->abort = 1;
    } else if (warp_wait(smem_u32(&tail->obar), 0)) {
      tmem_fence_after();
      const bool stop = __any_sync(0xffffffffu, tail->abort);
      PrefillState *st = pt.parts > 1 ? a.parts + ((static_cast<int64_t>(b) * a.tiles + tile) * kHkv + h) * a.nsplit + split
                                      : nullptr;
      if (st && !stop) write_ref(&st->ref[tid], m, l, mo);
      const float inv = ex2(mo - m) / l;
      float o[64];
      tmem_ld64(trow + 128, o);
      if (stop) {
      } else if (st) {
        float4 *dst = reinterpret_cast<float4 *>(st->o[tid]);
#pragma unroll
        for (int c = 0; c < 64; c += 4) dst[c >> 2] = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
      } else if (row_ok) {
        uint4 *dst = reinterpret_cast<uint4 *>(a.out + ((row0 + t) * kHq + 2 * h + hl) * kDim);
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
          float o8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o8[e] = o[c + e] * inv;
          dst[c >> 3] = pack8(o8);
        }
      }
      if (tail->nan_any && !stop) {
        // over what was written: a loop of few instructions (as part of the output it cost every call 0.4 us)
#pragma unroll 1
        for (int c = 0; c < 64; ++c) {
          if (tail->nan_key[c] > qpos) continue;
          if (st) st->o[tid][c] = __int_as_float(0x7fffffff);
          else if (row_ok) a.out[((row0 + t) * kHq + 2 * h + hl) * kDim + c] = 0x7fff;
        }
      }
    } else {
      atomicOr(a.err, B2_DEV_TIMEOUT);
      tail->abort = 1;
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (warp == 4) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tail->tmem), "n"(kPfTmemCols));
  }
}

// The parts of a split tile's rows: 16 threads per row, 4 dims each; grid
// (tile and head, 8 groups of 16 rows, sequence).
__global__ void __launch_bounds__(256) kv8_merge_kernel(const PrefillArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tile = static_cast<int>(blockIdx.x) / kHkv, h = static_cast<int>(blockIdx.x) % kHkv, b = blockIdx.z;
  PrefillTile pt;
  if (!prefill_tile(a, b, tile * kBlock, false, pt) || pt.parts == 1) return;
  const int r = static_cast<int>(blockIdx.y) * 16 + (static_cast<int>(threadIdx.x) >> 4), d = 4 * (threadIdx.x & 15);
  const int hl = r >> 6, t = r & 63;
  if (t >= pt.rows) return;
  const PrefillState *st = a.parts + (static_cast<int64_t>(b) * gridDim.x + blockIdx.x) * a.nsplit;
  float m = kUnset, l = 0.f, mo = kUnset;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < pt.parts; p0 += 8) {
    float4 ref[8], x[8];
    float n = m, no = mo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const PrefillState *q = st + min(p0 + e, pt.parts - 1);
      ref[e] = __ldcg(&q->ref[r]);
      x[e] = __ldcg(reinterpret_cast<const float4 *>(&q->o[r][d]));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (p0 + e >= pt.parts) ref[e] = make_float4(kUnset, 0.f, kUnset, 0.f);
      n = fmaxf(n, ref[e].x);
      no = fmaxf(no, ref[e].z);
    }
    l *= ex2(m - n);
    const float again = ex2(mo - no);
    m = n;
    mo = no;
    o.x *= again;
    o.y *= again;
    o.z *= again;
    o.w *= again;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = p0 + e < pt.parts ? ex2(ref[e].z - no) : 0.f;
      l = fmaf(ref[e].y, ex2(ref[e].x - n), l);
      o.x = fmaf(x[e].x, f, o.x);
      o.y = fmaf(x[e].y, f, o.y);
      o.z = fmaf(x[e].z, f, o.z);
      o.w = fmaf(x[e].w, f, o.w);
    }
  }
  const float inv = ex2(mo - m) / l;
  *reinterpret_cast<uint2 *>(a.out + ((pt.row + t) * kHq + 2 * h + hl) * kDim + d) =
      make_uint2(pack_bf16x2_rn(o.x * inv, o.y * inv), pack_bf16x2_rn(o.z * inv, o.w * inv));
}

// the step's counters and states, then the prompt's states
constexpr int64_t kWorkspaceBytes = kStepBytes + kPfMaxParts * static_cast<int64_t>(sizeof(PrefillState));

bool prefill_ready() {
  static std::atomic<bool> done[128];  // the attribute is per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return false;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kv8_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPfSmem) != cudaSuccess)
      return false;
    done[dev] = true;
  }
  return true;
}

int launch_prefill(PrefillArgs a, int batch, int max_blocks, cudaStream_t st) {
  if (!prefill_ready()) return fail(B2_ERR_CUDA, "cannot set the prefill kernel's shared memory size");
  // (no chunk is longer than its table; longer ones are refused by their first tile)
  const int64_t longest = a.tokens < static_cast<int64_t>(max_blocks) * kBlock ? a.tokens : static_cast<int64_t>(max_blocks) * kBlock;
  const int tiles = a.tiles = static_cast<int>((longest + kBlock - 1) / kBlock);
  const int64_t ctas = static_cast<int64_t>(tiles) * kHkv * batch;
  // Split the keys when the tiles leave SMs without a CTA: about two CTAs per
  // SM, of at least 4 blocks each (as far as the table's width tells).
  a.nsplit = 1;
  const int want = 2 * sm_count() < kPfMaxParts ? 2 * sm_count() : kPfMaxParts;
  if (ctas * 2 <= want) {
    int64_t n = want / ctas;
    if (n > kPfMaxSplit) n = kPfMaxSplit;
    if (n > (max_blocks + 3) / 4) n = (max_blocks + 3) / 4;
    if (n > 1) a.nsplit = static_cast<int>(n);
  }
  cudaLaunchConfig_t cfg = {};
  // More CTAs than start at once: the longest tiles first, so that the launch
  // does not end on one that came late.
  a.sorted = a.batch > 1 && a.batch <= kPfSortMax && ctas > 2 * sm_count();
  if (ctas * a.nsplit > 0x7fffffff) return fail(B2_ERR_ARG, "batch * tokens too large");
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * a.nsplit));
  cfg.blockDim = dim3(kPfThreads);
  cfg.dynamicSmemBytes = kPfSmem;
  cfg.stream = st;
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  int rc = launched(cudaLaunchKernelEx(&cfg, kv8_prefill_kernel, a), "kv8_prefill_kernel");
  if (rc || a.nsplit == 1) return rc;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * kHkv), 8, static_cast<unsigned>(batch));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return launched(cudaLaunchKernelEx(&cfg, kv8_merge_kernel, a), "kv8_merge_kernel");
}

// ------------------------------------------------------------------ host checks

int check_cache(const void *k_pool, const void *v_pool, const void *k_scale, const void *v_scale, int32_t num_blocks) {
  if (!k_pool || !v_pool || !k_scale || !v_scale) return fail(B2_ERR_ARG, "null cache pointer");
  if (!aligned16(k_pool) || !aligned16(v_pool) || !aligned16(k_scale) || !aligned16(v_scale))
    return fail(B2_ERR_ARG, "pools and scales must be 16-byte aligned");
  if (num_blocks <= 0 || num_blocks > kMaxPoolBlocks) return fail(B2_ERR_ARG, "num_blocks must be in [1, 2^22)");
  return B2_OK;
}

int check_rows(const void *qkv, int64_t row_stride, int32_t mode, const void *gamma_q, const void *gamma_k,
               const void *cos, const void *sin, int32_t rope_rows) {
  if (mode & ~(B2_NORM_QK | B2_ROPE_QK | B2_STORE_KV)) return fail(B2_ERR_ARG, "unknown mode bits");
  if (row_stride < kQkvWidth || row_stride % 8 != 0)
    return fail(B2_ERR_ARG, "row_stride must be >= 2048 and a multiple of 8");
  if (!qkv || !aligned16(qkv)) return fail(B2_ERR_ARG, "qkv must be 16-byte aligned and not null");
  if ((mode & B2_NORM_QK) && (!gamma_q || !gamma_k || !aligned16(gamma_q) || !aligned16(gamma_k)))
    return fail(B2_ERR_ARG, "B2_NORM_QK needs 16-byte aligned gamma_q and gamma_k");
  if ((mode & B2_ROPE_QK) && (!cos || !sin || rope_rows <= 0 || !aligned16(cos) || !aligned16(sin)))
    return fail(B2_ERR_ARG, "B2_ROPE_QK needs 16-byte aligned cos/sin tables with rope_rows > 0");
  return B2_OK;
}

int check_tables(const void *tables, int32_t max_blocks, const void *past_lens) {
  if (!tables || !past_lens) return fail(B2_ERR_ARG, "block_tables and past_lens are required");
  if (max_blocks <= 0 || max_blocks > kMaxTableWidth) return fail(B2_ERR_ARG, "max_blocks_per_seq must be in [1, 2^25)");
  return B2_OK;
}

template <int kWindow>
int launch_append(const AppendArgs &a, cudaStream_t st) {
  static std::atomic<bool> done[128];  // the attribute is per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return fail(B2_ERR_CUDA, "no current device");
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kv8_append_kernel<kWindow>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(AppendShared))) != cudaSuccess)
      return fail(B2_ERR_CUDA, "cannot set the append kernel's shared memory size");
    done[dev] = true;
  }
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + kWindow - 1) / kWindow);
  kv8_append_kernel<kWindow><<<dim3(grid, 2 * kHkv / kAppendWarps), kAppendThreads, sizeof(AppendShared), st>>>(a);
  return launched(cudaSuccess, "kv8_append_kernel");
}

}  // namespace

// ------------------------------------------------------------------ C ABI

extern "C" int64_t b2_kv8_workspace_bytes(void) { return kWorkspaceBytes; }

extern "C" int b2_kv8_append(const uint16_t *qkv, int64_t row_stride, int32_t rows, const int32_t *slots,
                             const int32_t *positions, const int32_t *past_lens, const int32_t *chunk_lens,
                             int32_t tokens, const int32_t *block_tables, int32_t max_blocks_per_seq,
                             const uint16_t *gamma_q, const uint16_t *gamma_k, float eps, const uint16_t *rope_cos,
                             const uint16_t *rope_sin, int32_t rope_rows, uint8_t *k_pool, uint8_t *v_pool,
                             float *k_scale, float *v_scale, int32_t num_blocks, uint16_t *q_out, int32_t mode,
                             int32_t *dev_err, void *stream) {
  if (rows < 0 || tokens < 0) return fail(B2_ERR_ARG, "rows and tokens must be >= 0");
  if (rows == 0) return b2_clear_error();
  int rc = check_rows(qkv, row_stride, mode, gamma_q, gamma_k, rope_cos, rope_sin, rope_rows);
  if (rc) return rc;
  if (!dev_err) return fail(B2_ERR_ARG, "dev_err is required");
  if (!(mode & B2_STORE_KV) && !q_out) return fail(B2_ERR_ARG, "nothing to write: neither B2_STORE_KV nor q_out");
  if (q_out && !aligned16(q_out)) return fail(B2_ERR_ARG, "q_out must be 16-byte aligned");
  if (mode & B2_STORE_KV) {
    rc = check_cache(k_pool, v_pool, k_scale, v_scale, num_blocks);
    if (rc) return rc;
  }
  if (slots) {
    if (num_blocks <= 0 || num_blocks > kMaxPoolBlocks) return fail(B2_ERR_ARG, "num_blocks must be in [1, 2^22)");
    if ((mode & B2_ROPE_QK) && !positions) return fail(B2_ERR_ARG, "B2_ROPE_QK with slots needs positions");
  } else {
    rc = check_tables(block_tables, max_blocks_per_seq, past_lens);
    if (rc) return rc;
    if (tokens <= 0 || rows % tokens) return fail(B2_ERR_ARG, "without slots, rows must be a multiple of tokens");
  }
  AppendArgs a{qkv, row_stride, rows, slots, positions, past_lens, chunk_lens, tokens, block_tables,
               max_blocks_per_seq, gamma_q, gamma_k, eps, rope_cos, rope_sin, rope_rows, k_pool, v_pool,
               k_scale, v_scale, num_blocks, q_out, mode, dev_err};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool short_runs = slots ? rows <= 1024 : tokens <= 16;
  return short_runs ? launch_append<8>(a, st) : launch_append<kMaxWindow>(a, st);
}

extern "C" int b2_kv8_decode_step(const uint16_t *qkv, int64_t row_stride, int32_t rows, const int32_t *row_start,
                                  int32_t tokens, const int32_t *chunk_lens,
                                  const uint16_t *gamma_q, const uint16_t *gamma_k, float eps,
                                  const uint16_t *rope_cos, const uint16_t *rope_sin, int32_t rope_rows,
                                  const int32_t *past_lens, const int32_t *block_tables, int32_t max_blocks_per_seq,
                                  uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale,
                                  int32_t num_blocks, int32_t batch, float scale, int32_t mode, uint16_t *out,
                                  void *workspace, int64_t workspace_bytes, int32_t *dev_err, void *stream) {
  if (batch < 0 || rows < 0) return fail(B2_ERR_ARG, "batch and rows must be >= 0");
  if (tokens < 1 || tokens > kMaxStepTokens) return fail(B2_ERR_ARG, "tokens must be in [1, 4]");
  if (batch == 0) return b2_clear_error();
  if (!row_start && static_cast<int64_t>(batch) * tokens > rows)
    return fail(B2_ERR_ARG, "without row_start, rows must be >= batch * tokens");
  int rc = check_rows(qkv, row_stride, mode, gamma_q, gamma_k, rope_cos, rope_sin, rope_rows);
  if (!rc) rc = check_tables(block_tables, max_blocks_per_seq, past_lens);
  if (!rc) rc = check_cache(k_pool, v_pool, k_scale, v_scale, num_blocks);
  if (rc) return rc;
  if (!out || !dev_err || !aligned16(out)) return fail(B2_ERR_ARG, "out (16-byte aligned) and dev_err are required");
  if (!workspace || !aligned16(workspace) || workspace_bytes < kWorkspaceBytes)
    return fail(B2_ERR_ARG, "workspace must be 16-byte aligned and hold b2_kv8_workspace_bytes()");
  if (!(scale > 0.f)) return fail(B2_ERR_ARG, "scale must be positive");
  StepArgs a{qkv, row_stride, rows, row_start, tokens, chunk_lens, gamma_q, gamma_k, eps, rope_cos, rope_sin, rope_rows,
             past_lens, block_tables, max_blocks_per_seq, k_pool, v_pool, k_scale, v_scale, num_blocks, batch,
             scale * 1.4426950408889634f, mode, out, static_cast<int32_t *>(workspace),
             reinterpret_cast<float *>(static_cast<char *>(workspace) + kCounterBytes), dev_err, b2_wait_limit_ns()};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return tokens <= 2 ? launch_step<2>(a, st) : launch_step<kMaxStepTokens>(a, st);
}

extern "C" int b2_kv8_prefill_attn(const uint16_t *q, int64_t q_stride, int32_t rows, const int32_t *row_start,
                                   const int32_t *past_lens, const int32_t *chunk_lens, int32_t tokens,
                                   const int32_t *block_tables, int32_t max_blocks_per_seq, const uint8_t *k_pool,
                                   const uint8_t *v_pool, const float *k_scale, const float *v_scale,
                                   int32_t num_blocks, int32_t batch, float scale, uint16_t *out, void *workspace,
                                   int64_t workspace_bytes, int32_t *dev_err, void *stream) {
  if (batch < 0 || tokens < 0 || rows < 0) return fail(B2_ERR_ARG, "batch, tokens and rows must be >= 0");
  if (batch == 0 || tokens == 0 || rows == 0) return b2_clear_error();
  if (batch > 65535) return fail(B2_ERR_ARG, "batch must be <= 65535");
  int rc = check_tables(block_tables, max_blocks_per_seq, past_lens);
  if (!rc) rc = check_cache(k_pool, v_pool, k_scale, v_scale, num_blocks);
  if (rc) return rc;
  if (!q || !out || !dev_err) return fail(B2_ERR_ARG, "q, out and dev_err are required");
  if (!aligned16(q) || !aligned16(out)) return fail(B2_ERR_ARG, "q and out must be 16-byte aligned");
  if (q_stride < kHq * kDim || q_stride % 8) return fail(B2_ERR_ARG, "q_stride must be >= 1024 and a multiple of 8");
  if (!row_start && static_cast<int64_t>(batch) * tokens > rows)
    return fail(B2_ERR_ARG, "without row_start, rows must be >= batch * tokens");
  if (!workspace || !aligned16(workspace) || workspace_bytes < kWorkspaceBytes)
    return fail(B2_ERR_ARG, "workspace must be 16-byte aligned and hold b2_kv8_workspace_bytes()");
  if (!(scale > 0.f)) return fail(B2_ERR_ARG, "scale must be positive");
  PrefillArgs a{q, q_stride, rows, row_start, past_lens, chunk_lens, tokens, block_tables, max_blocks_per_seq,
                k_pool, v_pool, k_scale, v_scale, num_blocks, scale * 1.4426950408889634f, out, batch, 0, false, 1,
                reinterpret_cast<PrefillState *>(static_cast<char *>(workspace) + kStepBytes), dev_err,
                b2_wait_limit_ns()};
  return launch_prefill(a, batch, max_blocks_per_seq, static_cast<cudaStream_t>(stream));
}
