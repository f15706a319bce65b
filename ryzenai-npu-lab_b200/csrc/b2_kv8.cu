// The 8-bit paged KV cache (include/b2_kv8.h): e4m3 codes with a power-of-two
// scale for each block of 64 tokens and KV head.
//
//   kv8_append_kernel  q/k norm + RoPE and the quantised append of new tokens
//   kv8_step_kernel    a whole decode step: append and split attention
//   kv8_attn_kernel    causal attention of a prompt chunk over the cache

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

constexpr int kWindow = 8;                          // rows whose runs start in one CTA
constexpr int kSeen = 1 + kWindow + kBlock;         // the row before, the window, and a run's rows behind it
constexpr int kNoSlot = -1;

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
  if (chunk > a.tokens) {
    flag |= B2_DEV_BAD_LENGTH;
    return kNoSlot;
  }
  if (t >= chunk) return kNoSlot;
  const int64_t pos = static_cast<int64_t>(a.past_lens[b]) + t;
  if (pos < 0 || pos >= static_cast<int64_t>(a.max_blocks) * kBlock) {
    flag |= B2_DEV_BAD_LENGTH;
    return kNoSlot;
  }
  position = static_cast<int>(pos);
  if (!(a.mode & B2_STORE_KV)) return 0;
  const int blk = a.block_tables[static_cast<int64_t>(b) * a.max_blocks + pos / kBlock];
  if (blk < 0 || blk >= a.num_blocks) {
    flag |= B2_DEV_BAD_BLOCK;
    return kNoSlot;
  }
  return blk * kBlock + static_cast<int>(pos % kBlock);
}

// One CTA per window of rows, warp = KV head.  A run is a sequence of adjacent
// rows that go to adjacent slots of one block; the warp whose window holds
// the run's first row quantises the whole run for its head, so a block's scale
// is found and its codes are written by one warp alone, with no atomics.
// 8 lanes own one 64-wide head vector, 8 values each (four rows per pass).
__global__ void __launch_bounds__(256) kv8_append_kernel(const AppendArgs a) {
  __shared__ int slot[kSeen], place[kSeen];  // entry i: row row0 - 1 + i
  const int row0 = blockIdx.x * kWindow;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane & 7, grp = lane >> 3;
  for (int i = threadIdx.x; i < kSeen; i += 256) {
    const int r = row0 - 1 + i;
    int position = 0, flag = 0;
    slot[i] = r >= 0 && r < a.rows ? row_place(a, r, position, flag) : kNoSlot;
    place[i] = position;
    if (i >= 1 && i <= kWindow) {
      if (slot[i] >= 0 && (a.mode & B2_ROPE_QK) && (position < 0 || position >= a.rope_rows)) flag |= B2_DEV_BAD_POSITION;
      if (flag) atomicOr(a.err, flag);
    }
  }
  __syncthreads();

  // head vector `vec` of row r as this lane's 8 values, normalised and rotated
  auto load = [&](int r, int i, int vec, bool norm, const uint16_t *gamma, bool rope, float x[8]) {
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (r >= 0) w = *reinterpret_cast<const uint4 *>(a.qkv + static_cast<int64_t>(r) * a.row_stride + vec * kDim + j * 8);
    unpack8(w, x);
    const int pos = place[i];
    const bool turn = rope && pos >= 0 && pos < a.rope_rows;
    if (norm || rope)
      norm_rope8(x, j, norm, turn, gamma, a.eps, turn ? a.cos + static_cast<int64_t>(pos) * kDim : nullptr,
                 turn ? a.sin + static_cast<int64_t>(pos) * kDim : nullptr);
  };
  const bool norm = (a.mode & B2_NORM_QK) != 0, rope = (a.mode & B2_ROPE_QK) != 0;

  if (a.q_out) {
    // warp w: the 16 query heads of row row0 + w
    const int i = 1 + warp, r = row0 + warp;
    if (r < a.rows && slot[i] >= 0) {
      for (int p = 0; p < kHq / 4; ++p) {
        const int vec = 4 * p + grp;
        float x[8];
        load(r, i, vec, norm, a.gamma_q, rope, x);
        *reinterpret_cast<uint4 *>(a.q_out + (static_cast<int64_t>(r) * kHq + vec) * kDim + j * 8) = pack8(x);
      }
    }
  }
  if (!(a.mode & B2_STORE_KV)) return;

  const int h = warp;
  for (int i0 = 1; i0 <= kWindow; ++i0) {
    const int s0 = slot[i0];
    if (s0 < 0) continue;
    const int blk = s0 / kBlock, r0 = s0 % kBlock;
    const int prev = slot[i0 - 1];
    if (prev >= 0 && prev + 1 == s0 && r0 != 0) continue;  // inside a run
    int n = 1;
    while (r0 + n < kBlock && slot[i0 + n] == s0 + n) ++n;
    const int row = row0 - 1 + i0;
    const int64_t tile = (static_cast<int64_t>(blk) * kHkv + h) * kTile;
    const int64_t si = static_cast<int64_t>(blk) * kHkv + h;
    for (int which = 0; which < 2; ++which) {
      const bool is_v = which == 1;
      const int vec = kHq + (is_v ? kHkv : 0) + h;
      float amax = 0.f;
      for (int i = 0; i < n; i += 4) {
        const bool live = i + grp < n;
        float x[8];
        load(live ? row + i + grp : -1, live ? i0 + i + grp : 0, vec, norm && !is_v, a.gamma_k, rope && !is_v, x);
        if (live) {
#pragma unroll
          for (int e = 0; e < 8; ++e) amax = fmaxf(amax, limited_abs(x[e]));
        }
      }
      float *sp = (is_v ? a.v_scale : a.k_scale) + si;
      uint8_t *codes = (is_v ? a.v_pool : a.k_pool) + tile;
      const float old = r0 > 0 ? *sp : 0.f;
      const float s = fmaxf(scale_for(warp_max(amax)), old);
      if (r0 > 0 && s > old) {
        // the rows in front of the run move to the larger scale: K rows are
        // whole 16-byte pieces, V's are the first r0 bytes of every dim
        const float ratio = old / s;
        if (!is_v) {
          for (int c = lane; c < r0 * 4; c += 32) {
            uint4 *p = reinterpret_cast<uint4 *>(codes) + c;
            *p = rescale16(*p, ratio, 16);
          }
        } else {
          const int per = (r0 + 15) / 16;
          for (int c = lane; c < kDim * per; c += 32) {
            const int d = c / per, q = c - d * per;
            uint4 *p = reinterpret_cast<uint4 *>(codes + d * kBlock) + q;
            *p = rescale16(*p, ratio, r0 - 16 * q);
          }
        }
      }
      __syncwarp();
      if (lane == 0) *sp = s;
      const float inv = 1.0f / s;
      for (int i = 0; i < n; i += 4) {
        const bool live = i + grp < n;
        float x[8];
        load(live ? row + i + grp : -1, live ? i0 + i + grp : 0, vec, norm && !is_v, a.gamma_k, rope && !is_v, x);
        if (!live) continue;
        uint32_t c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = e4m3x2(limited(x[2 * e]) * inv, limited(x[2 * e + 1]) * inv);
        const int at = r0 + i + grp;
        if (!is_v) {
          *reinterpret_cast<uint2 *>(codes + at * kDim + j * 8) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) codes[(8 * j + e) * kBlock + at] = static_cast<uint8_t>(c[e >> 1] >> (8 * (e & 1)));
        }
      }
    }
  }
}

// ------------------------------------------------------------------ attention

struct AttnArgs {
  const uint16_t *q;
  int64_t q_stride;
  int rows;
  const int32_t *row_start, *past_lens, *chunk_lens;
  int tokens;
  const int32_t *block_tables;
  int max_blocks;
  const uint8_t *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  int num_blocks, batch;
  float scale_log2;
  uint16_t *out;
  int32_t *err;
};

// One CTA per (new token, KV head): its 4 warps take the 64-token blocks in
// turn, each with its own running maximum and sum (log2 units), and are merged
// at the end.  Lane l scores tokens l and l + 32 and sums dims l and l + 32.
__global__ void __launch_bounds__(128) kv8_attn_kernel(const AttnArgs a) {
  __shared__ float qs[2][kDim];
  __shared__ float ps[4][2][kBlock];
  __shared__ float red[4][2][2 + kDim];
  const int b = blockIdx.x / a.tokens, t = blockIdx.x - b * a.tokens, h = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = a.chunk_lens ? a.chunk_lens[b] : a.tokens;
  if (t >= chunk) return;
  const int past = a.past_lens[b];
  const int64_t row = (a.row_start ? static_cast<int64_t>(a.row_start[b]) : static_cast<int64_t>(b) * a.tokens) + t;
  if (past < 0 || chunk > a.tokens || static_cast<int64_t>(past) + chunk > static_cast<int64_t>(a.max_blocks) * kBlock ||
      row < 0 || row >= a.rows) {
    if (threadIdx.x == 0) atomicOr(a.err, B2_DEV_BAD_LENGTH);
    return;
  }
  if (threadIdx.x < 2 * kDim) {
    const int g = threadIdx.x >> 6, d = threadIdx.x & 63;
    qs[g][d] = __uint_as_float(static_cast<uint32_t>(a.q[row * a.q_stride + (2 * h + g) * kDim + d]) << 16) * a.scale_log2;
  }
  __syncthreads();
  const int n = past + t + 1, nblk = (n + kBlock - 1) / kBlock;
  float m[2] = {-1.0e30f, -1.0e30f}, l[2] = {0.f, 0.f}, o[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  for (int i = warp; i < nblk; i += 4) {
    const int blk = a.block_tables[static_cast<int64_t>(b) * a.max_blocks + i];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) atomicOr(a.err, B2_DEV_BAD_BLOCK);
      continue;
    }
    const int64_t si = static_cast<int64_t>(blk) * kHkv + h;
    const uint8_t *k = a.k_pool + si * kTile, *v = a.v_pool + si * kTile;
    const float ks = a.k_scale[si], vs = a.v_scale[si];
    const int valid = min(kBlock, n - i * kBlock);
    float s[2][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int tok = lane + 32 * half;
      float s0 = 0.f, s1 = 0.f;
      for (int d = 0; d < kDim; d += 2) {
        const float2 x = from_e4m3x2(*reinterpret_cast<const uint16_t *>(k + tok * kDim + d));
        s0 += x.x * qs[0][d] + x.y * qs[0][d + 1];
        s1 += x.x * qs[1][d] + x.y * qs[1][d + 1];
      }
      s[half][0] = tok < valid ? s0 * ks : -INFINITY;
      s[half][1] = tok < valid ? s1 * ks : -INFINITY;
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const float mn = fmaxf(m[g], warp_max(fmaxf(s[0][g], s[1][g])));
      const float c = ex2(m[g] - mn);
      m[g] = mn;
      const float p0 = ex2(s[0][g] - mn), p1 = ex2(s[1][g] - mn);
      l[g] = l[g] * c + p0 + p1;
      o[g][0] *= c;
      o[g][1] *= c;
      ps[warp][g][lane] = p0 * vs;
      ps[warp][g][lane + 32] = p1 * vs;
    }
    __syncwarp();
    for (int tok = 0; tok < valid; ++tok) {
      const float v0 = from_e4m3x2(v[lane * kBlock + tok]).x, v1 = from_e4m3x2(v[(lane + 32) * kBlock + tok]).x;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        o[g][0] = fmaf(ps[warp][g][tok], v0, o[g][0]);
        o[g][1] = fmaf(ps[warp][g][tok], v1, o[g][1]);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int g = 0; g < 2; ++g) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], off);
    red[warp][g][2 + lane] = o[g][0];
    red[warp][g][2 + lane + 32] = o[g][1];
    if (lane == 0) {
      red[warp][g][0] = m[g];
      red[warp][g][1] = l[g];
    }
  }
  __syncthreads();
  const int g = threadIdx.x >> 6, d = threadIdx.x & 63;
  float M = -1.0e30f, L = 0.f, O = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, red[w][g][0]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float c = ex2(red[w][g][0] - M);
    L = fmaf(red[w][g][1], c, L);
    O = fmaf(red[w][g][2 + d], c, O);
  }
  a.out[(row * kHq + 2 * h + g) * kDim + d] = static_cast<uint16_t>(bf16_bits(O / L));
}

// ------------------------------------------------------------------ decode step

// The step streams the cache once: 64-token tiles of one (sequence, KV head),
// 4 KiB of K and 4 KiB of V codes and their two scales.  All tiles of the batch
// in the order (sequence, head, block) are cut into equal ranges, one per warp,
// so every warp streams the same number of tiles whatever the lengths are.  A
// warp is its own pipeline: lane 0 copies the tiles of the warp's range
// (cp.async.bulk on an mbarrier per stage) kStages ahead, the warp multiplies
// them with mma.sync m16n8k16 in f16 (e4m3 codes are exact in f16) and hands
// the stage back to itself, with no barrier between warps until the end.
//
//   S[64 x 8]   = K[64 x 64] . Q^T       columns: new token x head of the pair
//   O^T[64 x 8] += V^T[64 x 64] . P^T    V is stored dim-major, so both A
//                                        operands are rows of 16-byte pieces
// Which tokens and dims the rows and k slots of a fragment stand for is free as
// long as both operands agree: a lane's 16 k slots of four mma steps are 16
// adjacent bytes of a row, so an operand of 16 rows is two 16-byte loads per
// lane, free of bank conflicts without a swizzle.
//
// Scales: a column's scores are c * (q factor * k scale).  The sum of p runs
// against the reference m (log2 units), moved only when a score exceeds m + 8
// (a vote, no shuffles, in all other tiles).  The products p * v scale are
// rounded to f16 against a reference of their own, mo: g = v scale * 2^(m -
// mo) <= 2^7 keeps p * g below 2^15; above that the tile's true maximum
// decides whether mo moves.  f16 holds 11 bits of p (bf16 would hold 8) down to
// 2^-14 of the reference.
//
// Ends: a segment (sequence, head) inside one warp's range is written by that
// warp.  Others leave partial states in shared memory, merged by the CTA after
// its last tile; what crosses CTAs goes through the workspace, and the last
// CTA to arrive merges it in CTA order (the result does not depend on who is
// last).  At most two segments of a CTA are open, so the workspace has two
// slots and one counter per CTA whatever the batch.
constexpr int kStages = 3;
constexpr int kWarps = 8;
constexpr int kStepThreads = kWarps * 32;
constexpr int kMaxSeqs = 2048;   // sequences per launch (prefix sums in shared memory)
constexpr int kMaxCtas = 256;
constexpr uint64_t kDrainNs = 2000000000ull;
constexpr float kSlack = 8.0f;          // log2 units that p may exceed 1 by
constexpr float kMaxGain = 128.0f;      // g without a look at the tile's maximum
constexpr float kUnset = -1.0e30f;

template <int kT>
struct __align__(128) StepShared {
  static constexpr int kCols = 2 * kT;
  struct State {  // unnormalised output, then (m, l), of every column
    float o[kCols][kDim];
    float ml[kCols][2];
  };
  uint8_t codes[kWarps][kStages][2 * kTile];
  float scales[kWarps][kStages][8];  // k scales of 4 adjacent heads, v scales
  union {
    uint16_t q[8][kDim];             // f16, scaled per column
    uint16_t out[8][kDim];           // bf16, on the way to memory
  } row[kWarps];
  State head[kWarps];                // a segment that began before the warp's range
  float factor[kWarps][8];
  uint64_t full[kWarps][kStages];
  int tile[kWarps][kStages];         // block * 8 + head, -1: no such block
  int open[kWarps][2];               // segments of the warp's partial states (head[], codes[][0]), -1: none
  int warp_sum[kWarps];
  int prefix[kMaxSeqs + 1];          // blocks of sequences 0 .. b-1
};

struct StepArgs {
  const uint16_t *qkv;
  int64_t row_stride;
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
  int32_t *counters;  // [kMaxCtas], zero between calls
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

// A 16 x 64 operand of codes: this lane's 16 bytes of rows g and g + 8.
__device__ __forceinline__ void mma_codes(float c[4], const uint4 &r0, const uint4 &r1, const uint32_t b[4][2]) {
  const uint32_t u[4] = {r0.x, r0.y, r0.z, r0.w}, w[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a0, a1, a2, a3;
    codes_f16(u[i], a0, a2);
    codes_f16(w[i], a1, a3);
    mma_f16(c, a0, a1, a2, a3, b[i][0], b[i][1]);
  }
}

// First tile of unit u of `units` over `total` tiles.
__device__ __forceinline__ int unit_start(int u, int total, int units) {
  return static_cast<int>(static_cast<int64_t>(u) * total / units);
}

// Running sum of partial states: lane (16 lanes per column) owns columns 2 v +
// lane / 16 and 4 dims of each.
template <int kT>
struct StateSum {
  float m[kT], l[kT];
  float4 o[kT];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int v = 0; v < kT; ++v) {
      m[v] = kUnset;
      l[v] = 0.f;
      o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __device__ __forceinline__ void add(int v, float2 ml, float4 x) {
    const float n = fmaxf(m[v], ml.x);
    const float c0 = ex2(m[v] - n), c1 = ex2(ml.x - n);
    m[v] = n;
    l[v] = l[v] * c0 + ml.y * c1;
    o[v].x = o[v].x * c0 + x.x * c1;
    o[v].y = o[v].y * c0 + x.y * c1;
    o[v].z = o[v].z * c0 + x.z * c1;
    o[v].w = o[v].w * c0 + x.w * c1;
  }
  __device__ __forceinline__ void store(typename StepShared<kT>::State *to, int lane) const {
    const int d = 4 * (lane & 15);
#pragma unroll
    for (int v = 0; v < kT; ++v) {
      const int col = 2 * v + (lane >> 4);
      *reinterpret_cast<float4 *>(&to->o[col][d]) = o[v];
      if (d == 0) *reinterpret_cast<float2 *>(to->ml[col]) = make_float2(m[v], l[v]);
    }
  }
  // the context rows of `ntok` tokens, kHq * kDim apart
  __device__ __forceinline__ void write(uint16_t *out, int ntok, int lane) const {
#pragma unroll
    for (int v = 0; v < kT; ++v) {
      if (v >= ntok) break;
      const float inv = 1.0f / l[v];
      *reinterpret_cast<uint2 *>(out + (v * kHq + (lane >> 4)) * kDim + 4 * (lane & 15)) =
          make_uint2(pack_bf16x2_rn(o[v].x * inv, o[v].y * inv), pack_bf16x2_rn(o[v].z * inv, o[v].w * inv));
    }
  }
};

template <int kT>
__global__ void __launch_bounds__(kStepThreads, 1) kv8_step_kernel(const StepArgs a) {
  using Shared = StepShared<kT>;
  using State = typename Shared::State;
  extern __shared__ uint8_t smem_raw[];
  Shared &sh = *reinterpret_cast<Shared *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;   // mma: row (column) group, thread in group
  const int j = lane & 7, grp = lane >> 3;  // head vectors: 8 values, vector of four
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&sh.full[warp][s]), 1);
    mbar_fence_init();
    sh.open[warp][0] = sh.open[warp][1] = -1;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // blocks of every sequence, and their prefix sums
  auto lengths = [&](int b, int &past, int &ntok) -> bool {
    past = __ldg(a.past_lens + b);
    ntok = a.chunk_lens ? __ldg(a.chunk_lens + b) : a.tokens;
    return past >= 0 && ntok >= 0 && ntok <= a.tokens &&
           static_cast<int64_t>(past) + ntok <= static_cast<int64_t>(a.max_blocks) * kBlock;
  };
  int running = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kStepThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int n = 0;
    if (b < a.batch) {
      int past, ntok;
      if (lengths(b, past, ntok)) n = ntok > 0 ? (past + ntok + kBlock - 1) / kBlock : 0;
      else if (blockIdx.x == 0) atomicOr(a.err, B2_DEV_BAD_LENGTH);
    }
    int incl = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
    }
    if (lane == 31) sh.warp_sum[warp] = incl;
    __syncthreads();
    int before = running, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int v = sh.warp_sum[w];
      before += w < warp ? v : 0;
      all += v;
    }
    if (b < a.batch) sh.prefix[b + 1] = before + incl;
    running += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) sh.prefix[0] = 0;
  __syncthreads();
  const int total = running * kHkv;
  // as many CTAs as there are warps' tiles to hand out
  const int ctas = min(static_cast<int>(gridDim.x), (total + kWarps - 1) / kWarps);
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const int units = ctas * kWarps, unit = static_cast<int>(blockIdx.x) * kWarps + warp;
  const int x0 = unit_start(unit, total, units), x1 = unit_start(unit + 1, total, units);

  // the sequence that block number p of the batch belongs to
  auto sequence_of = [&](int p) {
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh.prefix[mid] <= p) lo = mid; else hi = mid;
    }
    return lo;
  };
  // pool tile of tile number x (table entry read by this lane), -1: no such block
  auto pool_tile = [&](int x) {
    if (x >= x1) return -1;
    const int b = sequence_of(x / kHkv);
    const int n = sh.prefix[b + 1] - sh.prefix[b], r = x - sh.prefix[b] * kHkv;
    const int h = r / n;
    const int blk = __ldg(a.block_tables + static_cast<int64_t>(b) * a.max_blocks + (r - h * n));
    return blk < 0 || blk >= a.num_blocks ? -1 : blk * kHkv + h;
  };

  const uint64_t policy = evict_first_policy();
  int entry = pool_tile(x0 + lane), entry_next = pool_tile(x0 + 32 + lane);  // of 32 tiles of the range each
  int issued = 0;
  auto issue = [&]() {
    if (x0 + issued >= x1) return;
    if (issued > 0 && (issued & 31) == 0) {
      entry = entry_next;
      entry_next = pool_tile(x0 + issued + 32 + lane);
    }
    const int id = __shfl_sync(0xffffffffu, entry, issued & 31);
    if (lane == 0) {
      const int s = issued % kStages;
      const int from = id < 0 ? 0 : id;  // a tile that exists; its result is flagged as bad
      if (id < 0) atomicOr(a.err, B2_DEV_BAD_BLOCK);
      sh.tile[warp][s] = id;
      const uint32_t bar = smem_u32(&sh.full[warp][s]), dst = smem_u32(sh.codes[warp][s]);
      mbar_expect_tx(bar, 2 * kTile + 32);
      bulk_load(dst, a.k_pool + static_cast<int64_t>(from) * kTile, kTile, bar, policy);
      bulk_load(dst + kTile, a.v_pool + static_cast<int64_t>(from) * kTile, kTile, bar, policy);
      const uint32_t sc = smem_u32(sh.scales[warp][s]);
      bulk_load(sc, a.k_scale + (from & ~3), 16, bar, policy);
      bulk_load(sc + 16, a.v_scale + (from & ~3), 16, bar, policy);
    }
    ++issued;
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue();

  // state of the current segment: columns 2t, 2t + 1 in the lanes of thread t
  uint32_t bq[4][2];
  float o[4][4], m0 = kUnset, m1 = kUnset, mo0 = kUnset, mo1 = kUnset, l0 = 0.f, l1 = 0.f, f0 = 0.f, f1 = 0.f;
  uint4 fresh[kT];  // bf16 k (lanes 16-23) and v (24-31) of the segment's new tokens
  int b = 0, h = 0, blk = 0, nblk = 0, past = 0, ntok = 0;
  bool ok = true;
  if (x0 < x1) {
    b = sequence_of(x0 / kHkv);
    nblk = sh.prefix[b + 1] - sh.prefix[b];
    const int r = x0 - sh.prefix[b] * kHkv;
    h = r / nblk;
    blk = r - h * nblk;
  }
  bool begin = true;      // the next tile is the segment's first in this warp
  bool from_start = blk == 0;  // ... and the segment's first of all
  for (int x = x0; x < x1; ++x) {
    const int k = x - x0, s = k % kStages;
    if (begin) {
      // queries of the segment: norm + RoPE, then f16 columns in shared memory
      lengths(b, past, ntok);
      const int vec = grp < 2 ? 2 * h + grp : (grp == 2 ? kHq + h : kHq + kHkv + h);
#pragma unroll
      for (int i = 0; i < kT; ++i)
        if (i < ntok)
          fresh[i] = __ldg(reinterpret_cast<const uint4 *>(
              a.qkv + (static_cast<int64_t>(b) * a.tokens + i) * a.row_stride + vec * kDim + j * 8));
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
          // the column's largest value at 2^8: f16 keeps all bf16 bits of values down to 2^-22 of it
          int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
          e = e < -100 ? -100 : e;
          const float up = __uint_as_float(static_cast<uint32_t>(135 - e) << 23);
          uint4 w;
          w.x = pack_f16x2(y[0] * up, y[1] * up);
          w.y = pack_f16x2(y[2] * up, y[3] * up);
          w.z = pack_f16x2(y[4] * up, y[5] * up);
          w.w = pack_f16x2(y[6] * up, y[7] * up);
          *reinterpret_cast<uint4 *>(&sh.row[warp].q[2 * i + grp][8 * j]) = w;
          if (j == 0) sh.factor[warp][2 * i + grp] = __uint_as_float(static_cast<uint32_t>(119 + e) << 23) * a.scale_log2;
        }
      }
      __syncwarp();
      const bool mine = g < 2 * ntok;
      uint4 w0 = make_uint4(0u, 0u, 0u, 0u), w1 = w0;
      if (mine) {
        const uint4 *p = reinterpret_cast<const uint4 *>(&sh.row[warp].q[g][16 * t]);
        w0 = p[0];
        w1 = p[1];
      }
      bq[0][0] = w0.x; bq[0][1] = w0.y; bq[1][0] = w0.z; bq[1][1] = w0.w;
      bq[2][0] = w1.x; bq[2][1] = w1.y; bq[3][0] = w1.z; bq[3][1] = w1.w;
      f0 = t < ntok ? sh.factor[warp][2 * t] : 0.f;
      f1 = t < ntok ? sh.factor[warp][2 * t + 1] : 0.f;
      m0 = m1 = mo0 = mo1 = kUnset;
      l0 = l1 = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      begin = false;
    }
    if (!mbar_wait(smem_u32(&sh.full[warp][s]), (k / kStages) & 1, a.wait_ns)) ok = false;
    if (__any_sync(0xffffffffu, !ok)) {
      ok = false;
      if (lane == 0) atomicOr(a.err, B2_DEV_TIMEOUT);
      break;
    }
    uint8_t *kc = sh.codes[warp][s], *vc = kc + kTile;
    float ks = sh.scales[warp][s][h & 3], vs = sh.scales[warp][s][4 + (h & 3)];
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

    // S = K . Q^T: row g of m-tile i, half u, is token 16 (g / 2) + 4 i + 2 u + g % 2
    float c[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *p = kc + (16 * (g >> 1) + 4 * i + (g & 1)) * kDim + 16 * t;
      const uint4 r0 = *reinterpret_cast<const uint4 *>(p), r1 = *reinterpret_cast<const uint4 *>(p + 2 * kDim);
#pragma unroll
      for (int e = 0; e < 4; ++e) c[i][e] = 0.f;
      mma_codes(c[i], r0, r1, bq);
    }
    // scores in log2 units against the reference m
    const float w0 = f0 * ks, w1 = f1 * ks;
    const bool tail = key0 + kBlock > past + 1;  // some token does not see the whole tile
    if (tail) {
      const int lim = past + t + 1 - key0;  // token t sees rows < lim
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = 16 * (g >> 1) + 4 * i + (e & 2) + (g & 1);
          if (tok >= lim) c[i][e] = -INFINITY;
          else c[i][e] *= (e & 1) ? w1 : w0;
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[i][e] *= (e & 1) ? w1 : w0;
    }
    float top0 = c[0][0], top1 = c[0][1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top0 = fmaxf(top0, fmaxf(c[i][0], c[i][2]));
      top1 = fmaxf(top1, fmaxf(c[i][1], c[i][3]));
    }
    if (__any_sync(0xffffffffu, t < ntok && (top0 > m0 + kSlack || top1 > m1 + kSlack))) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, off));
        top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, off));
      }
      const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
      l0 *= ex2(m0 - n0);
      l1 *= ex2(m1 - n1);
      m0 = n0;
      m1 = n1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i][0] = ex2(c[i][0] - m0);
      c[i][1] = ex2(c[i][1] - m1);
      c[i][2] = ex2(c[i][2] - m0);
      c[i][3] = ex2(c[i][3] - m1);
      l0 += c[i][0] + c[i][2];
      l1 += c[i][1] + c[i][3];
    }
    // p * v scale against the reference mo (mantissa and exponent of the scale apart)
    const uint32_t vbits = __float_as_uint(vs);
    const float vmant = __uint_as_float((vbits & 0x007fffffu) | 0x3f800000u);
    const float vexp = static_cast<float>(static_cast<int>(vbits >> 23) - 127);
    float g0 = vmant * ex2(m0 - mo0 + vexp), g1 = vmant * ex2(m1 - mo1 + vexp);
    if (__any_sync(0xffffffffu, t < ntok && (g0 > kMaxGain || g1 > kMaxGain))) {
      float p0 = c[0][0], p1 = c[0][1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p0 = fmaxf(p0, fmaxf(c[i][0], c[i][2]));
        p1 = fmaxf(p1, fmaxf(c[i][1], c[i][3]));
      }
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        p0 = fmaxf(p0, __shfl_xor_sync(0xffffffffu, p0, off));
        p1 = fmaxf(p1, __shfl_xor_sync(0xffffffffu, p1, off));
      }
      // the largest product at 1
      const float n0 = p0 > 0.f ? fmaxf(mo0, m0 + vexp + __log2f(p0)) : mo0;
      const float n1 = p1 > 0.f ? fmaxf(mo1, m1 + vexp + __log2f(p1)) : mo1;
      const float a0 = ex2(mo0 - n0), a1 = ex2(mo1 - n1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i][0] *= a0;
        o[i][1] *= a1;
        o[i][2] *= a0;
        o[i][3] *= a1;
      }
      mo0 = n0;
      mo1 = n1;
      g0 = vmant * ex2(m0 - mo0 + vexp);
      g1 = vmant * ex2(m1 - mo1 + vexp);
    }
    uint32_t bp[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bp[i][0] = transpose8x8(pack_f16x2(c[i][0] * g0, c[i][1] * g1));
      bp[i][1] = transpose8x8(pack_f16x2(c[i][2] * g0, c[i][3] * g1));
    }
    // O^T += V^T . P^T: row g of m-tile i, half u, is dim 16 i + 8 u + g
    uint4 keep = make_uint4(~0u, ~0u, ~0u, ~0u);  // codes of rows past the sequence must not meet p = 0
    if (tail) {
      const int n = past + ntok - key0 - 16 * t;
      auto mask = [&](int i) { return n >= 4 * i + 4 ? ~0u : (n <= 4 * i ? 0u : (1u << (8 * (n - 4 * i))) - 1u); };
      keep = make_uint4(mask(0), mask(1), mask(2), mask(3));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t *p = vc + (16 * i + g) * kBlock + 16 * t;
      uint4 r0 = *reinterpret_cast<const uint4 *>(p), r1 = *reinterpret_cast<const uint4 *>(p + 8 * kBlock);
      if (tail) {
        r0.x &= keep.x; r0.y &= keep.y; r0.z &= keep.z; r0.w &= keep.w;
        r1.x &= keep.x; r1.y &= keep.y; r1.z &= keep.z; r1.w &= keep.w;
      }
      mma_codes(o[i], r0, r1, bp);
    }
    __syncwarp();
    issue();  // the stage is read: its next tile

    const bool last = blk + 1 == nblk;  // of the segment
    if (last || x + 1 == x1) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      // the output in units of 2^m, as the sum
      float s0 = ex2(mo0 - m0), s1 = ex2(mo1 - m1);
      if (last && from_start) {
        s0 /= l0;
        s1 /= l1;
        if (t < ntok) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sh.row[warp].out[2 * t][16 * i + g] = static_cast<uint16_t>(bf16_bits(o[i][0] * s0));
            sh.row[warp].out[2 * t + 1][16 * i + g] = static_cast<uint16_t>(bf16_bits(o[i][1] * s1));
            sh.row[warp].out[2 * t][16 * i + 8 + g] = static_cast<uint16_t>(bf16_bits(o[i][2] * s0));
            sh.row[warp].out[2 * t + 1][16 * i + 8 + g] = static_cast<uint16_t>(bf16_bits(o[i][3] * s1));
          }
        }
        __syncwarp();
        for (int c8 = lane; c8 < 2 * ntok * 8; c8 += 32) {
          const int col = c8 >> 3;
          *reinterpret_cast<uint4 *>(a.out + ((static_cast<int64_t>(b) * a.tokens + (col >> 1)) * kHq + 2 * h + (col & 1)) * kDim +
                                     8 * (c8 & 7)) = *reinterpret_cast<const uint4 *>(&sh.row[warp].out[col][8 * (c8 & 7)]);
        }
        __syncwarp();
      } else {
        // open: began before this range (head), or goes on behind it (in the ring, idle by then)
        const int which = from_start ? 1 : 0;
        State *st = which ? reinterpret_cast<State *>(sh.codes[warp][0]) : &sh.head[warp];
        if (t < kT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            st->o[2 * t][16 * i + g] = o[i][0] * s0;
            st->o[2 * t + 1][16 * i + g] = o[i][1] * s1;
            st->o[2 * t][16 * i + 8 + g] = o[i][2] * s0;
            st->o[2 * t + 1][16 * i + 8 + g] = o[i][3] * s1;
          }
          if (g == 0) {
            st->ml[2 * t][0] = m0;
            st->ml[2 * t][1] = l0;
            st->ml[2 * t + 1][0] = m1;
            st->ml[2 * t + 1][1] = l1;
          }
        }
        if (lane == 0) sh.open[warp][which] = b * kHkv + h;
      }
      if (last) {
        begin = from_start = true;
        blk = -1;
        if (++h == kHkv) {
          h = 0;
          if (x + 1 < x1) {
            do ++b; while (sh.prefix[b + 1] == sh.prefix[b]);
            nblk = sh.prefix[b + 1] - sh.prefix[b];
          }
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

  // The CTA's partial states in tile order: run r of states of one segment is
  // merged by warp r % kWarps
  int run = 0;
  for (int i = 0;; ++run) {
    while (i < 2 * kWarps && sh.open[i >> 1][i & 1] < 0) ++i;
    if (i == 2 * kWarps) break;
    const int seg = sh.open[i >> 1][i & 1];
    uint32_t members = 0;
    for (; i < 2 * kWarps; ++i) {
      const int other = sh.open[i >> 1][i & 1];
      if (other == seg) members |= 1u << i;
      else if (other >= 0) break;
    }
    if (run % kWarps != warp) continue;
    StateSum<kT> sum;
    sum.clear();
    for (uint32_t rest = members; rest; rest &= rest - 1) {
      const int e = __ffs(rest) - 1;
      const State *st = (e & 1) ? reinterpret_cast<const State *>(sh.codes[e >> 1][0]) : &sh.head[e >> 1];
#pragma unroll
      for (int v = 0; v < kT; ++v) {
        const int col = 2 * v + (lane >> 4);
        sum.add(v, *reinterpret_cast<const float2 *>(st->ml[col]),
                *reinterpret_cast<const float4 *>(&st->o[col][4 * (lane & 15)]));
      }
    }
    const int sb = seg / kHkv, sh_head = seg - sb * kHkv;
    const int n = sh.prefix[sb + 1] - sh.prefix[sb];
    const int64_t first_tile = static_cast<int64_t>(sh.prefix[sb]) * kHkv + sh_head * n;
    // the CTAs that hold tiles of the segment (CTA c starts at tile c * total / ctas)
    const int cf = static_cast<int>(((first_tile + 1) * ctas - 1) / total);
    const int cl = static_cast<int>(((first_tile + n) * ctas - 1) / total);
    int spast, stok;
    lengths(sb, spast, stok);
    uint16_t *dst = a.out + (static_cast<int64_t>(sb) * a.tokens * kHq + 2 * sh_head) * kDim;
    if (cf == cl) {
      sum.write(dst, stok, lane);
      continue;
    }
    // the segment's first CTA leaves its state in slot 1, the others in slot 0
    State *slots = reinterpret_cast<State *>(a.slots);
    const int cta = static_cast<int>(blockIdx.x);
    sum.store(slots + 2 * cta + (cta == cf ? 1 : 0), lane);
    __syncwarp();
    int arrived = 0;
    if (lane == 0) {
      __threadfence();
      arrived = atomicAdd(a.counters + cf, 1) == cl - cf;
      if (arrived) __threadfence();
    }
    if (!__shfl_sync(0xffffffffu, arrived, 0)) continue;
    __syncwarp();
    sum.clear();
    for (int c0 = cf; c0 <= cl; c0 += 8) {
      // eight states' loads in flight together
#pragma unroll
      for (int v = 0; v < kT; ++v) {
        const int col = 2 * v + (lane >> 4);
        float2 ml[8];
        float4 x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = min(c0 + e, cl);
          const State *st = slots + 2 * c + (c == cf ? 1 : 0);
          ml[e] = __ldcg(reinterpret_cast<const float2 *>(st->ml[col]));
          x[e] = __ldcg(reinterpret_cast<const float4 *>(&st->o[col][4 * (lane & 15)]));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e <= cl) sum.add(v, ml[e], x[e]);
      }
    }
    sum.write(dst, stok, lane);
    if (lane == 0) a.counters[cf] = 0;
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

constexpr int64_t kCounterBytes = kMaxCtas * 4;
constexpr int64_t kWorkspaceBytes = kCounterBytes + 2 * kMaxCtas * static_cast<int64_t>(sizeof(StepShared<kMaxStepTokens>::State));

template <int kT>
int launch_step(StepArgs a, cudaStream_t st) {
  if (!step_ready<kT>()) return fail(B2_ERR_CUDA, "cannot set the step kernel's shared memory size");
  // launches of at most kMaxSeqs sequences whose tiles an int32 counts
  const int64_t most = ((int64_t(1) << 28) - 1) / a.max_blocks;
  const int per = static_cast<int>(most < kMaxSeqs ? (most < 1 ? 1 : most) : kMaxSeqs);
  const int batch = a.batch;
  for (int b0 = 0; b0 < batch; b0 += per) {
    a.batch = batch - b0 < per ? batch - b0 : per;
    const int64_t tiles = static_cast<int64_t>(a.batch) * a.max_blocks * kHkv;
    int64_t ctas = (tiles + kWarps - 1) / kWarps;
    if (ctas > sm_count()) ctas = sm_count();
    if (ctas > kMaxCtas) ctas = kMaxCtas;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kStepThreads);
    cfg.dynamicSmemBytes = sizeof(StepShared<kT>) + 128;
    cfg.stream = st;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const int rc = launched(cudaLaunchKernelEx(&cfg, kv8_step_kernel<kT>, a), "kv8_step_kernel");
    if (rc) return rc;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens;
    a.qkv += rows * a.row_stride;
    a.out += rows * kHq * kDim;
    a.past_lens += a.batch;
    if (a.chunk_lens) a.chunk_lens += a.batch;
    a.block_tables += static_cast<int64_t>(a.batch) * a.max_blocks;
  }
  return b2_clear_error();
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

int launch_append(const AppendArgs &a, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + kWindow - 1) / kWindow);
  kv8_append_kernel<<<grid, 256, 0, st>>>(a);
  return launched(cudaSuccess, "kv8_append_kernel");
}

int launch_attn(const AttnArgs &a, cudaStream_t st) {
  kv8_attn_kernel<<<dim3(static_cast<unsigned>(a.batch * a.tokens), kHkv), 128, 0, st>>>(a);
  return launched(cudaSuccess, "kv8_attn_kernel");
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
  return launch_append(a, static_cast<cudaStream_t>(stream));
}

extern "C" int b2_kv8_decode_step(const uint16_t *qkv, int64_t row_stride, int32_t tokens, const int32_t *chunk_lens,
                                  const uint16_t *gamma_q, const uint16_t *gamma_k, float eps,
                                  const uint16_t *rope_cos, const uint16_t *rope_sin, int32_t rope_rows,
                                  const int32_t *past_lens, const int32_t *block_tables, int32_t max_blocks_per_seq,
                                  uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale,
                                  int32_t num_blocks, int32_t batch, float scale, int32_t mode, uint16_t *out,
                                  void *workspace, int64_t workspace_bytes, int32_t *dev_err, void *stream) {
  if (batch < 0) return fail(B2_ERR_ARG, "batch must be >= 0");
  if (tokens < 1 || tokens > kMaxStepTokens) return fail(B2_ERR_ARG, "tokens must be in [1, 4]");
  if (batch == 0) return b2_clear_error();
  if (static_cast<int64_t>(batch) * tokens > 0x7fffffff) return fail(B2_ERR_ARG, "batch * tokens too large");
  int rc = check_rows(qkv, row_stride, mode, gamma_q, gamma_k, rope_cos, rope_sin, rope_rows);
  if (!rc) rc = check_tables(block_tables, max_blocks_per_seq, past_lens);
  if (!rc) rc = check_cache(k_pool, v_pool, k_scale, v_scale, num_blocks);
  if (rc) return rc;
  if (!out || !dev_err || !aligned16(out)) return fail(B2_ERR_ARG, "out (16-byte aligned) and dev_err are required");
  if (!workspace || !aligned16(workspace) || workspace_bytes < kWorkspaceBytes)
    return fail(B2_ERR_ARG, "workspace must be 16-byte aligned and hold b2_kv8_workspace_bytes()");
  if (!(scale > 0.f)) return fail(B2_ERR_ARG, "scale must be positive");
  StepArgs a{qkv, row_stride, tokens, chunk_lens, gamma_q, gamma_k, eps, rope_cos, rope_sin, rope_rows, past_lens,
             block_tables, max_blocks_per_seq, k_pool, v_pool, k_scale, v_scale, num_blocks, batch,
             scale * 1.4426950408889634f, mode, out, static_cast<int32_t *>(workspace),
             reinterpret_cast<float *>(static_cast<char *>(workspace) + kCounterBytes), dev_err, b2_wait_limit_ns()};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return tokens == 1 ? launch_step<1>(a, st) : launch_step<kMaxStepTokens>(a, st);
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
  if (static_cast<int64_t>(batch) * tokens > 0x7fffffff) return fail(B2_ERR_ARG, "batch * tokens too large");
  AttnArgs a{q, q_stride, rows, row_start, past_lens, chunk_lens, tokens, block_tables, max_blocks_per_seq,
             k_pool, v_pool, k_scale, v_scale, num_blocks, batch, scale * 1.4426950408889634f, out, dev_err};
  return launch_attn(a, static_cast<cudaStream_t>(stream));
}
