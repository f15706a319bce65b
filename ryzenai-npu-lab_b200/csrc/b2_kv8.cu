// The 8-bit paged KV cache (include/b2_kv8.h): e4m3 codes with a power-of-two
// scale for each block of 64 tokens and KV head.
//
//   kv8_append_kernel  q/k norm + RoPE and the quantised append of new tokens
//   kv8_attn_kernel    causal attention of new tokens over the cache

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

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

// ------------------------------------------------------------------ host checks

int check_cache(const void *k_pool, const void *v_pool, const void *k_scale, const void *v_scale, int32_t num_blocks) {
  if (!k_pool || !v_pool || !k_scale || !v_scale) return fail(B2_ERR_ARG, "null cache pointer");
  if (!aligned16(k_pool) || !aligned16(v_pool)) return fail(B2_ERR_ARG, "pools must be 16-byte aligned");
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

constexpr int64_t kWorkspaceBytes = 4 << 20;

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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rows = batch * tokens;
  const bool turned = mode & (B2_NORM_QK | B2_ROPE_QK);
  uint16_t *q = turned ? static_cast<uint16_t *>(workspace) : nullptr;
  if (turned && static_cast<int64_t>(rows) * kHq * kDim * 2 > workspace_bytes) return fail(B2_ERR_ARG, "batch too large");
  if (mode) {
    AppendArgs p{qkv, row_stride, rows, nullptr, nullptr, past_lens, chunk_lens, tokens, block_tables,
                 max_blocks_per_seq, gamma_q, gamma_k, eps, rope_cos, rope_sin, rope_rows, k_pool, v_pool,
                 k_scale, v_scale, num_blocks, q, mode, dev_err};
    rc = launch_append(p, st);
    if (rc) return rc;
  }
  AttnArgs a{turned ? q : qkv, turned ? kHq * kDim : row_stride, rows, nullptr, past_lens, chunk_lens, tokens,
             block_tables, max_blocks_per_seq, k_pool, v_pool, k_scale, v_scale, num_blocks, batch,
             scale * 1.4426950408889634f, out, dev_err};
  return launch_attn(a, st);
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
