// The cache held in 8 bits: appending keys and values to it, and reading back what it holds.
//
// Keys and values are e4m3 codes (sign, four exponent bits, three mantissa bits; steps of 2^-9 near zero, 448 at most) in
// pages [page][kv head][position][d], with one float32 scale per block of `block` positions and kv head, keys and values
// apart: value = code * scale.  A scale is a power of two, the least 2^e, e in [-60, 119], that holds the block's largest
// value: amax <= 448 * 2^e.  So the division by it rounds nothing, and a block whose scale grows later (a token with larger
// values joins it) keeps its codes but for their exponents: code * old / new is exact down to the smallest steps, where it
// is rounded once more (to nearest even).  Codes are written by rounding to nearest even; past 448 * 2^119 they stay
// there, NaN stays NaN and does not count for the scale.
//
// A block that begins with the first new position takes its scale from the new values alone: what it held before (another
// sequence's, or tokens that were dropped) has no part in it.  Otherwise scale = max(old, needed).
#include "rb_rotary.cuh"

#include <cuda_fp8.h>

RB_CHECK_READER(cache8)

namespace {

constexpr int LOWEST = -60, HIGHEST = 119;     // exponents that a scale may have
constexpr int MOST_BLOCK = 64;                 // positions of a block, at most

// the scale for values up to amax: 448 = 1.75 * 2^8
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, LOWEST), HIGHEST);            // (zero and denormal values: the lowest; infinity: the highest)
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ uint8_t to_code(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float of_code(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

struct Append8 {
  __nv_bfloat16* q_out;          // [T, H, D]
  const __nv_bfloat16* qkv;      // [T, (H + 2 Kh) D], rows qkv_stride apart (H D without writing)
  int64_t qkv_stride;
  const float* inv_freq;
  const int* tok_pos;
  const int* tok_slot;
  const int* tile_tok0;          // null: tile i is row i alone
  const int* tile_ntok;
  RbPagedLayer cache;
  float* k_scale;
  float* v_scale;
  int block, H, write_kv, interleaved, rot_dim;
};

// One block of threads per (tile, kv head): a tile is the new rows of one block of positions.  It turns the tile's query heads
// of the kv head, then makes its keys and its values, each through shared memory because the scale comes before the codes.
__global__ void __launch_bounds__(256) append8_kernel(Append8 p) {
  rb_pdl_launch_dependents();
  extern __shared__ float rows[];                // [tokens of the tile][D]
  __shared__ float scratch[33];
  const int D = p.cache.head_dim, Kh = p.cache.n_kv_heads, G = p.H / Kh, half = D / 2, rhalf = p.rot_dim / 2;
  const int kvh = blockIdx.y;
  const int tok0 = p.tile_tok0 ? p.tile_tok0[blockIdx.x] : (int)blockIdx.x;
  const int n = p.tile_ntok ? p.tile_ntok[blockIdx.x] : 1;
  const int slot = p.tok_slot[tok0], pos0 = p.tok_pos[tok0];
  rb_pdl_wait();
  // values 2i, 2i+1 of a head after the rotation (of its first rot_dim values), as (where a, value a, where b, value b)
  auto pair = [&](int tok, int64_t head, int i, bool turn, int& a, int& b, float& ya, float& yb) {
    const __nv_bfloat16* src = p.qkv + (int64_t)(tok0 + tok) * p.qkv_stride + head * D;
    if (!turn || i >= rhalf) {
      a = turn ? p.rot_dim + 2 * (i - rhalf) : 2 * i;
      b = a + 1;
      ya = __bfloat162float(src[a]);
      yb = __bfloat162float(src[b]);
      return;
    }
    a = p.interleaved ? 2 * i : i;
    b = p.interleaved ? 2 * i + 1 : i + rhalf;
    const float x0 = __bfloat162float(src[a]), x1 = __bfloat162float(src[b]);
    float sn, cs;
    angle_sincos(pos0 + tok, (double)p.inv_freq[i], 1.0f, &sn, &cs);
    ya = x0 * cs - x1 * sn;
    yb = x0 * sn + x1 * cs;
  };
  int a, b;
  float ya, yb;
  for (int idx = threadIdx.x; idx < n * G * half; idx += blockDim.x) {
    const int tok = idx / (G * half), g = idx / half % G;
    pair(tok, kvh * G + g, idx % half, true, a, b, ya, yb);
    __nv_bfloat16* dst = p.q_out + ((int64_t)(tok0 + tok) * p.H + kvh * G + g) * D;
    dst[a] = __float2bfloat16_rn(ya);
    dst[b] = __float2bfloat16_rn(yb);
  }
  if (!p.write_kv) return;
  const int before = pos0 % p.block;             // positions that the block holds already
  const int64_t at = rb_page_offset(p.cache, slot, pos0, kvh) - (int64_t)before * D;       // of the block's first code
  for (int stream = 0; stream < 2; ++stream) {
    uint8_t* codes = (uint8_t*)(stream == 0 ? p.cache.k : p.cache.v) + at;
    float* scale = (stream == 0 ? p.k_scale : p.v_scale) + at / ((int64_t)p.block * D);
    float amax = 0.f;
    for (int idx = threadIdx.x; idx < n * half; idx += blockDim.x) {
      const int tok = idx / half;
      pair(tok, p.H + stream * Kh + kvh, idx % half, stream == 0, a, b, ya, yb);
      rows[tok * D + a] = ya;
      rows[tok * D + b] = yb;
      amax = fmaxf(amax, fmaxf(fabsf(ya), fabsf(yb)));
    }
    amax = rb_block_max(amax, scratch);          // (its barriers also make the rows visible)
    const float old = before > 0 ? *scale : 0.f, now = fmaxf(old, scale_for(amax)), inv = 1.0f / now;
    if (old < now) {
      const float ratio = old * inv;
      for (int idx = threadIdx.x; idx < before * D; idx += blockDim.x) codes[idx] = to_code(of_code(codes[idx]) * ratio);
    }
    for (int idx = threadIdx.x; idx < n * D; idx += blockDim.x) codes[(int64_t)before * D + idx] = to_code(rows[idx] * inv);
    __syncthreads();                             // everybody has read the old scale and the rows
    if (threadIdx.x == 0) *scale = now;
  }
}

// The values of whole pages: item i is (slot, page of the sequence, positions in use); what lies behind those is zero.
__global__ void __launch_bounds__(256) cache8_values_kernel(__nv_bfloat16* k_out, __nv_bfloat16* v_out, RbPagedLayer c, const float* k_scale,
                                                           const float* v_scale, const int* items, int block) {
  rb_pdl_launch_dependents();
  const int i = blockIdx.x, kvh = blockIdx.y, D = c.head_dim, n = c.page_size * D;
  const int slot = items[3 * i], page = items[3 * i + 1], used = items[3 * i + 2];
  rb_pdl_wait();
  const int64_t at = rb_page_offset(c, slot, page * c.page_size, kvh), to = ((int64_t)i * c.n_kv_heads + kvh) * n;
  const uint8_t* k = (const uint8_t*)c.k + at;
  const uint8_t* v = (const uint8_t*)c.v + at;
  const int64_t s = at / ((int64_t)block * D);
  for (int idx = threadIdx.x; idx < n; idx += blockDim.x) {
    const int pos = idx / D;
    const bool in = pos < used;
    k_out[to + idx] = __float2bfloat16_rn(in ? of_code(k[idx]) * k_scale[s + pos / block] : 0.f);
    v_out[to + idx] = __float2bfloat16_rn(in ? of_code(v[idx]) * v_scale[s + pos / block] : 0.f);
  }
}

}  // namespace

// Positions of a block for pages of `page_size` positions (0: such pages are not taken): a whole page of up to 64, else 64.
RB_EXPORT int rb_cache8_block(int page_size) {
  if (page_size <= 0) return 0;
  if (page_size <= MOST_BLOCK) return page_size;
  return page_size % MOST_BLOCK == 0 ? MOST_BLOCK : 0;
}

// q_out[T, H, D] = turned q rows; k (turned) and v rows enter the cache.  Tile i is the tile_ntok[i] rows from tile_tok0[i] on: new
// positions of one block of one sequence, in order (null: every row is a tile of its own).
RB_EXPORT int rb_append8(void* q_out, const void* qkv, int64_t qkv_stride, const float* inv_freq, const int* tok_pos, const int* tok_slot,
                         const int* tile_tok0, const int* tile_ntok, int n_tiles, void* cache_k, void* cache_v, float* k_scale,
                         float* v_scale, const int* page_table, int max_pages, int page_size, int H, int Kh, int D, int write_kv,
                         int rot_dim, int interleaved, cudaStream_t stream) {
  if (n_tiles == 0) return 0;
  RB_REQUIRE(D > 0 && D % 2 == 0 && D <= 512, "rb_append8: head_dim %d must be even, and 512 at most", D);
  RB_REQUIRE(rot_dim >= 0 && rot_dim <= D && rot_dim % 2 == 0, "rb_append8: the rotated prefix %d must be even and at most %d", rot_dim, D);
  RB_REQUIRE(H > 0 && Kh > 0 && H % Kh == 0 && Kh <= 65535, "rb_append8: %d heads on %d kv heads", H, Kh);
  const int block = rb_cache8_block(page_size);
  RB_REQUIRE(block > 0, "rb_append8: a page of %d positions must be 64 at most, or a multiple of 64", page_size);
  Append8 p;
  p.q_out = (__nv_bfloat16*)q_out; p.qkv = (const __nv_bfloat16*)qkv; p.qkv_stride = qkv_stride;
  p.inv_freq = inv_freq; p.tok_pos = tok_pos; p.tok_slot = tok_slot; p.tile_tok0 = tile_tok0; p.tile_ntok = tile_ntok;
  p.cache = RbPagedLayer{cache_k, cache_v, page_table, max_pages, page_size, Kh, D};
  p.k_scale = k_scale; p.v_scale = v_scale;
  p.block = block; p.H = H; p.write_kv = write_kv; p.interleaved = interleaved; p.rot_dim = rot_dim;
  static RbOncePerDevice configured;
  if (configured.first())
    RB_CUDA(cudaFuncSetAttribute(append8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_BLOCK * 512 * 4));
  const int rows = tile_tok0 ? block : 1;
  RB_LAUNCH("rb_append8", (append8_kernel), dim3(n_tiles, Kh), 256, (size_t)rows * D * 4, stream, p);
  return 0;
}

// k_out, v_out [n, Kh, page_size, D] bfloat16: the values of n pages, items[i] = (slot, page of the sequence, positions in use).
RB_EXPORT int rb_cache8_values(void* k_out, void* v_out, const int* items, int n, void* cache_k, void* cache_v, const float* k_scale,
                               const float* v_scale, const int* page_table, int max_pages, int page_size, int Kh, int D,
                               cudaStream_t stream) {
  if (n == 0) return 0;
  const int block = rb_cache8_block(page_size);
  RB_REQUIRE(block > 0 && Kh > 0 && Kh <= 65535 && D > 0, "rb_cache8_values: bad sizes page=%d Kh=%d D=%d", page_size, Kh, D);
  RbPagedLayer c{cache_k, cache_v, page_table, max_pages, page_size, Kh, D};
  RB_LAUNCH("rb_cache8_values", (cache8_values_kernel), dim3(n, Kh), 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, c, k_scale, v_scale,
            items, block);
  return 0;
}
