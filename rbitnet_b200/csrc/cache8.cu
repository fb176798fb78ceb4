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
#include "rb_common.cuh"

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

// Sixteen codes (16 bytes) times a scale as sixteen bfloat16 values (32 bytes); exact: a code has four binary digits.
__device__ __forceinline__ void values16(const uint4& codes, float scale, uint4 (&out)[2]) {
  const uint32_t in[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t to[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(in[i >> 1] >> (i & 1) * 16), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale, f.y * scale);
    to[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  out[0] = make_uint4(to[0], to[1], to[2], to[3]);
  out[1] = make_uint4(to[4], to[5], to[6], to[7]);
}
// Eight values times a power of two as codes (8 bytes).
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inv) {
  uint32_t out[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    out[i] = lo | hi << 16;
  }
  return make_uint2(out[0], out[1]);
}
// Codes of `count` values brought to another scale by `n` threads: count is a multiple of 16, the address of 16 bytes.
__device__ __forceinline__ void rescale16(uint8_t* codes, int count, float ratio, int me, int n) {
  for (int i = me; i < count / 16; i += n) {
    uint4 c = reinterpret_cast<uint4*>(codes)[i];
    uint32_t* w = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t two[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[x] >> h * 16), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        two[h] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3);
      }
      w[x] = two[0] | two[1] << 16;
    }
    reinterpret_cast<uint4*>(codes)[i] = c;
  }
}

// Sine and cosine of position * frequency: the turns in float64, their fraction in (-1/2, 1/2] in float32, so that far positions
// lose nothing.
__device__ __forceinline__ float2 turn_of(int pos, float freq) {
  const double turns = (double)pos * ((double)freq * 0.15915494309189533577);
  float sn, cs;
  const double whole = turns + 6755399441055744.0;         // 1.5 * 2^52: rounds to whole numbers
  sincospif((float)(turns - (whole - 6755399441055744.0)) * 2.0f, &sn, &cs);
  return make_float2(sn, cs);
}

// A turned pair x, y (of length r <= |x| + |y|) may be off by this: the float32 angle by pi 2^-25, which moves it by pi 2^-25 r; its sine and
// cosine by 2^-24 each, sqrt(2) 2^-24 r; the products by 2^-24 r and the sum by 2^-24 r: 9.98 2^-25 r.  And 2^-24 r for the sums |x| +- off
// that are looked at: where both have one code, x has it; else a border between two codes is near, and the pair is turned in float64.
__device__ __forceinline__ float pair_off(float x, float y) { return (fabsf(x) + fabsf(y)) * 0x1.8p-22f; }

// A pair turned in float64, rounded to odd, so that the rounding to a code that follows is the only one: what is stored does not depend on
// how well float32 sines are rounded.
__device__ __forceinline__ float to_odd(double y) {
  const float f = __double2float_rz(y);
  return (double)f == y ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ float2 exact_turned(float x0, float x1, float freq, int pos, float inv) {
  const double turns = (double)pos * ((double)freq * 0.15915494309189533577);
  double sn, cs;
  sincospi((turns - rint(turns)) * 2.0, &sn, &cs);
  return make_float2(to_odd((x0 * cs - x1 * sn) * (double)inv), to_odd((x0 * sn + x1 * cs) * (double)inv));
}
// Of eight pairs at `to`, the codes of those that are marked: a byte that is not zero in `da` or `db`, at the pair's values in the pieces
// that begin at a0 and b0.  (Rare, so not a part of the kernels' straight line; the thread has written these codes itself.)
__device__ __noinline__ void exact_codes(uint8_t* to, const __nv_bfloat16* head, const float* freq, int pos, float inv, uint2 da, uint2 db, int a0, int b0,
                                         int interleaved) {
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const uint32_t wa = i < 4 ? da.x : da.y, wb = i < 4 ? db.x : db.y;                               // words of byte i
    const uint32_t w = i < 4 ? (i < 2 ? da.x : da.y) : (i < 6 ? db.x : db.y);                        // of bytes 2i, 2i + 1
    if (!(interleaved ? w >> 16 * (i & 1) & 0xffffu : (wa | wb) >> 8 * (i & 3) & 0xffu)) continue;
    const int x = interleaved ? a0 + 2 * i : a0 + i, y = interleaved ? x + 1 : b0 + i;
    const float2 v = exact_turned(__bfloat162float(head[x]), __bfloat162float(head[y]), freq[i], pos, inv);
    to[x] = to_code(v.x);
    to[y] = to_code(v.y);
  }
}

// The scale too is that of the exact rotation.  Both values of a pair are `amax` at most, so the exact largest value lies within 2 amax 0x1.8p-22
// of it, 11 steps of its mantissa beside a border of scales, 448 * 2^e = 1.75 * 2^(e + 8).  Where a border lies that near (of 500,000 blocks one),
// the pairs are turned in float64 and compared with it, in functions of their own: a step's kernel runs once a layer, from instructions that
// are fetched anew, and pays for those that it passes over too.
__device__ __forceinline__ bool near_border(float amax) { return __builtin_expect((__float_as_uint(amax) - (0x600000u - 11) & 0x7fffffu) <= 22, 0); }
// The border, or 0: the bounds of a scale, or an old one, leave no choice.
__device__ __forceinline__ float open_border(float amax, float old) {
  const float lo = scale_for(amax * (1.f - 0x1.8p-21f)), hi = scale_for(amax * (1.f + 0x1.8p-21f));
  return lo < hi && old < hi ? 448.f * lo : 0.f;
}
__device__ __forceinline__ float scale_at_border(float border, bool passed) { return scale_for(border) * (passed ? 2.f : 1.f); }
// Whether one of eight pairs exceeds the border, the pairs in the pieces that begin at a0 and b0.
__device__ __noinline__ bool pieces_pass(const __nv_bfloat16* head, const float* freq, int pos, float border, int a0, int b0, int interleaved) {
  bool passed = false;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const int x = interleaved ? a0 + 2 * i : a0 + i, y = interleaved ? x + 1 : b0 + i;
    const float2 v = exact_turned(__bfloat162float(head[x]), __bfloat162float(head[y]), freq[i], pos, 1.f);
    passed |= fmaxf(fabsf(v.x), fabsf(v.y)) > border;        // (rounded to odd: above the border stays above it)
  }
  return passed;
}
// The scale of a token's key of head size D, by a warp.
__device__ __noinline__ float exact_scale(float amax, float old, const __nv_bfloat16* head, const float* freq, int pos, int D, int interleaved) {
  const float border = open_border(amax, old);
  if (!(border > 0.f)) return scale_for(amax);
  const int e = threadIdx.x & 31;
  const bool passed = e < D / 16 && pieces_pass(head, freq + 8 * e, pos, border, interleaved ? 16 * e : 8 * e, interleaved ? 16 * e + 8 : D / 2 + 8 * e,
                                                interleaved);
  return scale_at_border(border, __any_sync(0xffffffffu, passed));
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

// Any sizes.  One block of threads per (tile, kv head): a tile is the new rows of one block of positions.  It turns the tile's query heads
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
    const float2 t = turn_of(pos0 + tok, p.inv_freq[i]);
    ya = x0 * t.y - x1 * t.x;
    yb = x0 * t.x + x1 * t.y;
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
  const int64_t at = rb_page_offset(p.cache, slot, pos0 - before, kvh);       // of the block's first code
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
    const float old = before > 0 ? *scale : 0.f, border = stream == 0 && p.rot_dim > 0 && near_border(amax) ? open_border(amax, old) : 0.f;
    float needed = scale_for(amax);
    if (border > 0.f) {
      bool passed = false;
      for (int idx = threadIdx.x; idx < n * half; idx += blockDim.x) {
        const int tok = idx / half, i = idx % half;
        if (i >= rhalf) {
          a = p.rot_dim + 2 * (i - rhalf);
          passed |= fmaxf(fabsf(rows[tok * D + a]), fabsf(rows[tok * D + a + 1])) > border;
          continue;
        }
        const __nv_bfloat16* head = p.qkv + (int64_t)(tok0 + tok) * p.qkv_stride + (int64_t)(p.H + kvh) * D;
        const float x0 = __bfloat162float(head[p.interleaved ? 2 * i : i]), x1 = __bfloat162float(head[p.interleaved ? 2 * i + 1 : i + rhalf]);
        const float2 v = exact_turned(x0, x1, p.inv_freq[i], pos0 + tok, 1.f);
        passed |= fmaxf(fabsf(v.x), fabsf(v.y)) > border;
      }
      needed = scale_at_border(border, __syncthreads_or(passed) != 0);
    }
    const float now = fmaxf(old, needed), inv = 1.0f / now;
    if (old < now) {
      const float ratio = old * inv;
      for (int idx = threadIdx.x; idx < before * D; idx += blockDim.x) codes[idx] = to_code(of_code(codes[idx]) * ratio);
    }
    for (int idx = threadIdx.x; idx < n * half; idx += blockDim.x) {
      const int tok = idx / half, i = idx % half;
      uint8_t* to = codes + (int64_t)(before + tok) * D;
      if (stream == 1 || i >= rhalf) {
        a = stream == 1 ? 2 * i : p.rot_dim + 2 * (i - rhalf);
        to[a] = to_code(rows[tok * D + a] * inv);
        to[a + 1] = to_code(rows[tok * D + a + 1] * inv);
        continue;
      }
      a = p.interleaved ? 2 * i : i;
      b = p.interleaved ? 2 * i + 1 : i + rhalf;
      float x = rows[tok * D + a] * inv, y = rows[tok * D + b] * inv;
      const float off = pair_off(x, y);
      if (to_code(fabsf(x) - off) != to_code(fabsf(x) + off) || to_code(fabsf(y) - off) != to_code(fabsf(y) + off)) {
        const __nv_bfloat16* head = p.qkv + (int64_t)(tok0 + tok) * p.qkv_stride + (int64_t)(p.H + kvh) * D;
        const float2 exact = exact_turned(__bfloat162float(head[a]), __bfloat162float(head[b]), p.inv_freq[i], pos0 + tok, inv);
        x = exact.x;
        y = exact.y;
      }
      to[a] = to_code(x);
      to[b] = to_code(y);
    }
    __syncthreads();                             // everybody has read the old scale and the rows
    if (threadIdx.x == 0) *scale = now;
  }
}

// Eight pairs of a row: where their first and second values lie (two 16-byte pieces), and the rotation of them.
__device__ __forceinline__ int piece_a(const Append8& p, int e) { return p.interleaved ? 16 * e : 8 * e; }
__device__ __forceinline__ int piece_b(const Append8& p, int e) { return p.interleaved ? 16 * e + 8 : p.cache.head_dim / 2 + 8 * e; }
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Sines and cosines of pairs 8e .. 8e + 7 at a position.
__device__ __forceinline__ void turns8(const Append8& p, int pos, int e, float2 (&sc)[8]) {
  const float4 lo = *reinterpret_cast<const float4*>(p.inv_freq + 8 * e), hi = *reinterpret_cast<const float4*>(p.inv_freq + 8 * e + 4);
  const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) sc[i] = turn_of(pos, f[i]);
}
__device__ __forceinline__ void turn8(float (&a)[8], float (&b)[8], const float2 (&sc)[8], int interleaved) {
  if (interleaved) {                             // pair i is (2i, 2i + 1) of the sixteen values
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& x = i < 4 ? a[2 * i] : b[2 * i - 8];
      float& y = i < 4 ? a[2 * i + 1] : b[2 * i - 7];
      const float x0 = x, x1 = y;
      x = x0 * sc[i].y - x1 * sc[i].x;
      y = x0 * sc[i].x + x1 * sc[i].y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x0 = a[i], x1 = b[i];
    a[i] = x0 * sc[i].y - x1 * sc[i].x;
    b[i] = x0 * sc[i].x + x1 * sc[i].y;
  }
}
__device__ __forceinline__ float largest8(const float (&a)[8], const float (&b)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
  return m;
}

// Eight pairs at `to`, as codes; turned: a key's, of which those near a border are made anew from `head`, the row's head before the rotation.
__device__ __forceinline__ void store8(const Append8& p, uint8_t* to, const float (&a)[8], const float (&b)[8], bool turned, const __nv_bfloat16* head, int e,
                                       int pos, float inv) {
  *reinterpret_cast<uint2*>(to + piece_a(p, e)) = codes8(a, inv);
  *reinterpret_cast<uint2*>(to + piece_b(p, e)) = codes8(b, inv);
  if (!turned) return;
  float alow[8], ahigh[8], blow[8], bhigh[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float aoff = pair_off(a[i], p.interleaved ? a[i ^ 1] : b[i]), boff = pair_off(b[i], p.interleaved ? b[i ^ 1] : a[i]);
    alow[i] = fabsf(a[i]) - aoff;
    ahigh[i] = fabsf(a[i]) + aoff;
    blow[i] = fabsf(b[i]) - boff;
    bhigh[i] = fabsf(b[i]) + boff;
  }
  const uint2 al = codes8(alow, inv), ah = codes8(ahigh, inv), bl = codes8(blow, inv), bh = codes8(bhigh, inv);
  const uint2 da = make_uint2(al.x ^ ah.x, al.y ^ ah.y), db = make_uint2(bl.x ^ bh.x, bl.y ^ bh.y);
  if (da.x | da.y | db.x | db.y) exact_codes(to, head, p.inv_freq + 8 * e, pos, inv, da, db, piece_a(p, e), piece_b(p, e), p.interleaved);
}

// Heads of a multiple of 16 values, turned whole, rows on 16 bytes: a block of threads per (tile, kv head).  A thread takes one piece of
// eight pairs of one token (SPAN of them where a head is long), and of that piece everything: it makes the sines and cosines once, in
// registers, turns the key's piece and those of the G query heads with them, and keeps the key's and the value's pieces until the
// block's largest values have met.  16-byte loads and stores; the blocks of a tile's kv heads run side by side, so that rows are read whole.
// What bounds it is the chain of waits of a block (tile, positions, rows, the largest values), hidden behind the blocks beside it: 8,192
// tokens of 32 heads on 8 kv heads of 128, 184 MB in 51 us, 3.6 TB/s, of which looking for keys near a border takes 4 and turning those anew
// 2.5 (the same in one straight line: 51.5, and a row of the step kernel 3.7 for 2.7).  Measured without it: 44 us, sines and cosines through shared memory and 256
// threads 64, 92 registers and one block an SM 60.  16 sequences of up to five tokens, 32 heads of 64 on 4: 2.9 us.
template <int THREADS, int SPAN, bool SHARED>
__global__ void __launch_bounds__(THREADS, THREADS * SPAN == 512 ? 2 : 1) append8_tiles_kernel(Append8 p) {
  rb_pdl_launch_dependents();
  __shared__ float tops[2][THREADS / 32];
  const int D = p.cache.head_dim, Kh = p.cache.n_kv_heads, G = p.H / Kh, pieces = D / 16;
  const int tile = blockIdx.y, kvh = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tok0 = p.tile_tok0[tile], n = p.tile_ntok[tile];
  const int slot = p.tok_slot[tok0], pos0 = p.tok_pos[tok0];
  const int before = pos0 % p.block;             // positions that the block holds already
  int64_t at = 0, unit = 0;
  if (p.write_kv) {
    at = rb_page_offset(p.cache, slot, pos0 - before, kvh);                   // of the block's first code
    unit = at / ((int64_t)p.block * D);
  }
  // the thread's pieces; SHARED (tiles of few tokens): groups of threads share the query heads, the first has the key and the value too
  const int per = n * pieces, groups = SHARED ? min(THREADS / per, G) : 1, group = SHARED ? (int)threadIdx.x / per : 0;
  int tok[SPAN], e[SPAN];
  float2 sc[SPAN][8];
#pragma unroll
  for (int i = 0; i < SPAN; ++i) {
    const int item = i * THREADS + (int)threadIdx.x - group * per;
    tok[i] = group < groups ? item / pieces : n;
    e[i] = item % pieces;
    if (p.rot_dim && tok[i] < n) turns8(p, pos0 + tok[i], e[i], sc[i]);        // (frequencies and positions need no wait)
  }
  rb_pdl_wait();
  const __nv_bfloat16* rows = p.qkv + (int64_t)tok0 * p.qkv_stride;
  uint4 raw[2][SPAN][2];
  float old[2] = {0.f, 0.f};
  if (p.write_kv) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < SPAN; ++i) {
        raw[s][i][0] = raw[s][i][1] = make_uint4(0, 0, 0, 0);
        if (tok[i] < n && group == 0) {
          const __nv_bfloat16* src = rows + (int64_t)tok[i] * p.qkv_stride + (int64_t)(p.H + s * Kh + kvh) * D;
          raw[s][i][0] = *reinterpret_cast<const uint4*>(src + piece_a(p, e[i]));
          raw[s][i][1] = *reinterpret_cast<const uint4*>(src + piece_b(p, e[i]));
        }
      }
    if (before > 0) { old[0] = p.k_scale[unit]; old[1] = p.v_scale[unit]; }
  }
  // the query heads
#pragma unroll
  for (int i = 0; i < SPAN; ++i) {
    if (tok[i] >= n) continue;
    const __nv_bfloat16* src = rows + (int64_t)tok[i] * p.qkv_stride + (int64_t)kvh * G * D;
    __nv_bfloat16* dst = p.q_out + ((int64_t)(tok0 + tok[i]) * p.H + kvh * G) * D;
#pragma unroll 2
    for (int g = group; g < G; g += groups) {
      const uint4 qa = *reinterpret_cast<const uint4*>(src + g * D + piece_a(p, e[i])), qb = *reinterpret_cast<const uint4*>(src + g * D + piece_b(p, e[i]));
      float a[8], b[8];
      unpack8(qa, a);
      unpack8(qb, b);
      if (p.rot_dim) turn8(a, b, sc[i], p.interleaved);
      *reinterpret_cast<uint4*>(dst + g * D + piece_a(p, e[i])) = pack8(a);
      *reinterpret_cast<uint4*>(dst + g * D + piece_b(p, e[i])) = pack8(b);
    }
  }
  if (!p.write_kv) return;
  float ka[SPAN][8], kb[SPAN][8], top[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < SPAN; ++i) {
    float a[8], b[8];
    unpack8(raw[1][i][0], a); unpack8(raw[1][i][1], b);
    top[1] = fmaxf(top[1], largest8(a, b));
    unpack8(raw[0][i][0], ka[i]); unpack8(raw[0][i][1], kb[i]);
    if (p.rot_dim && tok[i] < n && group == 0) turn8(ka[i], kb[i], sc[i], p.interleaved);
    top[0] = fmaxf(top[0], largest8(ka[i], kb[i]));
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    top[s] = rb_warp_max(top[s]);
    if (lane == 0) tops[s][warp] = top[s];
  }
  __syncthreads();                               // (everybody has the old scales, too)
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float amax = tops[s][0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) amax = fmaxf(amax, tops[s][w]);
    float needed = scale_for(amax);
    if (s == 0 && near_border(amax) && p.rot_dim) {
      const float border = open_border(amax, old[0]);
      if (border > 0.f) {
        bool passed = false;
#pragma unroll 1
        for (int item = threadIdx.x; item < n * pieces; item += THREADS) {
          const int t = item / pieces, x = item % pieces;
          passed |= pieces_pass(rows + (int64_t)t * p.qkv_stride + (int64_t)(p.H + kvh) * D, p.inv_freq + 8 * x, pos0 + t, border, piece_a(p, x),
                                piece_b(p, x), p.interleaved);
        }
        needed = scale_at_border(border, __syncthreads_or(passed) != 0);
      }
    }
    const float now = fmaxf(old[s], needed), inv = 1.0f / now;
    uint8_t* codes = (uint8_t*)(s ? p.cache.v : p.cache.k) + at;
    if (old[s] < now) rescale16(codes, before * D, old[s] * inv, threadIdx.x, THREADS);
#pragma unroll
    for (int i = 0; i < SPAN; ++i) {
      if (tok[i] >= n || group > 0) continue;
      uint8_t* to = codes + (before + tok[i]) * D;
      if (s) {
        float a[8], b[8];
        unpack8(raw[1][i][0], a); unpack8(raw[1][i][1], b);
        *reinterpret_cast<uint2*>(to + piece_a(p, e[i])) = codes8(a, inv);
        *reinterpret_cast<uint2*>(to + piece_b(p, e[i])) = codes8(b, inv);
      } else {
        store8(p, to, ka[i], kb[i], p.rot_dim > 0, rows + (int64_t)tok[i] * p.qkv_stride + (int64_t)(p.H + kvh) * D, e[i], pos0 + tok[i], inv);
      }
    }
    if (threadIdx.x == 0) (s ? p.v_scale : p.k_scale)[unit] = now;
  }
}

// The same for one token a tile (a decode step): a warp per (row, kv head), up to 8 kv heads a block; the sines and cosines once a block.
// What bounds it is latency: a wait, the row, the old scales, the codes.  One row of 32 heads on 8 kv heads of 128: 2.7 us, 64 rows 3.5
// (3.1 where no key lies near a border).
__global__ void __launch_bounds__(256) append8_step_kernel(Append8 p) {
  rb_pdl_launch_dependents();
  extern __shared__ float2 turns[];              // [D / 2]
  const int D = p.cache.head_dim, Kh = p.cache.n_kv_heads, G = p.H / Kh, half = D / 2, pieces = D / 16;
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y * (blockDim.x >> 5) + warp;
  const int slot = p.tok_slot[row], pos = p.tok_pos[row];
  for (int i = threadIdx.x; p.rot_dim && i < half; i += blockDim.x)         // (positions and frequencies: not written by the kernel before)
    turns[i] = turn_of(pos, p.inv_freq[i]);
  const bool mine = kvh < Kh;
  int64_t at = 0, unit = 0;
  const int before = pos % p.block;
  if (mine && p.write_kv) {
    at = rb_page_offset(p.cache, slot, pos - before, kvh);
    unit = at / ((int64_t)p.block * D);
  }
  rb_pdl_wait();
  const __nv_bfloat16* src = p.qkv + (int64_t)row * p.qkv_stride;
  // items: the key's pieces, the value's, then the query heads'; the first two streams lie in the first turn (D <= 256)
  const int items = (p.write_kv ? 2 * pieces : 0) + G * pieces;
  const int ahead = p.write_kv ? 2 * pieces : 0;
  float old_k = 0.f, old_v = 0.f;
  if (mine && p.write_kv && before > 0) { old_k = p.k_scale[unit]; old_v = p.v_scale[unit]; }
  __syncthreads();
  if (!mine) return;
  for (int base = 0; base < items; base += 32) {
    const int item = base + lane;
    const bool is_k = item < ahead && item < pieces, is_v = item < ahead && !is_k, on = item < items;
    const int e = item % pieces;
    const int64_t head = is_k ? p.H + kvh : is_v ? p.H + Kh + kvh : kvh * G + (item - ahead) / pieces;
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    if (on) {
      unpack8(*reinterpret_cast<const uint4*>(src + head * D + piece_a(p, e)), a);
      unpack8(*reinterpret_cast<const uint4*>(src + head * D + piece_b(p, e)), b);
      if (!is_v && p.rot_dim) {
        float2 sc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i] = turns[8 * e + i];
        turn8(a, b, sc, p.interleaved);
      }
    }
    if (on && !is_k && !is_v) {
      __nv_bfloat16* dst = p.q_out + ((int64_t)row * p.H + head) * D;
      *reinterpret_cast<uint4*>(dst + piece_a(p, e)) = pack8(a);
      *reinterpret_cast<uint4*>(dst + piece_b(p, e)) = pack8(b);
    }
    if (base == 0 && p.write_kv) {
      const float big = largest8(a, b);
      const float top_k = rb_warp_max(is_k ? big : 0.f), top_v = rb_warp_max(is_v ? big : 0.f);
      float needed = scale_for(top_k);
      if (__builtin_expect(near_border(top_k) && p.rot_dim, 0))
        needed = exact_scale(top_k, old_k, src + (int64_t)(p.H + kvh) * D, p.inv_freq, pos, D, p.interleaved);
      const float now_k = fmaxf(old_k, needed), now_v = fmaxf(old_v, scale_for(top_v));
      uint8_t* k = (uint8_t*)p.cache.k + at;
      uint8_t* v = (uint8_t*)p.cache.v + at;
      if (old_k < now_k) rescale16(k, before * D, old_k / now_k, lane, 32);
      if (old_v < now_v) rescale16(v, before * D, old_v / now_v, lane, 32);
      if (is_k || is_v)
        store8(p, (is_k ? k : v) + before * D, a, b, is_k && p.rot_dim > 0, src + head * D, e, pos, 1.0f / (is_k ? now_k : now_v));
      if (lane == 0) { p.k_scale[unit] = now_k; p.v_scale[unit] = now_v; }
    }
  }
}

// The values of whole pages: item i is (slot, page of the sequence, positions in use); what lies behind those is zero, and all of a page
// that the sequence has given back (a negative number in its table).
__device__ __forceinline__ int in_use(const RbPagedLayer& c, int slot, int page, int used) {
  return c.page_table[(int64_t)slot * c.max_pages + page] < 0 ? 0 : used;
}
__global__ void __launch_bounds__(256) cache8_values_kernel(__nv_bfloat16* k_out, __nv_bfloat16* v_out, RbPagedLayer c, const float* k_scale,
                                                           const float* v_scale, const int* items, int block) {
  rb_pdl_launch_dependents();
  const int i = blockIdx.x, kvh = blockIdx.y, D = c.head_dim, n = c.page_size * D;
  const int slot = items[3 * i], page = items[3 * i + 1], used = in_use(c, slot, page, items[3 * i + 2]);
  rb_pdl_wait();
  const int64_t at = used > 0 ? rb_page_offset(c, slot, page * c.page_size, kvh) : 0, to = ((int64_t)i * c.n_kv_heads + kvh) * n;
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

// The same for heads of a multiple of 16 values: a thread turns 16 codes at a time, two pieces of them on their way.  Bounded by the wait for
// those: 128 pages of 8 heads of 128, 50 MB in 13 us, 3.8 TB/s (a code at a time: 49 us).
__global__ void __launch_bounds__(256) cache8_values16_kernel(__nv_bfloat16* k_out, __nv_bfloat16* v_out, RbPagedLayer c, const float* k_scale,
                                                             const float* v_scale, const int* items, int block) {
  rb_pdl_launch_dependents();
  const int i = blockIdx.x, kvh = blockIdx.y, D = c.head_dim, n = c.page_size * D;
  const int slot = items[3 * i], page = items[3 * i + 1], used = in_use(c, slot, page, items[3 * i + 2]);
  rb_pdl_wait();
  const int64_t at = used > 0 ? rb_page_offset(c, slot, page * c.page_size, kvh) : 0, to = ((int64_t)i * c.n_kv_heads + kvh) * n;
  const uint8_t* data = (const uint8_t*)(blockIdx.z ? c.v : c.k) + at;
  const float* scale = (blockIdx.z ? v_scale : k_scale) + at / ((int64_t)block * D);
  __nv_bfloat16* out = (blockIdx.z ? v_out : k_out) + to;
  for (int base = threadIdx.x * 16; base < n; base += 2 * 256 * 16) {              // (two pieces asked for together)
    uint4 codes[2];
    float by[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = base + i * 256 * 16, pos = idx / D;
      const bool in = idx < n && pos < used;
      codes[i] = in ? *reinterpret_cast<const uint4*>(data + idx) : make_uint4(0, 0, 0, 0);
      by[i] = in ? scale[block == c.page_size ? 0 : pos / block] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = base + i * 256 * 16;
      if (idx >= n) break;
      uint4 v[2];
      values16(codes[i], by[i], v);
      *reinterpret_cast<uint4*>(out + idx) = v[0];
      *reinterpret_cast<uint4*>(out + idx + 8) = v[1];
    }
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
// positions of one block of one sequence, in order, `tile_most` at most (null: every row is a tile of its own).
RB_EXPORT int rb_append8(void* q_out, const void* qkv, int64_t qkv_stride, const float* inv_freq, const int* tok_pos, const int* tok_slot,
                         const int* tile_tok0, const int* tile_ntok, int n_tiles, int tile_most, void* cache_k, void* cache_v, float* k_scale,
                         float* v_scale, const int* page_table, int max_pages, int page_size, int H, int Kh, int D, int write_kv,
                         int rot_dim, int interleaved, cudaStream_t stream) {
  if (n_tiles == 0) return 0;
  RB_REQUIRE(D > 0 && D % 2 == 0 && D <= 512, "rb_append8: head_dim %d must be even, and 512 at most", D);
  RB_REQUIRE(rot_dim >= 0 && rot_dim <= D && rot_dim % 2 == 0, "rb_append8: the rotated prefix %d must be even and at most %d", rot_dim, D);
  RB_REQUIRE(H > 0 && Kh > 0 && H % Kh == 0 && Kh <= 65535, "rb_append8: %d heads on %d kv heads", H, Kh);
  RB_REQUIRE(!tile_tok0 || n_tiles <= 65535, "rb_append8: %d tiles in one launch", n_tiles);
  const int block = rb_cache8_block(page_size);
  RB_REQUIRE(!tile_tok0 || (tile_ntok && tile_most >= 1 && tile_most <= block), "rb_append8: tiles of %d tokens", tile_most);
  RB_REQUIRE(block > 0, "rb_append8: a page of %d positions must be 64 at most, or a multiple of 64", page_size);
  Append8 p;
  p.q_out = (__nv_bfloat16*)q_out; p.qkv = (const __nv_bfloat16*)qkv; p.qkv_stride = qkv_stride;
  p.inv_freq = inv_freq; p.tok_pos = tok_pos; p.tok_slot = tok_slot; p.tile_tok0 = tile_tok0; p.tile_ntok = tile_ntok;
  p.cache = RbPagedLayer{cache_k, cache_v, page_table, max_pages, page_size, Kh, D};
  p.k_scale = k_scale; p.v_scale = v_scale;
  p.block = block; p.H = H; p.write_kv = write_kv; p.interleaved = interleaved; p.rot_dim = rot_dim;
  const uintptr_t bases = (uintptr_t)inv_freq | (uintptr_t)q_out | (uintptr_t)qkv | (uintptr_t)cache_k | (uintptr_t)cache_v;
  if (D % 16 == 0 && D <= 256 && (rot_dim == D || rot_dim == 0) && qkv_stride % 8 == 0 && (bases & 15) == 0) {
    if (!tile_tok0) {
      const int warps = Kh < 8 ? Kh : 8;
      RB_LAUNCH("rb_append8 (step)", (append8_step_kernel), dim3(n_tiles, (Kh + warps - 1) / warps), warps * 32, (size_t)D / 2 * 8, stream, p);
      return 0;
    }
    // (5 tokens of 32 heads of 64 on 4 kv heads, keys by float32 alone: 4.1 us by one group of threads, 2.3 shared; the shared form costs full
    // tiles 4 %)
    const bool shared = D <= 128 && 2 * tile_most * (D / 16) <= (D <= 64 ? 256 : 512);
    const dim3 grid(Kh, n_tiles);
    if (D <= 64 && shared) RB_LAUNCH("rb_append8 (tiles)", (append8_tiles_kernel<256, 1, true>), grid, 256, 0, stream, p);
    else if (D <= 64) RB_LAUNCH("rb_append8 (tiles)", (append8_tiles_kernel<256, 1, false>), grid, 256, 0, stream, p);
    else if (D <= 128 && shared) RB_LAUNCH("rb_append8 (tiles)", (append8_tiles_kernel<512, 1, true>), grid, 512, 0, stream, p);
    else if (D <= 128) RB_LAUNCH("rb_append8 (tiles)", (append8_tiles_kernel<512, 1, false>), grid, 512, 0, stream, p);
    else RB_LAUNCH("rb_append8 (tiles)", (append8_tiles_kernel<512, 2, false>), grid, 512, 0, stream, p);
    return 0;
  }
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
  if (D % 16 == 0 && (((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)cache_k | (uintptr_t)cache_v) & 15) == 0) {
    RB_LAUNCH("rb_cache8_values", (cache8_values16_kernel), dim3(n, Kh, 2), 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, c, k_scale,
              v_scale, items, block);
    return 0;
  }
  RB_LAUNCH("rb_cache8_values", (cache8_values_kernel), dim3(n, Kh), 256, 0, stream, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, c, k_scale, v_scale,
            items, block);
  return 0;
}
