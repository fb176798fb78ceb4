// Attention over the cache held in 8 bits (cache8.cu): value = code * scale, a power-of-two scale per block of positions and
// kv head.  Token t at position p of its sequence sees keys max(0, p - window + 1) .. p (and with keep_first the first keys);
// score = (q.k) * scale, in float32, capped where a soft cap is set; softmax with the running maximum and sum in float32 (the
// sink one more term of the sum); o = sum of p v.  A key that a row does not see is not multiplied by anything
// (but in steps of more than 64 rows a kv head, whose bfloat16 pages the prefill kernel reads: there a NaN value of a prompt reaches earlier tokens of its tile).
#include "attention8.cuh"

#include <cuda_fp8.h>

RB_CHECK_READER(attention8)

namespace {

__device__ __forceinline__ float of_code(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

// Any sizes (head sizes other than 64 and 128, pages that are no multiple of 64, more than 32 heads a kv head): one block of threads per
// (token, head); a thread takes a key of every 128 for the scores, then every 128th value.  Bounded by its single-byte loads, of a kv head's keys
// once for each of its query heads, and by one block's walk through a sequence: 64 sequences of up to 8,000 positions, 32 heads on 8 kv heads of
// 80, 1.9 ms, of 256 11.7 ms, 40 heads on one of 128 6.8 ms (the 16-bit cache's kernels: 0.14, 0.52 and 0.05).
__global__ void __launch_bounds__(128) attn8_simple_kernel(Params8 p) {
  extern __shared__ float smem[];                 // q [D], o [D]
  __shared__ float weight[128], v_unit[128], scratch[33];
  __shared__ int64_t where[128];
  rb_pdl_launch_dependents();
  rb_pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, D = p.cache.head_dim, kvh = h / (p.H / p.cache.n_kv_heads);
  const int pos = p.tok_pos[t], slot = p.tok_slot[t];
  float* q = smem;
  float* o = smem + D;
  for (int d = threadIdx.x; d < D; d += 128) {
    q[d] = __bfloat162float(p.q[((int64_t)t * p.H + h) * D + d]);
    o[d] = 0.f;
  }
  const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int kept = min(p.window > 0 ? p.keep : 0, lo);               // the first positions that stay visible, then the window
  const int n = pos - lo + 1 + kept;
  float m = -INFINITY, l = 0.f;
  if (p.sinks != nullptr) { m = p.sinks[h]; l = 1.f; }
  const uint8_t* K = (const uint8_t*)p.cache.k;
  const uint8_t* V = (const uint8_t*)p.cache.v;
  for (int i0 = 0; i0 < n; i0 += 128) {
    __syncthreads();
    const int i = i0 + threadIdx.x;
    float s = -INFINITY;
    if (i < n) {
      const int64_t off = rb_page_offset(p.cache, slot, i < kept ? i : lo + (i - kept), kvh);
      const int64_t unit = off / ((int64_t)p.block * D);
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(q[d], of_code(K[off + d]), dot);
      s = dot * p.k_scale[unit] * p.scale;
      if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
      where[threadIdx.x] = off;
      v_unit[threadIdx.x] = p.v_scale[unit];
    }
    const float m_new = fmaxf(m, rb_block_max(s, scratch));
    const float e = i < n ? expf(s - m_new) : 0.f, corr = m == -INFINITY ? 0.f : expf(m - m_new);
    weight[threadIdx.x] = e;
    l = l * corr + rb_block_sum(e, scratch);
    m = m_new;
    const int here = min(128, n - i0);
    for (int d = threadIdx.x; d < D; d += 128) {
      float acc = o[d] * corr;
      for (int j = 0; j < here; ++j) acc = fmaf(weight[j], of_code(V[where[j] + d]) * v_unit[j], acc);
      o[d] = acc;
    }
  }
  for (int d = threadIdx.x; d < D; d += 128) p.out[((int64_t)t * p.H + h) * D + d] = __float2bfloat16_rn(o[d] / l);
}


}  // namespace

// out[T, H * D]: attention of q[T, H, D] over the codes; rows of any steps (a row's own position and slot say what it sees).
RB_EXPORT int rb_attention8_simple(void* out, const void* q, void* cache_k, void* cache_v, const float* k_scale, const float* v_scale,
                                   const int* page_table, int max_pages, int page_size, const int* tok_pos, const int* tok_slot, int T,
                                   int H, int Kh, int D, float scale, int window, cudaStream_t stream) {
  const RbAttentionOptions opt = rb_attention_take();
  if (T == 0) return 0;
  const int block = rb_cache8_block(page_size);
  RB_REQUIRE(block > 0 && H > 0 && H <= 65535 && Kh > 0 && H % Kh == 0 && D > 0 && D <= 2048,
             "rb_attention8_simple: bad sizes H=%d Kh=%d D=%d page=%d", H, Kh, D, page_size);
  Params8 p;
  p.q = (const __nv_bfloat16*)q; p.out = (__nv_bfloat16*)out;
  p.cache = RbPagedLayer{cache_k, cache_v, page_table, max_pages, page_size, Kh, D};
  p.k_scale = k_scale; p.v_scale = v_scale; p.block = block;
  p.tok_pos = tok_pos; p.tok_slot = tok_slot; p.H = H;
  p.scale = scale; p.window = window; p.keep = opt.keep_first; p.sinks = opt.sinks; p.softcap = opt.softcap;
  RB_LAUNCH("rb_attention8_simple", (attn8_simple_kernel), dim3(T, H), 128, (size_t)2 * D * 4, stream, p);
  return 0;
}
