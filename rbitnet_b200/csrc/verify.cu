// Drafted tokens against the target's logits.
//
// A sequence b has rows first_row[b] .. first_row[b + 1] - 1 of logits.  Row r judges draft d = drafts[r] (the last row none):
// with p = softmax(z_r / T) and q the drafter's probabilities (no probabilities: the draft is certain, q = 1 at d),
//     accepted  while  u_r q(d) < p(d)                                 (u_r = uniforms[r][0], in [0, 1))
// and at the first row that does not accept, or at the last row, one token is taken from max(p - q, 0) (the last row: from p),
// as the first whose running sum in index order exceeds u'_r = uniforms[r][1] of the whole.  The tokens are then distributed
// as if each had been drawn from p alone.  T <= 0: the draft has to be the largest logit's token, the lowest of equals, and
// that is the token taken.  A logit that is NaN counts as -inf; a draft outside the vocabulary is not accepted and takes
// nothing from p; where p - q leaves nothing, the token is drawn from p.
//
// Exponentials and sums are float64: the running sum over 100,000 tokens decides on a single token, and in float32 it would
// move by more than the smallest probabilities, another way for every way of cutting the sum.
#include "rb_common.cuh"

namespace {

constexpr int CHUNK = 4096, THREADS = 256, PICK_THREADS = 1024;

struct Stat { double sum; float max; int arg; };

struct Verify {
  int* accepted;               // [B]
  int* tokens;                 // [B, most + 1]
  const float* logits;         // [R, V], rows `stride` apart
  int64_t stride;
  const float* probs;          // [R, V] or null, rows `probs_stride` apart
  int64_t probs_stride;
  const int* first_row;        // [B + 1]
  const int* drafts;           // [R]
  const float* temperature;    // [B]
  const float* uniforms;       // [R, 2]
  Stat* stats;                 // [R, chunks]
  int B, R, V, most, chunks;
};

__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v; }
// exp((z - m) / T), 1 at the maximum itself (also where that is infinite)
__device__ __forceinline__ double weight(float z, float m, double inv_t) {
  return z == m ? 1.0 : exp(((double)z - (double)m) * inv_t);
}

__global__ void __launch_bounds__(THREADS) verify_stats_kernel(Verify p) {
  rb_pdl_launch_dependents();
  rb_pdl_wait();
  __shared__ float scratch[33];
  __shared__ double sums[THREADS / 32];
  __shared__ int s_arg;
  const int r = blockIdx.x, c = blockIdx.y;
  int seq = 0;
  while (seq + 1 < p.B && p.first_row[seq + 1] <= r) ++seq;
  const float temp = p.temperature[seq];
  const float* z = p.logits + (int64_t)r * p.stride;
  const int lo = c * CHUNK, hi = min(p.V, lo + CHUNK);
  float m = -INFINITY;
  for (int i = lo + threadIdx.x; i < hi; i += THREADS) m = fmaxf(m, clean(z[i]));
  m = rb_block_max(m, scratch);
  if (threadIdx.x == 0) s_arg = hi;
  __syncthreads();
  for (int i = lo + threadIdx.x; i < hi; i += THREADS)
    if (clean(z[i]) == m) { atomicMin(&s_arg, i); break; }
  double sum = 0.0;
  if (temp > 0.f && m > -INFINITY) {
    const double inv_t = 1.0 / (double)temp;
    for (int i = lo + threadIdx.x; i < hi; i += THREADS) sum += weight(clean(z[i]), m, inv_t);
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) all += sums[w];
    p.stats[(int64_t)r * p.chunks + c] = Stat{all, m, s_arg};
  }
}

__global__ void __launch_bounds__(PICK_THREADS) verify_pick_kernel(Verify p) {
  rb_pdl_launch_dependents();
  rb_pdl_wait();
  __shared__ double part[PICK_THREADS];
  __shared__ double s_total, s_before;
  __shared__ float s_max;
  __shared__ int s_row, s_arg, s_owner, s_count, s_last;
  // (rows outside the logits, which only a wrong first_row can name, are left out)
  const int b = blockIdx.x, r0 = min(max(p.first_row[b], 0), p.R), r1 = min(p.first_row[b + 1], p.R);
  const float temp = p.temperature[b];
  const double inv_t = 1.0 / (double)temp;
  int* tokens = p.tokens + (int64_t)b * (p.most + 1);
  for (int j = threadIdx.x; j <= p.most; j += PICK_THREADS) tokens[j] = -1;
  __syncthreads();
  if (threadIdx.x == 0) {
    s_row = -1;
    int n = 0;
    for (int r = r0; r < r1; ++r) {
      const Stat* st = p.stats + (int64_t)r * p.chunks;
      float m = -INFINITY;
      int arg = 0;
      for (int c = 0; c < p.chunks; ++c)
        if (st[c].max > m) { m = st[c].max; arg = st[c].arg; }      // chunks ascend: the lowest of equals
      const bool greedy = !(temp > 0.f && m > -INFINITY);
      double total = 1.0;
      if (!greedy) {
        total = 0.0;
        for (int c = 0; c < p.chunks; ++c)
          if (st[c].max > -INFINITY) total += st[c].sum * weight(st[c].max, m, inv_t);
      }
      const int d = p.drafts[r];
      if (r + 1 < r1 && n < p.most && d >= 0 && d < p.V) {
        const double q = p.probs ? (double)p.probs[(int64_t)r * p.probs_stride + d] : 1.0;
        const double w = greedy ? (d == arg ? 1.0 : 0.0) : weight(clean(p.logits[(int64_t)r * p.stride + d]), m, inv_t);
        if ((double)p.uniforms[2 * (int64_t)r] * q * total < w) {
          tokens[n++] = d;
          continue;
        }
      }
      s_row = r; s_total = total; s_max = m; s_arg = greedy ? arg : -1;
      break;
    }
    p.accepted[b] = n;
    s_count = n;
  }
  __syncthreads();
  const int r = s_row;
  if (r < 0) return;                             // a sequence without rows
  if (s_arg >= 0) {
    if (threadIdx.x == 0) tokens[s_count] = s_arg;
    return;
  }
  const float* z = p.logits + (int64_t)r * p.stride;
  const int d = r + 1 < r1 ? p.drafts[r] : -1;
  const bool judged = d >= 0 && d < p.V;
  const float* q = judged && p.probs ? p.probs + (int64_t)r * p.probs_stride : nullptr;
  const double total = s_total;
  const float m = s_max;
  const int per = (p.V + PICK_THREADS - 1) / PICK_THREADS;
  const int lo = min(p.V, (int)threadIdx.x * per), hi = min(p.V, lo + per);
  // whole: from p itself, where p - q has nothing left
  for (int whole = judged ? 0 : 1; whole < 2; ++whole) {
    auto left = [&](int i) -> double {
      // (p - q) times the sum of the weights: without q nothing is divided, so that equal logits are equal steps exactly
      const double w = weight(clean(z[i]), m, inv_t);
      if (whole) return w;
      if (q) return fmax(w - (double)q[i] * total, 0.0);
      return i == d ? 0.0 : w;
    };
    double mine = 0.0;
    for (int i = lo; i < hi; ++i) mine += left(i);
    part[threadIdx.x] = mine;
    if (threadIdx.x == 0) s_last = -1;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int t = 0; t < PICK_THREADS; ++t) all += part[t];
      const double goal = (double)p.uniforms[2 * (int64_t)r + 1] * all;
      double before = 0.0;
      int owner = -1;
      for (int t = 0; t < PICK_THREADS && owner < 0; ++t) {
        if (before + part[t] > goal) owner = t;
        else before += part[t];
      }
      if (owner < 0)                             // rounding left the goal at the end: the last that has something
        for (int t = PICK_THREADS - 1; t >= 0 && owner < 0; --t)
          if (part[t] > 0.0) { owner = t; before = -1.0; }
      s_owner = owner;
      s_before = before;
      s_total = goal;
    }
    __syncthreads();
    if (s_owner >= 0) {
      if ((int)threadIdx.x == s_owner) {
        double run = s_before;
        int pick = -1;
        for (int i = lo; i < hi; ++i) {
          const double w = left(i);
          if (w > 0.0) pick = i;
          if (s_before >= 0.0) {
            run += w;
            if (run > s_total) break;
          }
        }
        tokens[s_count] = pick;
      }
      return;
    }
    __syncthreads();
  }
}

}  // namespace

// Bytes of scratch for R rows of V logits.
RB_EXPORT long long rb_verify_scratch_bytes(int R, int V) {
  return (long long)R * ((V + CHUNK - 1) / CHUNK) * (long long)sizeof(Stat);
}

RB_EXPORT int rb_verify(int* accepted, int* tokens, const float* logits, int64_t stride, const float* probs, int64_t probs_stride,
                        const int* first_row, const int* drafts, const float* temperature, const float* uniforms, int B, int R, int V,
                        int most, void* scratch, cudaStream_t stream) {
  if (B == 0) return 0;
  RB_REQUIRE(V > 0 && R >= 0 && most >= 0, "rb_verify: %d rows of %d logits, %d drafts", R, V, most);
  Verify p;
  p.accepted = accepted; p.tokens = tokens; p.logits = logits; p.stride = stride; p.probs = probs; p.probs_stride = probs_stride;
  p.first_row = first_row; p.drafts = drafts; p.temperature = temperature; p.uniforms = uniforms; p.stats = (Stat*)scratch;
  p.B = B; p.R = R; p.V = V; p.most = most; p.chunks = (V + CHUNK - 1) / CHUNK;
  if (R > 0) RB_LAUNCH("rb_verify (rows)", (verify_stats_kernel), dim3(R, p.chunks), THREADS, 0, stream, p);
  RB_LAUNCH("rb_verify (pick)", (verify_pick_kernel), B, PICK_THREADS, 0, stream, p);
  return 0;
}
