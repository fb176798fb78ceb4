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
// What decides on a single token is float64: the running sum over 100,000 tokens would move by more than the smallest
// probabilities in float32, another way for every way of cutting it.  But that sum is taken over ONE row a sequence, the row whose
// token is taken; whether a draft is accepted hangs on a row's whole sum, and float32 decides that too unless u q S lies within
// 2^-14 of p S.  So:
//   rows    every row's maximum and float32 sum, a block of threads per 8,192 logits: one pass, 16-byte loads, each logit read once
//   pick    a cluster per sequence.  The drafts in turn (a row whose float32 sum leaves it open is summed again in float64); then
//           the float64 sums of max(p - q, 0) over the blocks' and their warps' shares of the row taken, and the walk into one of them.
// The float32 sum S' is off by less than 2^-14 of itself: a term e^x is off by 2^-22 and by what rounding x = (z - max) / T does,
// 2^-23 |x|, which a term of a weight worth counting (|x| < 40) turns into 2^-17 of it; the sum adds 2^-19 at most (32 terms a thread, in four sums).
// One B200, 64 sequences of 4 drafts over 128,256 logits with the drafter's probabilities: the rows 32 us (164 MB, 5.1 TB/s), the pick 57
// (two rows of weights a sequence, the first for the sum that q is multiplied by: instructions, ten of them float64, and waits); 17 sequences
// of up to 7 certain drafts 11 and 10; one of 4 over 32,000 logits 9.4 in all.
#include "rb_common.cuh"

namespace {

constexpr int CHUNK = 8192, THREADS = 256, PICK_WARPS = 16, PICK_THREADS = PICK_WARPS * 32, MOST_ITEMS = 512;
constexpr double OPEN = 1.0 / 16384;             // float32 decides outside this share of the two sides

struct Stat { float max, sum; int arg, unused; };

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

// exp((z - m) / T) with c = log2(e) / T, 1 at the maximum itself (also where that is infinite): float32 and float64
__device__ __forceinline__ float weight_f32(float z, float m, float c) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((z - m) * c));
  return z == m ? 1.f : y;
}
// In float64 2^x, x = (z - m) c <= 0, is 2^k times 2^(j / 256) from a table (exp2's values, made by every block) times the first
// five terms of the series of e^(r ln 2), |r| <= 1/512 (the first left out is 4e-17 of the result): ten float64 operations.
constexpr int TABLE = 256;
__device__ __forceinline__ double weight(float z, float m, double c, const double* table) {
  const double x = ((double)z - (double)m) * c;  // (no branch: several of these run side by side)
  const double whole = x + 26388279066624.0;     // 1.5 * 2^44: rounds to 256ths, whose number is the low bits
  const double r = x - (whole - 26388279066624.0);
  const int n = __double2loint(whole);
  // ln 2 and its powers over the factorials
  double e = fma(r, 0.00961812910762847716, 0.05550410866482157995);
  e = fma(e, r, 0.24022650695910071233);
  e = fma(e, r, 0.69314718055994530942);
  const double t = table[n & (TABLE - 1)];
  e = fma(e * r, t, t);
  e = __hiloint2double(__double2hiint(e) + ((n >> 8) << 20), __double2loint(e));
  e = x > -1021.0 ? e : 0.0;                     // (also where x is no number)
  return z == m ? 1.0 : e;
}
__device__ __forceinline__ void make_table(double* table) {
  for (int i = threadIdx.x; i < TABLE; i += blockDim.x) table[i] = exp2((double)i / TABLE);
}
__device__ __forceinline__ double inverse_temperature(float temp) { return 1.4426950408889634074 / (double)temp; }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// VEC: rows begin on 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(THREADS) verify_rows_kernel(Verify p) {
  rb_pdl_launch_dependents();
  constexpr int PER = CHUNK / THREADS;
  __shared__ float s_max[THREADS / 32], s_sum[THREADS / 32];
  __shared__ int s_arg[THREADS / 32];
  const int r = blockIdx.x, lo = blockIdx.y * CHUNK, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  rb_pdl_wait();
  const float* z = p.logits + (int64_t)r * p.stride + lo;
  const int n = min(p.V - lo, CHUNK);
  float v[PER];
#pragma unroll
  for (int i = 0; i < PER / 4; ++i) {
    const int at = (i * THREADS + threadIdx.x) * 4;
    if (VEC && at + 4 <= n) {
      const float4 x = *reinterpret_cast<const float4*>(z + at);
      v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = at + j < n ? z[at + j] : -INFINITY;
    }
  }
  // the row's sequence: the last that begins at or before it
  int seq = 0;
  for (int a = 0, b = p.B; a < b;) {
    const int mid = (a + b) >> 1;
    if (p.first_row[mid] <= r) { seq = mid; a = mid + 1; } else { b = mid; }
  }
  const float temp = p.temperature[seq];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = clean(v[i]);
    m = fmaxf(m, v[i]);
  }
  m = rb_warp_max(m);
  if (lane == 0) s_max[warp] = m;
  __syncthreads();
  m = s_max[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) m = fmaxf(m, s_max[w]);
  float sum = 0.f;
  int arg = p.V;
  if (temp > 0.f) {
    if (m > -INFINITY) {
      const float c = (float)inverse_temperature(temp);
      float four[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < PER; ++i) four[i & 3] += weight_f32(v[i], m, c);
      sum = (four[0] + four[1]) + (four[2] + four[3]);
    }
  } else {
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (v[i] == m) arg = lo + ((i >> 2) * THREADS + (int)threadIdx.x) * 4 + (i & 3);
    arg = __reduce_min_sync(0xffffffffu, arg);
  }
  sum = rb_warp_sum(sum);
  if (lane == 0) { s_sum[warp] = sum; s_arg[warp] = arg; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 32; ++w) { sum += s_sum[w]; arg = min(arg, s_arg[w]); }
    p.stats[(int64_t)r * p.chunks + blockIdx.y] = Stat{m, sum, arg, 0};
  }
}

// The block's sum of a value per thread, the same in all of them (sums in a fixed order).
__device__ __forceinline__ double block_sum(double v, double* s) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < PICK_WARPS; ++w) all += s[w];
  return all;
}

// The first of the lanes' values at which the running sum after `before` exceeds `goal`, else the last above zero (else -1); `before` becomes
// the sum ahead of it, and `over` whether it exceeds.  All lanes get the same.
__device__ __forceinline__ int first_over(double v, double goal, double& before, bool& over) {
  const int lane = threadIdx.x & 31;
  double upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const uint32_t past = __ballot_sync(0xffffffffu, before + upto > goal && v > 0.0), some = __ballot_sync(0xffffffffu, v > 0.0);
  over = past != 0;
  const int at = over ? __ffs(past) - 1 : 31 - __clz(some);
  if (at < 0) return -1;
  before += __shfl_sync(0xffffffffu, upto - v, at);
  return at;
}

// A cluster per sequence: block c has logits c * share .. of the row whose token is taken, a warp a PICK_WARPS-th of those, `items` rows of 32.
// The weights are made again for every sum: kept in registers (32 a thread) they make the kernel a straight line of thousands of
// instructions that each run once a warp, and fetching those took 200 us of 64 sequences over 128,256 logits.
__global__ void __launch_bounds__(PICK_THREADS) verify_pick_kernel(Verify p, int blocks) {
  rb_pdl_launch_dependents();
  __shared__ double table[TABLE];
  __shared__ double s_rows[MOST_ITEMS];           // sums of the rows of 32 logits of the warp's share that the token lies in
  __shared__ double s_sums[PICK_WARPS];          // what the block's warps have
  __shared__ double s_shown[2];                  // what the cluster's blocks read
  __shared__ int s_found[PICK_WARPS], s_args[PICK_WARPS];
  __shared__ float s_maxima[PICK_WARPS];
  __shared__ int s_n, s_row, s_arg;
  __shared__ float s_m;
  const int rank = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  make_table(table);
  rb_pdl_wait();
  // (rows outside the logits, which only a wrong first_row can name, are left out)
  const int r0 = min(max(p.first_row[b], 0), p.R), r1 = min(p.first_row[b + 1], p.R);
  const float temp = p.temperature[b];
  const double c = inverse_temperature(temp);
  int* tokens = p.tokens + (int64_t)b * (p.most + 1);
  if (threadIdx.x == 0) { s_n = 0; s_row = -1; s_arg = -1; }
  if (rank == 0)
    for (int j = threadIdx.x; j <= p.most; j += PICK_THREADS) tokens[j] = -1;
  __syncthreads();
  auto total_of = [&](int r, float m) {          // a row's float64 sum, by the whole block
    const float* z = p.logits + (int64_t)r * p.stride;
    double mine = 0.0;
    for (int i = threadIdx.x; i < p.V; i += PICK_THREADS) mine += weight(clean(z[i]), m, c, table);
    return block_sum(mine, s_sums);
  };
  // ---- the drafts, PICK_WARPS rows at a time, a warp each: 1 accepted, 0 not, 2 open
  for (int at = r0; at < r1; at += PICK_WARPS) {
    const int r = at + warp;
    int found = 0, arg = p.V;
    float m = -INFINITY;
    if (r < r1) {
      const Stat* st = p.stats + (int64_t)r * p.chunks;
      for (int i = lane; i < p.chunks; i += 32) m = fmaxf(m, st[i].max);
      m = rb_warp_max(m);
      const bool greedy = !(temp > 0.f && m > -INFINITY);
      double total = 0.0;
      for (int i = lane; i < p.chunks; i += 32) {
        const Stat one = st[i];
        if (greedy) {
          if (one.max == m) arg = min(arg, temp > 0.f ? 0 : one.arg);
        } else if (one.max > -INFINITY) {
          total += (double)one.sum * weight(one.max, m, c, table);
        }
      }
      total = warp_sum(total);
      arg = greedy ? __reduce_min_sync(0xffffffffu, arg) : -1;
      const int d = p.drafts[r];
      if (r + 1 < r1 && r - r0 < p.most && d >= 0 && d < p.V) {
        const double q = p.probs ? (double)p.probs[(int64_t)r * p.probs_stride + d] : 1.0;
        const double left = (double)p.uniforms[2 * (int64_t)r] * q;
        if (greedy) {
          found = left < (d == arg ? 1.0 : 0.0) ? 1 : 0;
        } else {
          const double w = weight(clean(p.logits[(int64_t)r * p.stride + d]), m, c, table), side = left * total;
          found = side * (1.0 + OPEN) < w ? 1 : (side * (1.0 - OPEN) >= w ? 0 : 2);
        }
      }
    }
    if (lane == 0) { s_found[warp] = found; s_args[warp] = arg; s_maxima[warp] = m; }
    __syncthreads();
    int n = 0;
    for (; n < PICK_WARPS && at + n < r1; ++n) {
      int f = s_found[n];
      if (f == 2) {                              // (the same in all threads, and in all blocks of the cluster)
        const int row = at + n, d = p.drafts[row];
        const double q = p.probs ? (double)p.probs[(int64_t)row * p.probs_stride + d] : 1.0;
        const double total = total_of(row, s_maxima[n]);
        f = (double)p.uniforms[2 * (int64_t)row] * q * total < weight(clean(p.logits[(int64_t)row * p.stride + d]), s_maxima[n], c, table) ? 1 : 0;
      }
      if (f == 0) break;
      if (threadIdx.x == 0) {
        if (rank == 0) tokens[at - r0 + n] = p.drafts[at + n];
        ++s_n;
      }
    }
    const bool here = n < PICK_WARPS && at + n < r1;
    if (here && threadIdx.x == 0) { s_row = at + n; s_arg = s_args[n]; s_m = s_maxima[n]; }
    __syncthreads();
    if (here) break;
  }
  const int r = s_row, taken = s_n;
  if (rank == 0 && threadIdx.x == 0) p.accepted[b] = taken;
  if (r < 0) return;                             // a sequence without rows: all blocks of the cluster
  if (s_arg >= 0) {                              // nothing is drawn
    if (rank == 0 && threadIdx.x == 0) tokens[taken] = s_arg;
    return;
  }
  // ---- the token: sums over the blocks' and the warps' shares
  const float* z = p.logits + (int64_t)r * p.stride;
  const int d = r + 1 < r1 && r - r0 < p.most ? p.drafts[r] : -1;
  const bool judged = d >= 0 && d < p.V;
  const float* q = judged && p.probs ? p.probs + (int64_t)r * p.probs_stride : nullptr;
  const float m = s_m;
  const int per_warp = ((p.V + blocks - 1) / blocks + PICK_THREADS - 1) / PICK_THREADS * 32;       // a multiple of 32
  const int lo = (int)min((int64_t)p.V, ((int64_t)rank * PICK_WARPS + warp) * per_warp);
  int turn = 0;
  // the cluster's sum of a block's values, and of those ahead of this block
  auto over_cluster = [&](double v, double& ahead) {
    if (threadIdx.x == 0) s_shown[turn & 1] = v;
    __syncthreads();
    double all = v;
    ahead = 0.0;
    if (blocks > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      all = 0.0;
      for (int x = 0; x < blocks; ++x) {
        uint32_t at;
        double one;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(&s_shown[turn & 1])), "r"(x));
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(one) : "r"(at));
        if (x == rank) ahead = all;
        all += one;
      }
    }
    ++turn;
    return all;
  };
  const int items = per_warp / 32;
  double total = 0.0, ahead = 0.0;
  // (p - q) times the sum of the weights: without q nothing is divided, so that equal logits are equal steps exactly.  `gone`: the token
  // that is certain and was not accepted, or -1.  (A logit that is no number has the weight 0, as minus infinity has.)
  auto left = [&](float zi, float qi, double less) -> double {
    const double v = weight(zi, m, c, table) - (double)qi * less;
    return v > 0.0 ? v : 0.0;
  };
  auto logit = [&](int64_t at, int gone) -> float { return at < p.V && at != gone ? z[at] : -INFINITY; };
  // the sum over the warp's share, a lane's part of it: eight rows of 32 are asked for together
  auto share_sum = [&](int gone) -> double {
    double sum = 0.0;
    for (int i0 = 0; i0 < items; i0 += 8) {
      float zi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) zi[i] = i0 + i < items ? logit(lo + (i0 + i) * 32 + lane, gone) : -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += weight(zi[i], m, c, table);
    }
    return sum;
  };
  auto share_left = [&](double less) -> double {
    double sum = 0.0;
    for (int i0 = 0; i0 < items; i0 += 8) {
      float zi[8], qi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = lo + (i0 + i) * 32 + lane;
        zi[i] = i0 + i < items ? logit(at, -1) : -INFINITY;
        qi[i] = i0 + i < items && at < p.V ? q[at] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += left(zi[i], qi[i], less);
    }
    return sum;
  };
  if (q) total = over_cluster(block_sum(share_sum(-1), s_sums), ahead);
  // whole: from p itself, where p - q has nothing left
  for (int whole = judged ? 0 : 1; whole < 2; ++whole) {
    const float* qs = whole ? nullptr : q;
    const double less = whole ? 0.0 : total;
    const int gone = whole || q ? -1 : d;
    const double mine = qs ? share_left(total) : share_sum(gone);
    const double block = block_sum(mine, s_sums);
    const double all = over_cluster(block, ahead);
    if (!(all > 0.0) && whole == 0) continue;
    const double goal = (double)p.uniforms[2 * (int64_t)r + 1] * all;
    // the block whose share the goal falls into: the sums ahead of the blocks ascend (rounding cannot leave it out: the last block with
    // something ends at `all`, which is above the goal; a number that is not below 1 takes that block too)
    const bool mine_holds = block > 0.0 && ahead + block > goal && !(ahead > goal);
    const bool last_holds = !(all > goal) && block > 0.0 && !(ahead + block < all);
    if (mine_holds || last_holds) {
      double before = ahead;
      bool over;
      // (every warp for itself) the warp whose share holds the goal; then all warps sum that share's rows of 32, and the first finds the
      // row and the token
      const int w = first_over(lane < PICK_WARPS ? s_sums[lane] : 0.0, goal, before, over);
      const int64_t from = ((int64_t)rank * PICK_WARPS + w) * per_warp;
      for (int i = warp; i < items; i += PICK_WARPS) {
        const int64_t at = from + i * 32 + lane;
        const double sum = warp_sum(left(logit(at, gone), qs && at < p.V ? qs[at] : 0.f, less));
        if (lane == 0) s_rows[i] = sum;
      }
      __syncthreads();
      if (warp == 0) {
        int row = -1;
        for (int i0 = 0; i0 < items; i0 += 32) {
          double upto = before;
          const double v = i0 + lane < items ? s_rows[i0 + lane] : 0.0;
          const int y = first_over(v, goal, upto, over);
          if (y >= 0) { row = i0 + y; ahead = upto; }
          if (over) break;
          before += warp_sum(v);
        }
        const int64_t at = from + row * 32;
        const int y = row >= 0 ? first_over(left(logit(at + lane, gone), qs && at + lane < p.V ? qs[at + lane] : 0.f, less), goal, ahead, over) : -1;
        if (lane == 0) tokens[taken] = y >= 0 ? (int)at + y : -1;
      }
    }
    break;
  }
  if (blocks > 1) {                              // nobody's shared memory goes away while another block reads it
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
  RB_REQUIRE(V <= 8 * PICK_THREADS * MOST_ITEMS, "rb_verify: %d logits a row, %d at most", V, 8 * PICK_THREADS * MOST_ITEMS);
  RB_REQUIRE(V > 0 && R >= 0 && most >= 0 && B <= 65535, "rb_verify: %d sequences, %d rows of %d logits, %d drafts", B, R, V, most);
  Verify p;
  p.accepted = accepted; p.tokens = tokens; p.logits = logits; p.stride = stride; p.probs = probs; p.probs_stride = probs_stride;
  p.first_row = first_row; p.drafts = drafts; p.temperature = temperature; p.uniforms = uniforms; p.stats = (Stat*)scratch;
  p.B = B; p.R = R; p.V = V; p.most = most; p.chunks = (V + CHUNK - 1) / CHUNK;
  if (R > 0) {
    const bool vec = stride % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    if (vec) RB_LAUNCH("rb_verify (rows)", (verify_rows_kernel<true>), dim3(R, p.chunks), THREADS, 0, stream, p);
    else RB_LAUNCH("rb_verify (rows)", (verify_rows_kernel<false>), dim3(R, p.chunks), THREADS, 0, stream, p);
  }
  // blocks of a cluster: 8 logits a thread or more, 8 blocks at most
  int blocks = 1;
  while (blocks < 8 && V > 8 * PICK_THREADS * blocks) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, B, 1);
  cfg.blockDim = dim3(PICK_THREADS, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = rb_pdl_enabled() ? 2 : 1;
  RB_CUDA(cudaLaunchKernelEx(&cfg, verify_pick_kernel, p, blocks));
  return 0;
}
