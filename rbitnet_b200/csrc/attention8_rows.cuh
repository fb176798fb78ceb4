// Attention over the cache held in 8 bits for few rows a sequence: a decode step, drafted tokens.
//
// One block of four warps works for ONE kv head and a tile of at most 8 NT rows, (token, query head) pairs of one sequence whose heads
// share the kv head, over a range of its keys in tiles of 64 (a page, or an aligned part of one: one scale each of keys and of
// values).  A warp takes 32 keys of every other tile at a time and keeps a softmax of its own; the warps are joined at the end.
//
// The products are mma.sync m16n8k16 in float16 with the KEYS as the 16 rows of the first, and the head's values as the 16 rows of the
// second, so that eight query rows fill an instruction:
//     S^T[16 keys, 8 rows] = K[16, D] Q^T           O^T[D, 8 rows] += V^T[D, 16 keys] P^T[16 keys, 8 rows]
// A code is a float16 value (cvt, exactly), so neither product rounds its operands but P, to float16 (below; sums are float32);
// Q, bfloat16, is brought to the middle of float16's range by a power of two a row.  The order of a product's inner index
// and of its rows is free as long as both sides agree, and it is chosen so that every operand register is made of whole 16-byte pieces of
// the cache as they lie: of keys g and g + 8 the pieces 16 t .. 16 t + 15 of every 64 values, of values 2t, 2t + 1, 2t + 8, 2t + 9 the pieces
// D/8 g .. (lane = 4 g + t): no shuffle and no transposing load between the cache's bytes and the products.
// A warp has a ring of its own in shared memory, filled by TMA (two boxes of 32 positions, 128-byte swizzle, no bank conflicts) and waited
// for at its own barriers: the warps of a block meet only at the end.
//
// What a sum is made of is a weight times its values' scale, and either may be small where the other is large.  So the sum of weights goes by
// a row's largest score m (base-2 units), but O by r, the logarithm of the largest weight 2^(score - m) times scale so far: the second
// product's operand is P' = 2^(score - m) scale 2^(7 - r), rounded to float16, and O is kept times 2^(7 - r).  Both follow lazily, moved only where
// they have been passed by more than 8, so that P' is 2^15 at most.  Rounding leaves a P' within 2^-11 of itself where weight times
// scale is 2^-21 of the largest or more, and within 2^-32 of the largest below that.  (A tile's largest weight counts as 2^-96 at least for r,
// so that 2^(7 - r) scale is a float32 number, as the weights are: 2^-126 of the largest and less is 0.)
//
// Ranges of keys: in a small grid the parts of a (tile, kv head) are a thread-block cluster and merge on chip.  In a larger one
// all tiles of keys of all (row tile, kv head) pairs, in order, are dealt out evenly to the blocks, whatever the sequences' lengths; a
// pair that several blocks have worked on is merged by a second kernel.  Where pairs are many and short a pair is one warp's work.
//
// Bounded by the cache's bytes where sequences are long: one B200, 64 sequences of up to 8,000 positions, 32 heads on 8 kv heads of 128:
// 541 MB in 90 us within a captured graph and 96 called from Python, 6.0 and 5.7 TB/s (0.92 and 0.86 of a copy).  Short pairs are bound by what
// a pair costs to begin and to join (about 5 us in a block, two blocks an SM) or, a pair a warp, by a warp's chain from score to sum, a
// microsecond for 32 keys: 24 sequences of 32 heads with a window of 1,024, 202 MB in 43 us, 4.7 TB/s.  More rows add products and exponentials:
// 16 sequences of up to five tokens at up to 6,001 positions, 20 rows, 101 MB in 41 us.  One sequence at 2,048 positions: 8 us, waits.
// Measured beside an earlier form (the first of these, 91 us): 16-byte cp.async by every thread 154 us, of which the copies alone 136; boxes of 16 positions
// 126 to 136; two stages and three blocks an SM 109; pairs dealt out without what their beginnings cost 113.
#pragma once

#include "attention8.cuh"

#include <cuda_fp16.h>

RB_CHECK_READER(attention8_rows)

namespace rows8 {

constexpr int WARPS = 4, TILE = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FLOOR = -3.4028234663852886e38f;  // a maximum of nothing: -inf but for differences, which are numbers
constexpr float UP = 7.f, SLACK = 8.f, LEAST = -96.f;

struct Params {
  Params8 a;
  const int* tile_tok0;       // null: row tile i is row i alone
  const int* tile_ntok;
  int n_tiles, Kh, G;
  int parts;                  // > 0: the parts of a pair are a cluster; 0: the tiles are dealt out to gridDim.x blocks; -2, -3: a pair is a warp's, so many stages
  int least;                  // dealt out: tiles of a block, at least
  float4* part_o;             // dealt out: [blocks + pairs][NT][D / 16][lane], what the accumulators of a lane hold, and
  float2* part_ml;            // [blocks + pairs][8 NT] (maximum in base-2 units, sum)
};

// two codes (the low 16 bits, or the high ones) as two float16 values
__device__ __forceinline__ uint32_t half2_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t half2_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit values, a row's pair per lane, turned over its diagonal
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// N: stages of a warp's ring.
template <int D, int NT, int N = 3> struct Shape {
  static constexpr int KG = 2;                            // groups of 16 keys of a tile that a warp takes at a time
  static constexpr int CHUNK = KG * 16 * D;               // bytes of their codes, of keys and of values each
  static constexpr int STAGE = 2 * CHUNK;                 // of a warp
  static constexpr int NS = N;
  static constexpr int ROWS = 8 * NT;
  static constexpr bool Q_SHARED = NT >= 3;               // the query operands lie in shared memory, not in registers
  static constexpr int Q_BYTES = Q_SHARED ? (D / 16) * NT * 256 : 0;
  static constexpr int MT = D / 16;                       // accumulators' row tiles
  static constexpr int QT = MT / WARPS;                   // of them that a warp joins and hands on
  static constexpr int RING = WARPS * NS * STAGE;
  static constexpr int OFF_Q = RING;
  static constexpr int OFF_ML = OFF_Q + Q_BYTES;                        // [warp][row] maximum and sum; then of the block, [row]
  static constexpr int OFF_AT = OFF_ML + (WARPS + 1) * ROWS * 8;        // [warp] the stage that its accumulators begin in
  static constexpr int OFF_BAR = OFF_AT + 16;
  static constexpr int BYTES = OFF_BAR + WARPS * NS * 8 + 1024;         // + room to align
  static constexpr int LEFT = STAGE / (MT * 512);         // eights of rows whose accumulators a stage holds
  static constexpr int AHEAD = NS - (NT + LEFT - 1) / LEFT;             // stages of the next pair filled while a pair's warps are joined
  static_assert(N < 3 || AHEAD >= 1, "a warp leaves its accumulators in its own ring");
  static_assert(NT * MT * 512 <= RING, "what the cluster's other blocks read, over the ring");
};

// The block's sums of a pair: of every eight rows, row tiles WARP * QT .. of O^T as this lane's accumulators (rows 2t, 2t + 1), maxima and sums.
template <int D, int NT> struct Joined {
  float4 o[NT][Shape<D, NT>::QT];
  float m[NT][2], l[NT][2];
};

// A warp's ring between two pairs: copies asked for and copies used, whose numbers say the stage and its barrier's phase.
struct Ring { uint32_t asked, used; bool failed; };

// Where a thread's pieces lie in a warp's 32 keys (or values), rows of 128 bytes whose 16-byte pieces are exchanged by the row's low three
// bits (the 128-byte swizzle of the box): of key `first` + 8 r + g the piece j, and of value `first` + 2t + (0, 1, 8, 9)[k] the bytes D/8 g.
template <int D> __device__ __forceinline__ int key_place(int first, int r, int j, int g, int t) {
  if (D == 128) return (first + 8 * r + g) * 128 + (((4 * j + t) ^ g) << 4);
  return (first / 2 + 4 * r + (g >> 1)) * 128 + (((4 * (g & 1) + t) ^ (4 * r + (g >> 1))) << 4);
}
template <int D> __device__ __forceinline__ int value_place(int first, int k, int g, int t) {
  if (D == 128) return (first + 2 * t + (k & 1) + 8 * (k >> 1)) * 128 + ((g ^ (2 * t + (k & 1))) << 4);
  return (first / 2 + t + 4 * (k >> 1)) * 128 + (((4 * (k & 1) + (g >> 1)) ^ (t + 4 * (k >> 1))) << 4) + 8 * (g & 1);
}

// what a block does for one pair: tiles first .. last - 1 of the visited ones
struct Segment { int tile, kvh, first, last, visited; };

// the row tile's sequence: where its rows and its keys are
struct Where {
  int tok0, ntok, slot, pos0, key_lo, key_hi;
  __device__ __forceinline__ Where(const Params& p, int tile) {
    tok0 = p.tile_tok0 ? p.tile_tok0[tile] : tile;
    ntok = p.tile_ntok ? p.tile_ntok[tile] : 1;
    slot = p.a.tok_slot[tok0];
    pos0 = p.a.tok_pos[tok0];
    key_hi = pos0 + ntok - 1;
    key_lo = p.a.window > 0 ? max(0, pos0 - p.a.window + 1) : 0;
  }
};
__device__ __forceinline__ int visited_tiles(const Params& p, int tile) {
  const Where w(p, tile);
  return RbKeyTiles(w.key_lo, w.key_hi, p.a.keep, TILE).n;
}

// A warp's way through a segment: where the sequence lies, the tiles that it asks for next and their pages, scales of the tiles on their way.
// The positions, slots and page tables were written before the step began: `Job` may be made before the wait, `ask` not.
// It counts in units of 32 keys: of every other tile the warp's half, or (ALONE > 0: a pair is one warp's work, with a ring of so many stages)
// all halves in turn.
template <int D, int NT, int ALONE = 0> struct Job {
  using S = Shape<D, NT, ALONE ? ALONE : 3>;
  static constexpr int KEYS = 16 * S::KG, SHARES = TILE / KEYS, STEP = ALONE ? 1 : WARPS / SHARES;
  Segment seg;
  Where w;
  RbKeyTiles tiles;
  int begin, end, next;            // units; the one that is asked for next
  int page[S::NS];                 // pages of units next, next + STEP, ...
  float2 scales[S::NS - 1];        // of the units on their way (keys, values)
  __device__ __forceinline__ Job(const Params& p, const Segment& s)
      : seg(s), w(p, s.tile), tiles(w.key_lo, w.key_hi, p.a.keep, TILE) {
    const int warp = threadIdx.x >> 5;
    begin = next = ALONE ? seg.first * SHARES : seg.first + warp / SHARES;
    end = ALONE ? seg.last * SHARES : seg.last;
#pragma unroll
    for (int i = 0; i < S::NS; ++i) page[i] = page_of(p, next + i * STEP);
  }
  __device__ __forceinline__ int tile_of(int unit) const { return tiles.at(ALONE ? unit / SHARES : unit); }
  __device__ __forceinline__ int in_tile(int unit) const { return (ALONE ? unit % SHARES : (int)(threadIdx.x >> 5) % SHARES) * KEYS; }
  __device__ __forceinline__ int page_of(const Params& p, int unit) const {
    if (unit >= end) return 0;
    const int tile = tile_of(unit), per = p.a.cache.page_size / TILE;
#ifdef RB_CHECKED
    return (int)(rb_page_offset(p.a.cache, w.slot, tile * TILE, seg.kvh) / ((int64_t)p.Kh * p.a.cache.page_size * D));
#endif
    return p.a.cache.page_table[(int64_t)w.slot * p.a.cache.max_pages + (per == 1 ? tile : tile / per)];
  }
  // The next unit's codes on their way, and its scales (place i of the queue); nothing of one that lies behind the sequence.
  __device__ __forceinline__ void ask(const Params& p, const CUtensorMap* tmK, const CUtensorMap* tmV, uint8_t* stages, uint64_t* full,
                                      Ring& ring, int i) {
    const int kt = next, at = page[0];
    next += STEP;
#pragma unroll
    for (int j = 0; j + 1 < S::NS; ++j) page[j] = page[j + 1];
    page[S::NS - 1] = page_of(p, next + (S::NS - 1) * STEP);
    scales[i] = make_float2(1.f, 1.f);
    if (kt >= end || ring.failed) return;
    const int tile = tile_of(kt), in = in_tile(kt);
    if (tile * TILE + in > w.key_hi) return;
    const int per = p.a.cache.page_size / TILE;
    const int unit = (at * p.Kh + seg.kvh) * per + (per == 1 ? 0 : tile % per);     // the block's number in the pool
    const uint32_t s = ring.asked % S::NS;
    if (elect_one()) {
      mbar_expect_tx(&full[s], S::STAGE);
      const int row = (int)(((int64_t)unit * TILE + in) * D / 128);            // of 128 bytes
      tma_load_2d(stages + s * S::STAGE, tmK, 0, row, &full[s]);
      tma_load_2d(stages + s * S::STAGE + S::CHUNK, tmV, 0, row, &full[s]);
    }
    __syncwarp();
    ++ring.asked;
    scales[i] = make_float2(p.a.k_scale[unit], p.a.v_scale[unit]);
  }
};

// A warp's sums: O^T and what it is to be multiplied by, maxima in base-2 units, this lane's part of the sums of the weights; rows 2t, 2t + 1 of
// every eight.
template <int D, int NT> struct Sums {
  float o[NT][D / 16][4], by[NT][2], m[NT][2], l[NT][2];
};

// The warp's way through a segment, whose first S::NS - 1 units have been asked for.
// ONE: every row tile is a single token, so that its rows see the same keys (the code for a NaN that only some see,
// though not run there, cost such steps 94 -> 101 us where tiles are dealt out; the other kernels were not tried without it).
template <int D, int NT, int ALONE, bool ONE = false>
__device__ __forceinline__ void run(const Params& p, const CUtensorMap* tmK, const CUtensorMap* tmV, Job<D, NT, ALONE>& job, uint8_t* smem,
                                    uint8_t* stages, uint64_t* full, Ring& ring, Sums<D, NT>& sums) {
  using S = typename Job<D, NT, ALONE>::S;
  constexpr int KG = S::KG, KP = D / 64, MT = D / 16, VW = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Where w = job.w;
  const Segment seg = job.seg;
  const int kvh = seg.kvh, G = p.G, H = p.a.H, n_rows = w.ntok * G;

  // ---- the query rows as B operands: of row g of every eight, values 64 j + 16 t + 4 i + (0, 1) and (2, 3)
  uint32_t qf[S::Q_SHARED ? 1 : MT][S::Q_SHARED ? 1 : NT][2];
  uint2* q_shared = reinterpret_cast<uint2*>(smem + S::OFF_Q) + lane;
  float factor[NT][2];             // of rows 2t, 2t + 1: what a score is multiplied by, in base-2 units
  int pos[NT][2];                  // their positions (-1: no such row)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    const bool in = r < n_rows;
    uint32_t raw[KP][8];
    const __nv_bfloat16* src = p.a.q + ((int64_t)(w.tok0 + (in ? r / G : 0)) * H + kvh * G + (in ? r % G : 0)) * D;
    uint32_t big = 0;              // the largest exponent (and mantissa) among the row's values
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v = in ? *reinterpret_cast<const uint4*>(src + 64 * j + 16 * t + 8 * h) : make_uint4(0, 0, 0, 0);
        raw[j][4 * h] = v.x; raw[j][4 * h + 1] = v.y; raw[j][4 * h + 2] = v.z; raw[j][4 * h + 3] = v.w;
      }
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) big = max(big, max(raw[j][i] << 16 & 0x7fff0000u, raw[j][i] & 0x7fff0000u));
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // the row's largest value becomes 2^8 .. 2^9; rows of zeros, infinities or NaN as they are
    const int e = max((int)(big >> 23) - 127 - 8, -100);
    const bool plain = big == 0 || big >= 0x7f800000u;
    const float up = plain ? 1.f : __uint_as_float((uint32_t)(127 - e) << 23), down = plain ? 1.f : __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t two[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = raw[j][2 * i + h];
          two[h] = pack_half2(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xffff0000u) * up);
        }
        if (S::Q_SHARED) {
          if (warp == n % WARPS) q_shared[((4 * j + i) * NT + n) * 32] = make_uint2(two[0], two[1]);
        } else {
          qf[4 * j + i][n][0] = two[0];
          qf[4 * j + i][n][1] = two[1];
        }
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      factor[n][c] = __shfl_sync(0xffffffffu, down, (2 * t + c) * 4) * p.a.scale * (p.a.softcap > 0.f ? 1.f : LOG2E);
      const int rc = n * 8 + 2 * t + c;
      pos[n][c] = rc < n_rows ? w.pos0 + rc / G : -1;
    }
  }
  if (S::Q_SHARED) __syncthreads();

  auto& o = sums.o;
  auto& m = sums.m;
  auto& l = sums.l;
  float r[NT][2];                  // the logarithm of the largest weight times scale
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = r[n][c] = FLOOR;
      l[n][c] = 0.f;
      const int rc = n * 8 + 2 * t + c;
      if (p.a.sinks != nullptr && seg.first == 0 && seg.last > 0 && (ALONE || warp == 0) && rc < n_rows) {     // counted once: by the part with the first tile
        const float sink = p.a.sinks[kvh * G + rc % G] * LOG2E;
        m[n][c] = sink != sink ? sink : fminf(fmaxf(sink, FLOOR), -FLOOR);
        l[n][c] = g == 0 ? 1.f : 0.f;
      }
    }
  }

  for (int kt = job.begin; kt < job.end && !ring.failed; kt += job.STEP) {
    const float2 scales = job.scales[0];
#pragma unroll
    for (int i = 0; i + 2 < S::NS; ++i) job.scales[i] = job.scales[i + 1];
    job.ask(p, tmK, tmV, stages, full, ring, S::NS - 2);
    const int key0 = job.tile_of(kt) * TILE + job.in_tile(kt);
    if (key0 > w.key_hi) continue;
    const uint32_t stage = ring.used % S::NS;
    if (!mbar_wait_warp(&full[stage], (ring.used / S::NS) & 1, 15)) {
      ring.failed = true;              // the error word says so; the other copies on their way are waited for, with a limit too
      while (++ring.used != ring.asked) (void)mbar_wait_warp(&full[ring.used % S::NS], (ring.used / S::NS) & 1, 15);
      break;
    }
    ++ring.used;
    const uint8_t* at = stages + stage * S::STAGE;
    // ---- S^T = K Q^T
    float s[KG][NT][4];
#pragma unroll
    for (int u = 0; u < KG; ++u)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
    for (int j = 0; j < KP; ++j) {
      uint32_t wa[KG][4], wb[KG][4];
#pragma unroll
      for (int u = 0; u < KG; ++u) {
        const uint4 ka = *reinterpret_cast<const uint4*>(at + key_place<D>(16 * u, 0, j, g, t));
        const uint4 kb = *reinterpret_cast<const uint4*>(at + key_place<D>(16 * u, 1, j, g, t));
        wa[u][0] = ka.x; wa[u][1] = ka.y; wa[u][2] = ka.z; wa[u][3] = ka.w;
        wb[u][0] = kb.x; wb[u][1] = kb.y; wb[u][2] = kb.z; wb[u][3] = kb.w;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t q[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (S::Q_SHARED) {
            const uint2 two = q_shared[((4 * j + x) * NT + n) * 32];
            q[n][0] = two.x; q[n][1] = two.y;
          } else {
            q[n][0] = qf[4 * j + x][n][0]; q[n][1] = qf[4 * j + x][n][1];
          }
        }
#pragma unroll
        for (int u = 0; u < KG; ++u) {
          const uint32_t a0 = half2_lo(wa[u][x]), a1 = half2_lo(wb[u][x]), a2 = half2_hi(wa[u][x]), a3 = half2_hi(wb[u][x]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[u][n], a0, a1, a2, a3, q[n][0], q[n][1]);
        }
      }
    }
    // ---- scores in base-2 units (rows 2t, 2t + 1; keys g, g + 8 of every 16); the mask only where a row sees less than all
    const bool whole = key0 + 16 * KG - 1 <= w.pos0 && (p.a.window <= 0 || key0 >= w.key_hi - p.a.window + 1);
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float f = factor[n][c] * scales.x;
        float x = -INFINITY;
#pragma unroll
        for (int u = 0; u < KG; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& v = s[u][n][c + 2 * h];
            v *= f;
            x = fmaxf(x, v);
          }
        top[n][c] = x;
      }
    if (!whole || p.a.softcap > 0.f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = -INFINITY;
#pragma unroll
          for (int u = 0; u < KG; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float& v = s[u][n][c + 2 * h];
              if (p.a.softcap > 0.f) v = p.a.softcap * tanhf(v / p.a.softcap) * LOG2E;
              const int key = key0 + 16 * u + g + 8 * h, q = pos[n][c];
              if (key > q || (p.a.window > 0 && key <= q - p.a.window && key >= p.a.keep)) v = -INFINITY;
              x = fmaxf(x, v);
            }
          top[n][c] = x;
        }
    }
    // the values' scale as 2^at_scale x mantissa (a power of two but for a block that nothing was appended to, whose scale may be 0)
    const int exponent = (int)(__float_as_uint(scales.y) >> 23);
    const float at_scale = (float)(exponent - 127), mantissa = scales.y * __uint_as_float((uint32_t)(254 - exponent) << 23);
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) moved |= fmaxf(top[n][c] - m[n][c], LEAST) > fminf(r[n][c] + (SLACK - at_scale), SLACK);
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float corr[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = top[n][c];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          if (x - m[n][c] > SLACK) {
            l[n][c] *= exp2f(m[n][c] - x);
            r[n][c] += m[n][c] - x;
            m[n][c] = x;
          }
          const float y = fmaxf(x - m[n][c], LEAST) + at_scale;
          corr[c] = 1.f;
          if (y > r[n][c] + SLACK) {
            corr[c] = exp2f(r[n][c] - y);
            r[n][c] = y;
          }
        }
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          o[n][u][0] *= corr[0]; o[n][u][2] *= corr[0];
          o[n][u][1] *= corr[1]; o[n][u][3] *= corr[1];
        }
      }
    }
    // ---- P, its sums, and P^T as the B operand
    uint32_t pf[KG][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float m0 = m[n][0], m1 = m[n][1];
      const float f0 = exp2_fast(UP + at_scale - r[n][0]) * mantissa, f1 = exp2_fast(UP + at_scale - r[n][1]) * mantissa;
#pragma unroll
      for (int u = 0; u < KG; ++u) {
        const float p0 = exp2_fast(s[u][n][0] - m0), p1 = exp2_fast(s[u][n][1] - m1);
        const float p2 = exp2_fast(s[u][n][2] - m0), p3 = exp2_fast(s[u][n][3] - m1);
        l[n][0] += p0 + p2;
        l[n][1] += p1 + p3;
        pf[u][n][0] = transposed(pack_half2(p0 * f0, p1 * f1));
        pf[u][n][1] = transposed(pack_half2(p2 * f0, p3 * f1));
      }
    }
    // ---- O^T += V^T P^T: of keys 2t, 2t + 1, 2t + 8, 2t + 9 the bytes 2u (row g) and 2u + 1 (row g + 8)
#pragma unroll
    for (int u = 0; u < KG; ++u) {
      uint32_t v[4][VW];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* src = at + S::CHUNK + value_place<D>(16 * u, k, g, t);
        if constexpr (VW == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(src);
          v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(src);
          v[k][0] = x.x; v[k][1] = x.y;
        }
      }
      if (!whole) {                // a key that no row sees may hold anything: NaN times a weight of zero would stay
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = key0 + 16 * u + 2 * t + (k & 1) + (k >> 1) * 8;
          if (key > w.key_hi || (key < w.key_lo && key >= p.a.keep)) {
#pragma unroll
            for (int x = 0; x < VW; ++x) v[k][x] = 0u;
          }
        }
      }
      // (a NaN among values that some of the tile's tokens see and others do not would stay in the others' rows: a token at a time then)
      if (!ONE && !whole && w.ntok > 1) {
        uint32_t nan = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int x = 0; x < VW; ++x) nan |= ((v[k][x] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (__any_sync(0xffffffffu, nan != 0)) {
#pragma unroll 1
          for (int q = w.pos0; q <= w.key_hi; ++q) {
            uint32_t seen[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int key = key0 + 16 * u + 2 * t + (k & 1) + (k >> 1) * 8;
              seen[k] = key > q || (p.a.window > 0 && key <= q - p.a.window && key >= p.a.keep) ? 0u : 0xffffffffu;
            }
#pragma unroll
            for (int x = 0; x < VW; ++x)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t ab = __byte_perm(v[0][x] & seen[0], v[1][x] & seen[1], y == 0 ? 0x5140 : 0x7362);
                const uint32_t cd = __byte_perm(v[2][x] & seen[2], v[3][x] & seen[3], y == 0 ? 0x5140 : 0x7362);
                const uint32_t a0 = half2_lo(ab), a1 = half2_hi(ab), a2 = half2_lo(cd), a3 = half2_hi(cd);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  float (&to)[4] = o[n][2 * x + y];
                  float sum[4] = {to[0], to[1], to[2], to[3]};
                  mma_f16(sum, a0, a1, a2, a3, pf[u][n][0], pf[u][n][1]);
#pragma unroll
                  for (int c = 0; c < 4; ++c) to[c] = pos[n][c & 1] == q ? sum[c] : to[c];
                }
              }
          }
          continue;
        }
      }
#pragma unroll
      for (int x = 0; x < VW; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t ab = __byte_perm(v[0][x], v[1][x], y == 0 ? 0x5140 : 0x7362);
          const uint32_t cd = __byte_perm(v[2][x], v[3][x], y == 0 ? 0x5140 : 0x7362);
          const uint32_t a0 = half2_lo(ab), a1 = half2_hi(ab), a2 = half2_lo(cd), a3 = half2_hi(cd);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * x + y], a0, a1, a2, a3, pf[u][n][0], pf[u][n][1]);
        }
    }
    __syncwarp();                    // everybody has left this stage: it may be filled again
  }

#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) sums.by[n][c] = exp2f(r[n][c] - UP);
}

// The block's part of a pair, whose first S::AHEAD units have been asked for; `then` asks for those of the pair after it.
template <int D, int NT, bool ONE, typename F>
__device__ __forceinline__ void work(const Params& p, const CUtensorMap* tmK, const CUtensorMap* tmV, Job<D, NT>& job, uint8_t* smem,
                                     Ring& ring, Joined<D, NT>& joined, F then) {
  using S = Shape<D, NT>;
  constexpr int MT = S::MT, ROWS = S::ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* stages = smem + warp * S::NS * S::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR) + warp * S::NS;
#pragma unroll
  for (int i = S::AHEAD; i < S::NS - 1; ++i) job.ask(p, tmK, tmV, stages, full, ring, i);
  Sums<D, NT> sums;
  run<D, NT, 0, ONE>(p, tmK, tmV, job, smem, stages, full, ring, sums);
  auto& o = sums.o;
  auto& m = sums.m;
  auto& l = sums.l;
  auto& by = sums.by;
  // ---- the next pair's first tiles, which arrive meanwhile; then the four warps: each leaves its accumulators, as its lanes hold them,
  // in those stages of its own ring that are not being filled, and takes a quarter of the row tiles from all
  const uint32_t beside = ring.asked + S::AHEAD;
  then(stages, full);
  float2* ml = reinterpret_cast<float2*>(smem + S::OFF_ML);
  uint32_t* places = reinterpret_cast<uint32_t*>(smem + S::OFF_AT);
  // (of warp x, the accumulators of the n-th eight)
  auto left = [&](int x, uint32_t from, int n) {
    return reinterpret_cast<float4*>(smem + (x * S::NS + (from + n / S::LEFT) % S::NS) * S::STAGE) + n % S::LEFT * (MT * 32) + lane;
  };
  if (lane == 0) places[warp] = beside;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float4* to = left(warp, beside, n);
#pragma unroll
    for (int u = 0; u < MT; ++u) to[u * 32] = make_float4(o[n][u][0] * by[n][0], o[n][u][1] * by[n][1], o[n][u][2] * by[n][0], o[n][u][3] * by[n][1]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = l[n][c];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) ml[warp * ROWS + n * 8 + 2 * t + c] = make_float2(m[n][c], sum);
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float f[WARPS][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float2 of[WARPS];
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < WARPS; ++x) {
        of[x] = ml[x * ROWS + n * 8 + 2 * t + c];
        top = fmaxf(top, of[x].x);
      }
      const float use = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < WARPS; ++x) {
        f[x][c] = exp2_fast(of[x].x - use);
        sum += of[x].y * f[x][c];
      }
      joined.m[n][c] = top;
      joined.l[n][c] = sum;
    }
#pragma unroll
    for (int u = 0; u < S::QT; ++u) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < WARPS; ++x) {
        const float4 v = left(x, places[x], n)[(warp * S::QT + u) * 32];
        acc.x += v.x * f[x][0]; acc.y += v.y * f[x][1];
        acc.z += v.z * f[x][0]; acc.w += v.w * f[x][1];
      }
      joined.o[n][u] = acc;
    }
  }
  fence_async_shared();              // (the ring is filled by copies again, after the block's next barrier)
  __syncthreads();
}

// Values d, d + 1 of rows 2t, 2t + 1 of the n-th eight, unnormalised, with the rows' sums: d = D/8 g + 2u for row tile u of O^T.
template <int D>
__device__ __forceinline__ void store(const Params& p, const Where& w, int kvh, int n, int u, int lane, const float4& o, const float (&l)[2]) {
  const int d = D / 8 * (lane >> 2) + 2 * u;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = n * 8 + 2 * (lane & 3) + c;
    if (r < w.ntok * p.G) {
      const float inv = 1.0f / l[c];
      __nv_bfloat16* dst = p.a.out + ((int64_t)(w.tok0 + r / p.G) * p.a.H + kvh * p.G + r % p.G) * D + d;
      *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn((c ? o.y : o.x) * inv, (c ? o.w : o.z) * inv);
    }
  }
}
template <int D, int NT>
__device__ __forceinline__ void store(const Params& p, const Where& w, int kvh, const Joined<D, NT>& j) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < Shape<D, NT>::QT; ++u) store<D>(p, w, kvh, n, warp * Shape<D, NT>::QT + u, lane, j.o[n][u], j.l[n]);
}

// Another part joins the sums so far of rows 2t, 2t + 1 (`of`: its maximum and sum for both).
__device__ __forceinline__ void add_part(float4& acc, float (&m)[2], float (&l)[2], const float4& o, const float4& of) {
  float f[2], k[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float mz = c ? of.z : of.x, top = fmaxf(m[c], mz), use = top == -INFINITY ? 0.f : top;
    k[c] = exp2_fast(m[c] - use);
    f[c] = exp2_fast(mz - use);
    l[c] = l[c] * k[c] + (c ? of.w : of.y) * f[c];
    m[c] = top;
  }
  acc.x = acc.x * k[0] + o.x * f[0]; acc.y = acc.y * k[1] + o.y * f[1];
  acc.z = acc.z * k[0] + o.z * f[0]; acc.w = acc.w * k[1] + o.w * f[1];
}

// The warps' barriers; what follows is ordered by the caller's or the first barrier of the block.
template <typename S> __device__ __forceinline__ void begin(uint8_t* smem) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < WARPS * S::NS; ++i) mbar_init(reinterpret_cast<uint64_t*>(smem + S::OFF_BAR) + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  __syncthreads();
}

template <int D, int NT>
__global__ void __launch_bounds__(WARPS * 32) cluster_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, Params p) {
  rb_pdl_launch_dependents();
  using S = Shape<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  begin<S>(smem);
  Ring ring{0, 0, false};
  Segment seg;
  seg.tile = blockIdx.x; seg.kvh = blockIdx.y;
  seg.visited = visited_tiles(p, seg.tile);
  seg.first = (int)((int64_t)blockIdx.z * seg.visited / p.parts);
  seg.last = (int)((int64_t)(blockIdx.z + 1) * seg.visited / p.parts);
  Job<D, NT> job(p, seg);
  rb_pdl_wait();
  {
    uint8_t* stages = smem + (threadIdx.x >> 5) * S::NS * S::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR) + (threadIdx.x >> 5) * S::NS;
#pragma unroll
    for (int i = 0; i < S::AHEAD; ++i) job.ask(p, &tmK, &tmV, stages, full, ring, i);
  }
  Joined<D, NT> mine;
  work<D, NT, false>(p, &tmK, &tmV, job, smem, ring, mine, [](uint8_t*, uint64_t*) {});
  const Where& w = job.w;
  if (p.parts == 1) {
    store<D, NT>(p, w, seg.kvh, mine);
    return;
  }
  // what the cluster's other blocks read, over the ring
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float4* sO = reinterpret_cast<float4*>(smem);
  float2* sML = reinterpret_cast<float2*>(smem + S::OFF_ML) + WARPS * S::ROWS;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int u = 0; u < S::QT; ++u) sO[(n * S::MT + warp * S::QT + u) * 32 + lane] = mine.o[n][u];
    if (warp == 0 && lane < 4) {
      sML[n * 8 + 2 * lane] = make_float2(mine.m[n][0], mine.l[n][0]);
      sML[n * 8 + 2 * lane + 1] = make_float2(mine.m[n][1], mine.l[n][1]);
    }
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // every block finishes a share of the lanes' accumulators from all parts, in part order
  for (int idx = (int)blockIdx.z * WARPS * 32 + threadIdx.x; idx < NT * S::MT * 32; idx += p.parts * WARPS * 32) {
    const int n = idx / (S::MT * 32), u = idx / 32 % S::MT, row = n * 8 + 2 * (idx & 3);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int z0 = 0; z0 < p.parts; z0 += 4) {
      float4 o[4], of[4];            // (of: maximum and sum of both rows)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        o[z] = make_float4(0.f, 0.f, 0.f, 0.f);
        of[z] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
        if (z0 + z < p.parts) {
          uint32_t ao, am;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ao) : "r"(smem_u32(sO + idx)), "r"((uint32_t)(z0 + z)));
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(am) : "r"(smem_u32(sML + row)), "r"((uint32_t)(z0 + z)));
          asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(o[z].x), "=f"(o[z].y), "=f"(o[z].z), "=f"(o[z].w) : "r"(ao));
          asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(of[z].x), "=f"(of[z].y), "=f"(of[z].z), "=f"(of[z].w) : "r"(am));
        }
      }
#pragma unroll
      for (int z = 0; z < 4; ++z) add_part(acc, m, l, o[z], of[z]);
    }
    store<D>(p, w, seg.kvh, n, u, idx & 31, acc, l);
  }
  // nobody's shared memory goes away while another part reads it
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Dealt out: all pairs' tiles of keys in the order (row tile, kv head, tile); a block takes `share` of them, one after the other.  To begin
// and to end a pair costs as much as BEGIN tiles (measured for one eight of rows of 128, taken for all), which are dealt out with the others,
// ahead of the pair's own.
// What a block leaves for a pair that it shares goes to place block + pair of the scratch: no two blocks' places are the same,
// and those of one pair follow one another.
constexpr int BEGIN = 10;
__device__ __forceinline__ int64_t share_of(const Params& p, int64_t total, int blocks) {
  const int64_t even = (total + blocks - 1) / blocks;
  return even > p.least ? even : p.least;
}
// tiles of keys of the row tiles before `tile`, times the kv heads (and with tile = n_tiles: of all): the whole block, summed in shared memory
__device__ __forceinline__ int block_count(int v, int* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) s[warp] = v;
  __syncthreads();
  int sum = 0;
  for (int x = 0; x < n; ++x) sum += s[x];
  return sum;
}

template <int D, int NT, bool ONE>
__global__ void __launch_bounds__(WARPS * 32) dealt_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, Params p) {
  rb_pdl_launch_dependents();
  using S = Shape<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  begin<S>(smem);
  Ring ring{0, 0, false};
  __shared__ int counts[WARPS], s_tile, s_before;
  // positions, slots and page tables were written before the step began: the deal needs no wait
  int mine = 0;
  for (int i = threadIdx.x; i < p.n_tiles; i += WARPS * 32) mine += visited_tiles(p, i) + BEGIN;
  const int64_t total = (int64_t)block_count(mine, counts) * p.Kh;
  const int64_t share = share_of(p, total, gridDim.x);
  int64_t x = (int64_t)blockIdx.x * share;
  const int64_t end = x + share < total ? x + share : total;
  if (x >= end) return;
  // the row tile that tile x of all belongs to: the first warp walks over them, 32 at a time
  if (threadIdx.x < 32) {
    int before = 0;
    for (int i0 = 0; i0 < p.n_tiles; i0 += 32) {
      const int i = i0 + (int)threadIdx.x;
      const int n = i < p.n_tiles ? visited_tiles(p, i) + BEGIN : 0;
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if ((int)threadIdx.x >= o) upto += y;
      }
      const bool here = n > 0 && (int64_t)(before + upto) * p.Kh > x;
      const uint32_t who = __ballot_sync(0xffffffffu, here);
      if (who != 0) {
        if ((int)threadIdx.x == __ffs(who) - 1) { s_tile = i; s_before = before + upto - n; }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  int tile = s_tile;
  int64_t base = (int64_t)s_before * p.Kh;         // the first tile of the row tile's pairs
  // the block's next segment (tile < 0: none is left)
  auto next_segment = [&]() -> Segment {
    while (x < end) {
      Segment seg;
      seg.visited = visited_tiles(p, tile);
      const int length = seg.visited + BEGIN;
      if (x >= base + (int64_t)length * p.Kh) { base += (int64_t)length * p.Kh; ++tile; continue; }
      seg.tile = tile;
      seg.kvh = (int)((x - base) / length);
      const int64_t pair0 = base + (int64_t)seg.kvh * length;
      seg.first = max((int)(x - pair0) - BEGIN, 0);
      seg.last = (int)(end - pair0 < length ? end - pair0 : length) - BEGIN;
      x = pair0 + length;
      if (seg.last > seg.first) return seg;        // (else the range ends with what the pair's beginning costs)
    }
    return Segment{-1, 0, 0, 0, 0};
  };
  Segment seg = next_segment();
  if (seg.tile < 0) return;
  Job<D, NT> job(p, seg);
  rb_pdl_wait();
  {
    uint8_t* stages = smem + (threadIdx.x >> 5) * S::NS * S::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR) + (threadIdx.x >> 5) * S::NS;
#pragma unroll
    for (int i = 0; i < S::AHEAD; ++i) job.ask(p, &tmK, &tmV, stages, full, ring, i);
  }
  while (seg.tile >= 0) {
    const Segment now = seg;
    const Where w = job.w;
    Joined<D, NT> mine;
    work<D, NT, ONE>(p, &tmK, &tmV, job, smem, ring, mine, [&](uint8_t* stages, uint64_t* full) {
      seg = next_segment();
      if (seg.tile < 0) return;
      job = Job<D, NT>(p, seg);
#pragma unroll
      for (int i = 0; i < S::AHEAD; ++i) job.ask(p, &tmK, &tmV, stages, full, ring, i);
    });
    if (now.first == 0 && now.last == now.visited) {
      store<D, NT>(p, w, now.kvh, mine);
      continue;
    }
    const int64_t place = blockIdx.x + (int64_t)now.tile * p.Kh + now.kvh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int u = 0; u < S::QT; ++u) p.part_o[((place * NT + n) * S::MT + warp * S::QT + u) * 32 + lane] = mine.o[n][u];
      if (warp == 0 && lane < 4)
        *reinterpret_cast<float4*>(p.part_ml + place * S::ROWS + n * 8 + 2 * lane) = make_float4(mine.m[n][0], mine.l[n][0], mine.m[n][1], mine.l[n][1]);
    }
  }
}

// Pairs that several blocks have worked on: a block of threads per pair and 8 rows, a thread for what one lane's accumulators of a row tile hold.
template <int D, int NT>
__global__ void __launch_bounds__(D * 2) join_kernel(Params p, int blocks) {
  rb_pdl_launch_dependents();
  constexpr int MT = D / 16;
  __shared__ int counts[D / 16];
  const int tile = blockIdx.x, kvh = blockIdx.y, n = blockIdx.z;
  int all = 0, ahead = 0;
  for (int i = threadIdx.x; i < p.n_tiles; i += D * 2) {
    const int v = visited_tiles(p, i) + BEGIN;
    all += v;
    if (i < tile) ahead += v;
  }
  const int64_t total = (int64_t)block_count(all, counts) * p.Kh;
  const int64_t base = (int64_t)block_count(ahead, counts) * p.Kh;
  const Where w(p, tile);
  const int length = RbKeyTiles(w.key_lo, w.key_hi, p.a.keep, TILE).n + BEGIN;
  const int64_t share = share_of(p, total, blocks), pair0 = base + (int64_t)kvh * length;
  const int64_t first = (pair0 + BEGIN) / share, last = (pair0 + length - 1) / share;
  rb_pdl_wait();
  if (first == last || n * 8 >= w.ntok * p.G) return;
  const int64_t place = first + (int64_t)tile * p.Kh + kvh;
  const int parts = (int)(last - first) + 1, lane = threadIdx.x & 31;
  const float4* po = p.part_o + (place * NT + n) * MT * 32 + threadIdx.x;
  const float2* pm = p.part_ml + place * 8 * NT + n * 8 + 2 * (lane & 3);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  for (int z0 = 0; z0 < parts; z0 += 4) {
    float4 o[4], of[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      o[z] = make_float4(0.f, 0.f, 0.f, 0.f);
      of[z] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      if (z0 + z < parts) {
        o[z] = po[(int64_t)(z0 + z) * NT * MT * 32];
        of[z] = *reinterpret_cast<const float4*>(pm + (int64_t)(z0 + z) * 8 * NT);
      }
    }
#pragma unroll
    for (int z = 0; z < 4; ++z) add_part(acc, m, l, o[z], of[z]);
  }
  store<D>(p, w, kvh, n, (int)threadIdx.x >> 5, lane, acc, l);
}

// Pairs that are short, and many: each is ONE warp's work, from its first key to its output, and a block is one warp; nobody waits for
// anybody.  (24 sequences of 32 heads with a window of 1,024: 45 us, dealt out 49; 54 of up to 56 positions: 6.4, a block a pair 28.)
template <int D, int NT, int STAGES>
__global__ void __launch_bounds__(32) alone_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, Params p) {
  rb_pdl_launch_dependents();
  using S = typename Job<D, NT, STAGES>::S;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + STAGES * S::STAGE);
  const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(full + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  __syncwarp();
  Ring ring{0, 0, false};
  const int64_t pairs = (int64_t)p.n_tiles * p.Kh, step = gridDim.x;
  auto segment = [&](int64_t pair) {
    Segment seg;
    seg.tile = (int)(pair / p.Kh);
    seg.kvh = (int)(pair % p.Kh);
    seg.first = 0;
    seg.last = seg.visited = visited_tiles(p, seg.tile);
    return seg;
  };
  int64_t pair = blockIdx.x;
  Job<D, NT, STAGES> job(p, segment(pair));
  rb_pdl_wait();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) job.ask(p, &tmK, &tmV, stages, full, ring, i);
  for (; pair < pairs; pair += step) {
    Sums<D, NT> sums;
    run<D, NT, STAGES>(p, &tmK, &tmV, job, stages, stages, full, ring, sums);
    const Where w = job.w;
    const int kvh = job.seg.kvh;
    if (pair + step < pairs) {
      job = Job<D, NT, STAGES>(p, segment(pair + step));
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) job.ask(p, &tmK, &tmV, stages, full, ring, i);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = sums.l[n][c];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = n * 8 + 2 * t + c;
        if (r < w.ntok * p.G) {
          const float by = sums.by[n][c] / sum;
          uint32_t out[D / 16];
#pragma unroll
          for (int u = 0; u < D / 16; ++u) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(sums.o[n][u][c] * by, sums.o[n][u][c + 2] * by);
            out[u] = *reinterpret_cast<const uint32_t*>(&b);
          }
          uint4* dst = reinterpret_cast<uint4*>(p.a.out + ((int64_t)(w.tok0 + r / p.G) * p.a.H + kvh * p.G + r % p.G) * D + D / 8 * g);
#pragma unroll
          for (int x = 0; x < D / 64; ++x) dst[x] = make_uint4(out[4 * x], out[4 * x + 1], out[4 * x + 2], out[4 * x + 3]);
        }
      }
  }
}

// blocks of the kernel that an SM holds: by registers at the kernel's bound and by shared memory
template <int D, int NT> int per_sm() {
  static int n[RB_MAX_DEVICES] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= RB_MAX_DEVICES) dev = 0;
  if (n[dev] == 0) {
    int v = 0;
    if (cudaFuncSetAttribute(dealt_kernel<D, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D, NT>::BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(dealt_kernel<D, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D, NT>::BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(cluster_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D, NT>::BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(cluster_kernel<D, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v, dealt_kernel<D, NT, false>, WARPS * 32, Shape<D, NT>::BYTES) != cudaSuccess || v < 1)
      v = 1;
    (void)cudaGetLastError();
    n[dev] = v;
  }
  return n[dev];
}
// Clusters of `parts` blocks (2, 4, 8 or 16) that run together on the device (asked once): the GPCs' sizes leave fewer than the SMs' places
// would (72 clusters of 4 took two rounds where 296 blocks have places), and none of 16 on some devices.
template <int D, int NT> int clusters_at_once(int parts) {
  static int answer[RB_MAX_DEVICES][5] = {};
  int dev = 0, i = parts == 2 ? 1 : parts == 4 ? 2 : parts == 8 ? 3 : 4;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= RB_MAX_DEVICES) dev = 0;
  if (answer[dev][i] == 0) {
    per_sm<D, NT>();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, 1, parts);
    cfg.blockDim = dim3(WARPS * 32, 1, 1);
    cfg.dynamicSmemBytes = Shape<D, NT>::BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = parts;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    answer[dev][i] = cudaOccupancyMaxActiveClusters(&n, cluster_kernel<D, NT>, &cfg) == cudaSuccess && n >= 1 ? n : -1;
    (void)cudaGetLastError();      // a refusal is an answer, not an error of a later launch
  }
  return answer[dev][i];
}
inline int clusters(int D, int NT, int parts) {
  return D == 64 ? (NT == 1 ? clusters_at_once<64, 1>(parts) : NT == 2 ? clusters_at_once<64, 2>(parts) : NT == 3 ? clusters_at_once<64, 3>(parts) : clusters_at_once<64, 4>(parts))
                 : (NT == 1 ? clusters_at_once<128, 1>(parts) : NT == 2 ? clusters_at_once<128, 2>(parts) : NT == 3 ? clusters_at_once<128, 3>(parts) : clusters_at_once<128, 4>(parts));
}
inline int places(int D, int NT) {
  const int n = D == 64 ? (NT == 1 ? per_sm<64, 1>() : NT == 2 ? per_sm<64, 2>() : NT == 3 ? per_sm<64, 3>() : per_sm<64, 4>())
                        : (NT == 1 ? per_sm<128, 1>() : NT == 2 ? per_sm<128, 2>() : NT == 3 ? per_sm<128, 3>() : per_sm<128, 4>());
  return n * rb_sm_count();
}

// blocks: pairs; as many as the SMs hold at once take them in turn
template <int D, int NT, int STAGES>
int launch_alone(const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, int blocks, cudaStream_t stream) {
  constexpr int bytes = STAGES * Shape<D, NT, STAGES>::STAGE + STAGES * 8 + 1024;
  static int places[RB_MAX_DEVICES] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= RB_MAX_DEVICES) dev = 0;
  if (places[dev] == 0) {
    int n = 0;
    RB_CUDA(cudaFuncSetAttribute(alone_kernel<D, NT, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    RB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, alone_kernel<D, NT, STAGES>, 32, bytes));
    places[dev] = (n > 0 ? n : 1) * rb_sm_count();
  }
  RB_LAUNCH("rb_attention8_rows (alone)", (alone_kernel<D, NT, STAGES>), blocks < places[dev] ? blocks : places[dev], 32, bytes, stream, tk, tv, p);
  return 0;
}
template <int D, int NT>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, int blocks, cudaStream_t stream) {
  using S = Shape<D, NT>;
  if (p.parts < 0) {
    if constexpr (NT <= 2) return p.parts == -2 ? launch_alone<D, NT, 2>(tk, tv, p, blocks, stream) : launch_alone<D, NT, 3>(tk, tv, p, blocks, stream);
    RB_FAIL("rb_attention8_rows: %d rows do not go a pair a warp", S::ROWS);
  }
  per_sm<D, NT>();                                 // (sets the kernels' attributes)
  if (p.parts == 0) {
    if (p.tile_tok0) RB_LAUNCH("rb_attention8_rows", (dealt_kernel<D, NT, false>), blocks, WARPS * 32, S::BYTES, stream, tk, tv, p);
    else RB_LAUNCH("rb_attention8_rows", (dealt_kernel<D, NT, true>), blocks, WARPS * 32, S::BYTES, stream, tk, tv, p);
    RB_LAUNCH("rb_attention8_rows (join)", (join_kernel<D, NT>), dim3(p.n_tiles, p.Kh, NT), D * 2, 0, stream, p, blocks);
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_tiles, p.Kh, p.parts);
  cfg.blockDim = dim3(WARPS * 32, 1, 1);
  cfg.dynamicSmemBytes = S::BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = p.parts;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = rb_pdl_enabled() ? 2 : 1;
  RB_CUDA(cudaLaunchKernelEx(&cfg, cluster_kernel<D, NT>, tk, tv, p));
  return 0;
}
// Whether a warp a pair is sooner done than tiles dealt out: microseconds of the two on one B200, from 128 to 1,728 pairs of 1 to 30 tiles, heads
// of 128 with one eight of rows (taken for 64 and for two eights too).  A warp takes
// two units of 32 keys a tile, one a microsecond, eight warps an SM, or the bytes' time; dealt out a pair costs ten tiles beside its own.
// (Pairs x tiles, alone and dealt out: 320 x 4 10, 13; 960 x 5 17, 32; 768 x 17 45, 49; 1,024 x 30 78, 88; but 200 x 8 19, 13; 400 x 16 39, 29.)
inline bool alone_pays(long long pairs, int tiles, int D) {
  const double sms = rb_sm_count(), rounds = (double)((pairs + 8 * (long long)sms - 1) / (8 * (long long)sms));
  const double alone = rounds * (3.0 + 2.05 * tiles), bytes = 0.41 * pairs * tiles / sms * D / 128.0;
  return (alone > bytes ? alone : bytes) < 5.0 + 0.31 * pairs * (tiles + 10) / sms;
}

template <int D>
int launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, int NT, int blocks, cudaStream_t stream) {
  return NT == 1 ? launch<D, 1>(tk, tv, p, blocks, stream) : NT == 2 ? launch<D, 2>(tk, tv, p, blocks, stream)
       : NT == 3 ? launch<D, 3>(tk, tv, p, blocks, stream) : launch<D, 4>(tk, tv, p, blocks, stream);
}

}  // namespace rows8

// Whether the kernel of few rows takes these sizes (a token's heads of one kv head fit its rows, a tile of keys one page).
RB_EXPORT int rb_attention8_rows_supports(int H, int Kh, int D, int page_size) {
  if (Kh <= 0 || Kh > 65535 || H % Kh) return 0;
  return (D == 64 || D == 128) && page_size % rows8::TILE == 0 && H / Kh <= 32;
}

// How a launch of `n_tiles` row tiles of at most `rows` rows is cut, the longest sequence `context` positions: out4 = parts of a pair that
// are a cluster (0: dealt out), blocks when dealt out, floats of part_o, floats of part_ml.
// A cluster where two parts of every pair and more run at once and no part is long; a warp a pair (parts -2 or -3: the stages of its ring)
// where pairs are many and short; else all tiles are dealt out to as many blocks as the SMs hold at once, four tiles to a block at least.
// (Parts of up to 32 tiles: us as a cluster and dealt out, 8 sequences of 32 heads on 8 at 2,048 positions 11.9, 13.7, at 8,000 27.0, 29.0, but at
// unequal lengths up to 8,000 25.4, 20.7: a captured step's `context` is the longest its sequences may get, so most of its parts are shorter.)
RB_EXPORT int rb_attention8_rows_plan(int n_tiles, int rows, int Kh, int D, int context, long long* out4) {
  const int NT = (rows + 7) / 8, places = rows8::places(D, NT);
  const int tiles = (context + rows8::TILE - 1) / rows8::TILE;
  const long long pairs = (long long)n_tiles * Kh;
  RB_REQUIRE(n_tiles > 0 && Kh > 0 && rows > 0 && rows <= 32, "rb_attention8_rows_plan: %d tiles of %d rows, %d kv heads", n_tiles, rows, Kh);
  int parts = 1;
  while (parts * 2 <= tiles && parts < 16 && pairs <= rows8::clusters(D, NT, parts * 2)) parts *= 2;
  out4[0] = parts; out4[1] = out4[2] = out4[3] = 0;
  if (parts > 1 && tiles <= 32 * parts) return 0;
  if (NT <= 2 && pairs <= 2147483647ll && (tiles <= 1 || rows8::alone_pays(pairs, tiles, D))) {
    out4[0] = tiles <= 2 ? -2 : -3;
    out4[1] = pairs;
    return 0;
  }
  if (tiles <= 1) return 0;
  long long blocks = (pairs * tiles + 3) / 4;
  if (blocks > places) blocks = places;
  out4[0] = 0;
  out4[1] = blocks;
  out4[2] = (blocks + pairs) * 8 * NT * D;
  out4[3] = (blocks + pairs) * 8 * NT * 2;
  return 0;
}

// Few rows a sequence: row tile i is the tile_ntok[i] tokens from tile_tok0[i] on, of one sequence (null: row i alone), at most `rows` rows
// of H / Kh heads each; cut as rb_attention8_rows_plan says, with its scratch.
RB_EXPORT int rb_attention8_rows(void* out, const void* q, void* cache_k, void* cache_v, const float* k_scale, const float* v_scale, long long n_pages,
                                 const int* page_table, int max_pages, int page_size, const int* tok_pos, const int* tok_slot,
                                 const int* tile_tok0, const int* tile_ntok, int n_tiles, int rows, int H, int Kh, int D, float scale,
                                 int window, int parts, int blocks, float* part_o, float* part_ml, cudaStream_t stream) {
  const RbAttentionOptions opt = rb_attention_take();
  if (n_tiles == 0) return 0;
  RB_REQUIRE(rb_attention8_rows_supports(H, Kh, D, page_size) && rows >= H / Kh && rows <= 32,
             "rb_attention8_rows: sizes H=%d Kh=%d D=%d page=%d, %d rows not supported", H, Kh, D, page_size, rows);
  RB_REQUIRE(n_pages * Kh * page_size / rows8::TILE <= 2147483647ll && n_pages * Kh * page_size * D / 128 <= 2147483647ll,
             "rb_attention8_rows: a pool of %lld pages has too many blocks", n_pages);
  RB_REQUIRE(parts >= -3 && parts != -1 && parts <= 16 && (parts <= 0 || (parts & (parts - 1)) == 0) && (parts > 0 || blocks > 0) &&
                 (parts != 0 || (part_o && part_ml)), "rb_attention8_rows: %d parts, %d blocks", parts, blocks);
  rows8::Params p;
  p.a.q = (const __nv_bfloat16*)q; p.a.out = (__nv_bfloat16*)out;
  p.a.cache = RbPagedLayer{cache_k, cache_v, page_table, max_pages, page_size, Kh, D};
  p.a.k_scale = k_scale; p.a.v_scale = v_scale; p.a.block = rows8::TILE;
  p.a.tok_pos = tok_pos; p.a.tok_slot = tok_slot; p.a.H = H;
  p.a.scale = scale; p.a.window = window; p.a.keep = window > 0 ? opt.keep_first : 0; p.a.sinks = opt.sinks; p.a.softcap = opt.softcap;
  p.tile_tok0 = tile_tok0; p.tile_ntok = tile_ntok; p.n_tiles = n_tiles; p.Kh = Kh; p.G = H / Kh;
  p.parts = parts; p.least = 4; p.part_o = (float4*)part_o; p.part_ml = (float2*)part_ml;
  CUtensorMap tk, tv;                                // rows of 128 bytes, a warp's 32 positions a box
  const long long rows128 = n_pages * Kh * page_size * D / 128;
  if (rb_get_tensor_map(&tk, cache_k, rows128, 64, 64, 32 * D / 128) != 0) return -1;
  if (rb_get_tensor_map(&tv, cache_v, rows128, 64, 64, 32 * D / 128) != 0) return -1;
  const int NT = (rows + 7) / 8;
  return D == 64 ? rows8::launch_rows<64>(tk, tv, p, NT, blocks, stream) : rows8::launch_rows<128>(tk, tv, p, NT, blocks, stream);
}
