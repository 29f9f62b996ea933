// Mean key of every block of keys, and for every query the blocks whose mean has
// the largest product with it.
//
//   mean[b, h, n] = sum of block n's live keys / their number      (fp32, zero without one)
//   score[b, h, i, n] = (sum of the queries i of the heads that share key head h) . mean
//   sel[b, h, i] = the topk live blocks of largest score, ascending, then -1
//
// A choice hangs on which of two scores is larger, so means and scores are summed in
// float64: a program that computes them in another order (or another batch) chooses
// the same blocks, up to scores that agree in some 50 bits. Equal scores go to the lower
// block; a NaN counts as the lowest. Scores run on the fp64 matrix product,
// 16 queries x 16 blocks x 4 dimensions, at 1/16 of the bf16 one's rate; with D
// dimensions and NB blocks it is 2 D NB operations a query beside the 2 D bytes that
// the query costs to read, so long sequences are bound by it (64000 query groups,
// 125 blocks, D = 128: 28 us at the rate of a large fp64 product).
#include "capi.hpp"
#include "common.hpp"

namespace shrimp {
namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int MAX_TOPK = SHRIMP_BLOCK_MAX_TOPK;
constexpr int MAX_D = SHRIMP_BLOCK_MAX_D;
constexpr int MAX_BLOCKS = SHRIMP_BLOCK_MAX_BLOCKS;
constexpr int MAX_KEYS = 1 << 30;  // (a length and a block add up within an int)

template <typename T, int V>
using Vec = T __attribute__((ext_vector_type(V)));

struct MeanParams {
  const void* k;
  const int32_t* lens;
  float* means;
  int64_t sb, sh, sn;
  int B, Hk, Sk, D, NB, block;
  int lanes;  // lanes per row
  int last_only;
};

// One wave per block of keys: lanes take a row's dimensions, groups of lanes rows, U of
// them in flight.
template <typename T, int V, int U>
__global__ __launch_bounds__(256) void block_means_kernel(const MeanParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + wave_id();
  const int per = p.last_only ? 1 : p.NB;
  const int64_t bh = item / per;
  if (bh >= (int64_t)p.B * p.Hk) return;
  const int b = (int)(bh / p.Hk), h = (int)(bh - (int64_t)b * p.Hk);
  const int len = min(max(p.lens[b], 0), p.Sk);
  const int n = p.last_only ? max(len - 1, 0) / p.block : (int)(item - bh * per);
  const int64_t start = (int64_t)n * p.block;
  const int rows = (int)min((int64_t)p.block, len - start);  // live keys, none if <= 0
  const int ul = lane & (p.lanes - 1), group = lane / p.lanes, groups = 64 / p.lanes;
  float* out = p.means + (bh * p.NB + n) * p.D;
  const T* k = static_cast<const T*>(p.k) + b * p.sb + h * p.sh + start * p.sn;
  for (int d = ul * V; d < p.D; d += p.lanes * V) {
    double sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.0;
    for (int r0 = group; r0 < rows; r0 += groups * U) {
      Vec<T, V> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        x[u] = *reinterpret_cast<const Vec<T, V>*>(k + (int64_t)min(r0 + u * groups, rows - 1) * p.sn + d);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += r0 + u * groups < rows ? (double)(float)x[u][e] : 0.0;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      for (int m = p.lanes; m < 64; m <<= 1) sum[e] += __shfl_xor(sum[e], m, 64);
      if (group == 0) out[d + e] = rows > 0 ? (float)(sum[e] / (double)rows) : 0.f;
    }
  }
}

struct SelectParams {
  const void* q;
  const float* means;
  const int32_t* q_lens;
  const int32_t* k_lens;
  int32_t* sel;
  int64_t sb, sh, sn;
  int B, H, Hk, Sq, Sk, D, NB, block, topk;
  int group;   // query heads per key head
  int tiles;   // tiles of 16 queries per (sequence, key head)
  int chunk;   // blocks scored before a choice among them and the carried ones
  int vec;     // rows of q readable four elements at a time
};

// Order of doubles as order of unsigned integers; 0 is left for "none".
SHRIMP_DEV uint64_t order_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);  // -0 as 0
  if (x != x) return 1;
  return u >> 63 ? ~u : u | (1ull << 63);
}

template <typename T>
SHRIMP_DEV double load_f64(const T* p) {
  return (double)(float)*p;
}

// One wave: 16 queries of a (sequence, key head). LDS: per query row the carried keys
// and a chunk's keys, the carried indices, and the chosen of this chunk.
template <typename T, int DP>
__global__ __launch_bounds__(64) void block_select_kernel(const SelectParams p) {
  extern __shared__ uint64_t lds[];
  constexpr int DK = DP / 4;  // dimensions of a lane: of the four that a product takes
                              // at a time, lane group g supplies dimensions g DK + step
  const int lane = threadIdx.x, lr = lane & 15, lg = lane >> 4;
  const int64_t bh = blockIdx.x / p.tiles;
  const int tile = (int)(blockIdx.x - bh * p.tiles);
  const int b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  const int q_len = min(max(p.q_lens[b], 0), p.Sq), k_len = min(max(p.k_lens[b], 0), p.Sk);
  const int live = (k_len + p.block - 1) / p.block;
  const int i0 = tile * 16;
  const int entries = p.topk + p.chunk;
  uint64_t* keys = lds;                               // [16][entries]
  uint64_t* best_key = keys + 16 * entries;           // [16][topk]
  int* best_id = reinterpret_cast<int*>(best_key + 16 * p.topk);  // [16][topk]
  int* carry_id = best_id + 16 * p.topk;              // [16][topk]
  int32_t* sel = p.sel + (bh * p.Sq + i0) * p.topk;
  const int rows = min(16, p.Sq - i0);

  if (i0 >= q_len || live <= p.topk) {  // none, or every live block
    for (int j = lane; j < rows * p.topk; j += 64) {
      const int r = j / p.topk, t = j - r * p.topk;
      sel[j] = i0 + r < q_len && t < live ? t : -1;
    }
    return;
  }

  double a[DK];
#pragma unroll
  for (int s = 0; s < DK; ++s) a[s] = 0.0;
  if (i0 + lr < q_len) {
    for (int h = 0; h < p.group; ++h) {
      const T* q = static_cast<const T*>(p.q) + b * p.sb + (int64_t)(hk * p.group + h) * p.sh +
                   (int64_t)(i0 + lr) * p.sn;
      if (p.vec) {
#pragma unroll
        for (int s = 0; s < DK; s += 4) {
          const int d = lg * DK + s;
          if (d < p.D) {
            const Vec<T, 4> x = *reinterpret_cast<const Vec<T, 4>*>(q + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[s + e] += (double)(float)x[e];
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < DK; ++s)
          if (lg * DK + s < p.D) a[s] += load_f64(q + lg * DK + s);
      }
    }
  }

  const float* means = p.means + bh * p.NB * p.D;
  const bool mvec = p.D % 4 == 0;
  const int row = lane >> 2, sub = lane & 3;  // the choice: four lanes per query
  int carried = 0;
  for (int c0 = 0; c0 < live; c0 += p.chunk) {
    const int here = min(p.chunk, live - c0);
    for (int t = 0; t < here; t += 16) {
      const int n = c0 + t + lr;
      float m[DK];
#pragma unroll
      for (int s = 0; s < DK; ++s) m[s] = 0.f;
      if (n < live) {
        const float* row_n = means + (int64_t)n * p.D;
        if (mvec) {
#pragma unroll
          for (int s = 0; s < DK; s += 4) {
            const int d = lg * DK + s;
            if (d < p.D) {
              const f32x4 x = *reinterpret_cast<const f32x4*>(row_n + d);
#pragma unroll
              for (int e = 0; e < 4; ++e) m[s + e] = x[e];
            }
          }
        } else {
#pragma unroll
          for (int s = 0; s < DK; ++s)
            if (lg * DK + s < p.D) m[s] = row_n[lg * DK + s];
        }
      }
      f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int s = 0; s < DK; ++s)
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s], (double)m[s], acc, 0, 0, 0);
      // lane (lr, lg) holds block column lr of queries 4 i + lg
#pragma unroll
      for (int i = 0; i < 4; ++i)
        keys[(4 * i + lg) * entries + p.topk + t + lr] = n < live ? order_key(acc[i]) : 0;
    }
    __syncthreads();
    // the topk largest of the carried and the new, largest first
    const int first = carried ? 0 : p.topk, last = p.topk + ((here + 15) & ~15);
    uint64_t* mine = keys + row * entries;
    for (int it = 0; it < p.topk; ++it) {
      uint64_t key = 0;
      int at = -1;
      for (int j = first + sub; j < last; j += 4) {
        const uint64_t k = mine[j];
        if (k > key) {
          key = k;
          at = j;
        }
      }
#pragma unroll
      for (int m = 1; m <= 2; m <<= 1) {
        const uint64_t k = __shfl_xor(key, m, 64);
        const int j = __shfl_xor(at, m, 64);
        if (k > key || (k == key && k != 0 && j < at)) {
          key = k;
          at = j;
        }
      }
      if (sub == 0) {
        best_key[row * p.topk + it] = key;
        best_id[row * p.topk + it] =
            key == 0 ? -1 : at < p.topk ? carry_id[row * p.topk + at] : c0 + at - p.topk;
        if (key != 0) mine[at] = 0;
      }
      __syncthreads();
    }
    carried = 1;
    for (int j = lane; j < 16 * p.topk; j += 64) {
      const int r = j / p.topk, t = j - r * p.topk;
      keys[r * entries + t] = best_key[j];
      carry_id[j] = best_id[j];
    }
    __syncthreads();
  }
  // ascending: a chosen block's place is the number of chosen ones below it
  for (int j = lane; j < rows * p.topk; j += 64) {
    const int r = j / p.topk;
    const int id = best_id[j];
    int at = 0;
    for (int t = 0; t < p.topk; ++t) at += best_id[r * p.topk + t] < id;
    sel[r * p.topk + at] = i0 + r < q_len ? id : -1;
  }
}

// Up to 16 NT blocks: the scores stay in registers, and the choice works on 32-bit keys
// that are certain where they differ. A score, rounded to fp32 (which keeps the order),
// loses the low bits of its ordered form to the place it has: block tile and lane. Each
// lane sorts its NT keys of a query; the topk largest heads among the query's 16 lanes
// are taken off one by one (four queries side by side), 4 NT + 32 instructions each
// against 32 LDS reads of the kernel above. Where the last taken and the next key agree
// but for the place (scores within 2^-15 of each other: some row in ten thousand, or
// equal scores), float64 scores decide, computed again for that query by the whole wave.
// (For all 16 of the tile by matrix products, four times through the blocks, the few
// waves that met one ended 27 of 95 us after the others: 2 x 8000 queries, 125 blocks.)
constexpr int REG_WAVES = 4;

SHRIMP_DEV unsigned place_key(float x, unsigned drop, unsigned place) {
  const unsigned u = __float_as_uint(x + 0.f);
  const unsigned k = (int)u < 0 ? ~u : u | 0x80000000u;
  return (x != x ? 1u << drop : k >> drop << drop) | place;
}

SHRIMP_DEV uint64_t lane_u64(uint64_t v, int lane) {  // (lane: wave-uniform)
  return (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}

// The maxima over the 16 lanes of a row, for all of them: four side by side, a step of each
// between the steps of another (a DPP read waits for the write before it).
SHRIMP_DEV void row_max(unsigned (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = max(v[i], (unsigned)__builtin_amdgcn_mov_dpp((int)v[i], 0xB1, 0xF, 0xF, true));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = max(v[i], (unsigned)__builtin_amdgcn_mov_dpp((int)v[i], 0x4E, 0xF, 0xF, true));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = max(v[i], (unsigned)__builtin_amdgcn_mov_dpp((int)v[i], 0x141, 0xF, 0xF, true));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = max(v[i], (unsigned)__builtin_amdgcn_mov_dpp((int)v[i], 0x140, 0xF, 0xF, true));
}

template <int N>
SHRIMP_DEV void sort_down(unsigned (&x)[N]) {  // odd-even merge sort, largest first
#pragma unroll
  for (int p = 1; p < N; p <<= 1)
#pragma unroll
    for (int k = p; k >= 1; k >>= 1)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const unsigned a = x[i + j], b = x[i + j + k];
            x[i + j] = max(a, b);
            x[i + j + k] = min(a, b);
          }
}

// FULL: heads of exactly DP dimensions, rows readable four at a time.
template <typename T, int DP, int NT, bool FULL>
__global__ __launch_bounds__(REG_WAVES * 64) void block_select_reg_kernel(const SelectParams p) {
  constexpr int DK = DP / 4;
  constexpr unsigned TB = NT == 4 ? 2 : NT == 8 ? 3 : 4, DROP = TB + 4;  // bits of a place: tile, lane
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int64_t item = (int64_t)blockIdx.x * REG_WAVES + wave_id();
  const int64_t bh = item / p.tiles;
  if (bh >= (int64_t)p.B * p.Hk) return;
  const int tile = (int)(item - bh * p.tiles);
  const int b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  const int q_len = min(max(p.q_lens[b], 0), p.Sq), k_len = min(max(p.k_lens[b], 0), p.Sk);
  const int live = (k_len + p.block - 1) / p.block;
  const int i0 = tile * 16;
  int32_t* sel = p.sel + (bh * p.Sq + i0) * p.topk;
  const int rows = min(16, p.Sq - i0);
  if (i0 >= q_len || live <= p.topk) {
    for (int j = lane; j < rows * p.topk; j += 64) {
      const int r = j / p.topk, t = j - r * p.topk;
      sel[j] = i0 + r < q_len && t < live ? t : -1;
    }
    return;
  }

  // mean rows: lane (lr, lg) supplies dimensions lg DK .. of block 16 t + lr (past the
  // blocks the last one again, its scores not used)
  const float* means = p.means + bh * p.NB * p.D;
  auto load = [&](int t, float (&x)[DK]) {
    const float* m = means + (int64_t)min(t * 16 + lr, live - 1) * p.D;
    if (FULL || p.D % 4 == 0) {
#pragma unroll
      for (int s = 0; s < DK; s += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(m + (FULL ? lg * DK + s : min(lg * DK + s, p.D - 4)));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[s + e] = v[e];
      }
    } else {
#pragma unroll
      for (int s = 0; s < DK; ++s) x[s] = m[min(lg * DK + s, p.D - 1)];
    }
  };
  float x[DK];
  load(0, x);

  double a[DK];
#pragma unroll
  for (int s = 0; s < DK; ++s) a[s] = 0.0;
  const int mine = min(i0 + lr, q_len - 1);  // (past the queries: the last one again, not written)
  const T* q0 = static_cast<const T*>(p.q) + b * p.sb + (int64_t)(hk * p.group) * p.sh + (int64_t)mine * p.sn;
  if (FULL || p.vec) {
    Vec<T, 4> v[DK / 4], w[DK / 4];
    auto row = [&](int h, Vec<T, 4> (&y)[DK / 4]) {
#pragma unroll
      for (int s = 0; s < DK / 4; ++s)
        y[s] = *reinterpret_cast<const Vec<T, 4>*>(q0 + h * p.sh +
                                                   (FULL ? lg * DK + s * 4 : min(lg * DK + s * 4, p.D - 4)));
    };
    row(0, v);
    for (int h = 0; h < p.group; ++h) {  // the next head's row in flight
      row(min(h + 1, p.group - 1), w);
#pragma unroll
      for (int s = 0; s < DK; ++s) {
        const double y = (double)(float)v[s / 4][s % 4];
        a[s] += FULL || lg * DK + s < p.D ? y : 0.0;
      }
#pragma unroll
      for (int s = 0; s < DK / 4; ++s) v[s] = w[s];
    }
  } else {
    for (int h = 0; h < p.group; ++h)
#pragma unroll
      for (int s = 0; s < DK; ++s)
        a[s] += lg * DK + s < p.D ? load_f64(q0 + h * p.sh + min(lg * DK + s, p.D - 1)) : 0.0;
  }

  // scores of a block tile: lane (lr, lg) has block lr of queries 4 i + lg. Two chains of
  // products, so that one need not wait for the other.
  auto score = [&](const float (&m)[DK]) {
    f64x4 even = {0.0, 0.0, 0.0, 0.0}, odd = even;
#pragma unroll
    for (int s = 0; s < DK; s += 2) {
      const double y = FULL || lg * DK + s < p.D ? (double)m[s] : 0.0;
      const double z = FULL || lg * DK + s + 1 < p.D ? (double)m[s + 1] : 0.0;
      even = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s], y, even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s + 1], z, odd, 0, 0, 0);
    }
    return even + odd;
  };

  unsigned key[4][NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float next[DK];
    if (t + 1 < NT) load(t + 1, next);
    if (t * 16 < live) {
      const f64x4 acc = score(x);
      const bool on = t * 16 + lr < live;
      const unsigned place = (unsigned)(NT - 1 - t) << 4 | (unsigned)(15 - lr);
#pragma unroll
      for (int i = 0; i < 4; ++i) key[i][t] = on ? place_key((float)acc[i], DROP, place) : 0;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) key[i][t] = 0;
    }
    if (t + 1 < NT) {
#pragma unroll
      for (int s = 0; s < DK; ++s) x[s] = next[s];
    }
  }
  unsigned chosen[4], last[4];  // bit t: block 16 t + lr is chosen for query 4 i + lg
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sort_down(key[i]);
    chosen[i] = last[i] = 0;
  }
  for (int it = 0; it < p.topk; ++it) {
#pragma unroll
    for (int i = 0; i < 4; ++i) last[i] = key[i][0];
    row_max(last);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool win = key[i][0] == last[i];
      chosen[i] |= win ? 1u << (NT - 1 - (last[i] >> 4 & (NT - 1))) : 0;
#pragma unroll
      for (int t = 0; t + 1 < NT; ++t) key[i][t] = win ? key[i][t + 1] : key[i][t];
      key[i][NT - 1] = win ? 0 : key[i][NT - 1];
    }
  }
  // Queries whose last and next key differ in their places only are decided by float64
  // scores, one query at a time (bit r of `open`: query r).
  unsigned open = 0, then[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) then[i] = key[i][0];
  row_max(then);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t same = __ballot((then[i] ^ last[i]) >> DROP == 0);
#pragma unroll
    for (int g = 0; g < 4; ++g) open |= (unsigned)(same >> (16 * g) & 1) << (4 * i + g);
  }
  open &= (1u << min(16, q_len - i0)) - 1;
  for (unsigned left = open; left != 0; left &= left - 1) {
    const int r = __builtin_ctz(left);
    constexpr int NU = NT / 4;  // blocks of a lane: 64 u + lane
    double sum[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) sum[u] = 0.0;
#pragma unroll 1
    for (int part = 0; part < 4; ++part)
#pragma unroll
      for (int d0 = 0; d0 < DK; d0 += 4) {
        if (d0 % 16 == 0) __builtin_amdgcn_sched_barrier(0);  // (no more loads at a time than this)
        float m[NU][4];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const float* row = means + (int64_t)min(u * 64 + lane, live - 1) * p.D;
          const int d = part * DK + d0;
          if (FULL || p.D % 4 == 0) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(row + (FULL ? d : min(d, p.D - 4)));
#pragma unroll
            for (int e = 0; e < 4; ++e) m[u][e] = v[e];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) m[u][e] = row[min(d + e, p.D - 1)];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double x = __builtin_bit_cast(double, lane_u64(__builtin_bit_cast(uint64_t, a[d0 + e]), part * 16 + r));
          const bool in = FULL || part * DK + d0 + e < p.D;
#pragma unroll
          for (int u = 0; u < NU; ++u) sum[u] = __builtin_fma(x, in ? (double)m[u][e] : 0.0, sum[u]);
        }
      }
    uint64_t k[NU], edge = 0;  // the topk-th largest key, from its highest bit down
#pragma unroll
    for (int u = 0; u < NU; ++u) k[u] = u * 64 + lane < live ? order_key(sum[u]) : 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t next = edge | 1ull << bit;
      int n = 0;
#pragma unroll
      for (int u = 0; u < NU; ++u) n += __popcll(__ballot(k[u] >= next));
      if (n >= p.topk) edge = next;
    }
    int want = p.topk, at = 0;  // how many of those equal to it: the lowest blocks
#pragma unroll
    for (int u = 0; u < NU; ++u) want -= __popcll(__ballot(k[u] > edge));
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const uint64_t ties = __ballot(k[u] == edge);
      const bool is = k[u] > edge || (k[u] == edge && __popcll(ties & below) < want);
      const uint64_t of = __ballot(is);
      if (is) sel[r * p.topk + at + __popcll(of & below)] = u * 64 + lane;
      at += __popcll(of);
      want -= min(want, __popcll(ties));
    }
  }
  // ascending: the chosen blocks of earlier tiles, then of earlier lanes
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + lg;
    int base = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const bool is = chosen[i] >> t & 1;
      const unsigned of = (unsigned)(__ballot(is) >> (16 * lg)) & 0xFFFFu;
      if (is && i0 + row < q_len && !(open >> row & 1)) sel[row * p.topk + base + __popc(of & ((1u << lr) - 1))] = t * 16 + lr;
      base += __popc(of);
    }
    if (lr == 0 && row < rows && i0 + row >= q_len)
      for (int t = 0; t < p.topk; ++t) sel[row * p.topk + t] = -1;
  }
}

// Few queries (serving): a workgroup per query, 16 lanes per block's product.
constexpr int ROW_THREADS = 512;

// The topk largest keys by radix selection, a byte at a time: a histogram of the keys that
// share the bytes found so far, the bin in which the topk-th falls, until that bin is
// taken whole (three bytes or so) or all eight are done (equal scores: lowest blocks).
template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void block_select_row_kernel(const SelectParams p) {
  extern __shared__ uint64_t lds[];
  __shared__ int hist[256];
  __shared__ int state[3];  // bin, keys wanted of it, keys in it
  __shared__ int counts[2][ROW_THREADS / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int64_t bh = blockIdx.x / p.Sq;
  const int i = (int)(blockIdx.x - bh * p.Sq);
  const int b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  const int q_len = min(max(p.q_lens[b], 0), p.Sq), k_len = min(max(p.k_lens[b], 0), p.Sk);
  const int live = (k_len + p.block - 1) / p.block;
  int32_t* sel = p.sel + (bh * p.Sq + i) * p.topk;
  if (i >= q_len || live <= p.topk) {
    for (int t = tid; t < p.topk; t += ROW_THREADS) sel[t] = i < q_len && t < live ? t : -1;
    return;
  }
  double* q = reinterpret_cast<double*>(lds);  // [MAX_D]
  uint64_t* keys = lds + MAX_D;                // [live]
  if (tid < MAX_D) {
    double s = 0.0;
    if (tid < p.D)
      for (int h = 0; h < p.group; ++h)
        s += load_f64(static_cast<const T*>(p.q) + b * p.sb + (int64_t)(hk * p.group + h) * p.sh +
                      (int64_t)i * p.sn + tid);
    q[tid] = s;
  }
  __syncthreads();
  const float* means = p.means + bh * p.NB * p.D;
  const int part = tid & 15;
  constexpr int U = 4, STEP = ROW_THREADS / 16;  // blocks in flight per 16 lanes
  for (int n0 = tid >> 4; n0 < live; n0 += U * STEP) {
    double s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = 0.0;
    if (p.D % 4 == 0) {
      for (int d = part * 4; d < p.D; d += 64) {
        f32x4 m[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          m[u] = *reinterpret_cast<const f32x4*>(means + (int64_t)min(n0 + u * STEP, live - 1) * p.D + d);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u] = __builtin_fma(q[d + e], (double)m[u][e], s[u]);
      }
    } else {
      for (int d = part; d < p.D; d += 16)
#pragma unroll
        for (int u = 0; u < U; ++u)
          s[u] = __builtin_fma(q[d], (double)means[(int64_t)min(n0 + u * STEP, live - 1) * p.D + d], s[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      for (int x = 1; x < 16; x <<= 1) s[u] += __shfl_xor(s[u], x, 64);
      if (part == 0 && n0 + u * STEP < live) keys[n0 + u * STEP] = order_key(s[u]);
    }
  }
  uint64_t found = 0, known = 0;  // bytes of the topk-th key, and which they are
  int want = p.topk;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int n = tid; n < live; n += ROW_THREADS)
      if (((keys[n] ^ found) & known) == 0) atomicAdd(&hist[keys[n] >> shift & 255], 1);
    __syncthreads();
    if (wave == 0) {  // bins 4 lane .. + 3: how many keys lie above them
      int c[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += c[e] = hist[4 * lane + e];
      int up = sum;
      for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_down(up, m, 64);
        if (lane + m < 64) up += o;
      }
      int over = up - sum;
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        if (over < want && over + c[e] >= want) {
          state[0] = 4 * lane + e;
          state[1] = want - over;
          state[2] = c[e];
        }
        over += c[e];
      }
    }
    __syncthreads();
    found |= (uint64_t)state[0] << shift;
    known |= 255ull << shift;
    want = state[1];
    const bool whole = state[1] == state[2];
    __syncthreads();
    if (whole) break;
  }
  // keys above, and `want` of those that agree in the known bytes (all of them, or equal
  // ones), in ascending order of the blocks
  int base = 0, ties = 0;
  for (int n0 = 0; n0 < live; n0 += ROW_THREADS) {
    const int n = n0 + tid;
    const uint64_t k = n < live ? keys[n] & known : 0;
    const bool over = n < live && k > found, tie = n < live && k == found;
    const uint64_t over_b = __ballot(over), tie_b = __ballot(tie), below = (1ull << lane) - 1;
    if (lane == 0) {
      counts[0][wave] = __popcll(over_b);
      counts[1][wave] = __popcll(tie_b);
    }
    __syncthreads();
    int over_at = 0, tie_at = 0, over_all = 0, tie_all = 0;
#pragma unroll
    for (int w = 0; w < ROW_THREADS / 64; ++w) {
      over_at += w < wave ? counts[0][w] : 0;
      tie_at += w < wave ? counts[1][w] : 0;
      over_all += counts[0][w];
      tie_all += counts[1][w];
    }
    over_at += __popcll(over_b & below);
    tie_at += ties + __popcll(tie_b & below);
    if (over || (tie && tie_at < want)) sel[base + over_at + min(tie_at, want)] = n;
    ties += tie_all;
    base += over_all;
    __syncthreads();
  }
}

int pow2_ceil(int n) {
  int v = 1;
  while (v < n) v <<= 1;
  return v;
}

int dt_size(int dt) { return dt == SHRIMP_DT_F32 ? 4 : 2; }

bool row_vec(int v, const void* base, int64_t sb, int64_t sh, int64_t sn, int D, int es) {
  return D % v == 0 && sb % v == 0 && sh % v == 0 && sn % v == 0 &&
         reinterpret_cast<uintptr_t>(base) % (uintptr_t)(v * es) == 0;
}

template <typename T>
void means_grid(const MeanParams& p, int vec, dim3 grid, hipStream_t st) {
  constexpr int WIDE = 16 / sizeof(T);
  if (vec == WIDE && WIDE > 4)
    hipLaunchKernelGGL((block_means_kernel<T, WIDE, 8>), grid, dim3(256), 0, st, p);
  else if (vec == 4)
    hipLaunchKernelGGL((block_means_kernel<T, 4, 4>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((block_means_kernel<T, 1, 4>), grid, dim3(256), 0, st, p);
}

int means_launch(const void* k, int64_t sb, int64_t sh, int64_t sn, int dt, const int32_t* lens,
                 float* means, int B, int Hk, int Sk, int D, int block, bool last_only,
                 void* stream, const char* what) {
  SHRIMP_REQUIRE(dt == SHRIMP_DT_BF16 || dt == SHRIMP_DT_F16 || dt == SHRIMP_DT_F32,
                 "%s: element type %d", what, dt);
  SHRIMP_REQUIRE(B >= 0 && Hk >= 0 && Sk >= 0, "%s: negative size", what);
  SHRIMP_REQUIRE(D >= 1 && D <= MAX_D, "%s: head dim %d outside [1, %d]", what, D, MAX_D);
  SHRIMP_REQUIRE(block >= 1 && block <= MAX_KEYS && Sk <= MAX_KEYS, "%s: block of %d keys of %d", what, block, Sk);
  const int64_t nb = ((int64_t)Sk + block - 1) / block;
  SHRIMP_REQUIRE(nb <= MAX_BLOCKS, "%s: %lld blocks, at most %d", what, (long long)nb, MAX_BLOCKS);
  if (B == 0 || Hk == 0 || nb == 0) return SHRIMP_OK;
  SHRIMP_REQUIRE(k && lens && means, "%s: null pointer", what);
  const int64_t items = mul_sat({B, Hk, last_only ? 1 : nb});
  SHRIMP_REQUIRE(items <= INT32_MAX, "%s: %lld blocks of keys", what, (long long)items);
  const int wide = 16 / dt_size(dt);
  // 16-byte accesses for long blocks; for short ones 8, which leave fewer lanes to add up
  // (111 x 3 heads x 37 blocks of 16, D = 64: 10.7 against 14.7 us)
  const int vec = block >= 64 && row_vec(wide, k, sb, sh, sn, D, dt_size(dt)) ? wide
                  : row_vec(4, k, sb, sh, sn, D, dt_size(dt))                 ? 4
                                                                              : 1;
  const int units = D / vec;
  const MeanParams p{k, lens, means, sb, sh, sn, B, Hk, Sk, D, (int)nb, block,
                     pow2_ceil(units < 64 ? units : 64), last_only};
  const dim3 grid((unsigned)((items + 3) / 4));
  hipStream_t st = as_stream(stream);
  if (dt == SHRIMP_DT_F32)
    means_grid<float>(p, vec, grid, st);
  else if (dt == SHRIMP_DT_F16)
    means_grid<_Float16>(p, vec, grid, st);
  else
    means_grid<__bf16>(p, vec, grid, st);
  return check_launch(what);
}

template <typename T>
void select_launch(const SelectParams& p, int64_t rows, size_t row_lds, size_t tile_lds, bool by_row,
                   hipStream_t st) {
  if (by_row) {
    hipLaunchKernelGGL((block_select_row_kernel<T>), dim3((unsigned)rows), dim3(ROW_THREADS), row_lds,
                       st, p);
    return;
  }
  const int64_t tiles = (int64_t)p.B * p.Hk * p.tiles;
  const dim3 reg_grid((unsigned)((tiles + REG_WAVES - 1) / REG_WAVES)), reg_block(REG_WAVES * 64);
#define REG_LAUNCH(DP, NT)                                                                              \
  do {                                                                                                  \
    if (p.D == DP && p.vec)                                                                             \
      hipLaunchKernelGGL((block_select_reg_kernel<T, DP, NT, true>), reg_grid, reg_block, 0, st, p);    \
    else                                                                                                \
      hipLaunchKernelGGL((block_select_reg_kernel<T, DP, NT, false>), reg_grid, reg_block, 0, st, p);   \
    return;                                                                                             \
  } while (0)
#define REG_LAUNCH_D(NT)                 \
  do {                                   \
    if (p.D <= 32) REG_LAUNCH(32, NT);   \
    if (p.D <= 64) REG_LAUNCH(64, NT);   \
    REG_LAUNCH(128, NT);                 \
  } while (0)
  if (p.NB <= 64) REG_LAUNCH_D(4);
  if (p.NB <= 128) REG_LAUNCH_D(8);
  if (p.NB <= 256) REG_LAUNCH_D(16);
#undef REG_LAUNCH_D
#undef REG_LAUNCH
  const dim3 grid((unsigned)tiles);
  if (p.D <= 32)
    hipLaunchKernelGGL((block_select_kernel<T, 32>), grid, dim3(64), tile_lds, st, p);
  else if (p.D <= 64)
    hipLaunchKernelGGL((block_select_kernel<T, 64>), grid, dim3(64), tile_lds, st, p);
  else
    hipLaunchKernelGGL((block_select_kernel<T, 128>), grid, dim3(64), tile_lds, st, p);
}

}  // namespace
}  // namespace shrimp

extern "C" int shrimp_block_means(const void* k, int64_t k_sb, int64_t k_sh, int64_t k_sn, int dt,
                                  const int32_t* k_lens, float* means, int B, int Hk, int Sk, int D,
                                  int block, int last_only, void* stream) {
  return shrimp::means_launch(k, k_sb, k_sh, k_sn, dt, k_lens, means, B, Hk, Sk, D, block,
                              last_only != 0, stream, "block_means");
}

extern "C" int shrimp_block_select(const shrimp_block_select_args* a, void* stream) {
  using namespace shrimp;
  SHRIMP_REQUIRE(a != nullptr, "block_select: null arguments");
  SHRIMP_REQUIRE(a->dt == SHRIMP_DT_BF16 || a->dt == SHRIMP_DT_F16 || a->dt == SHRIMP_DT_F32,
                 "block_select: element type %d", a->dt);
  SHRIMP_REQUIRE(a->B >= 0 && a->H >= 0 && a->Sq >= 0 && a->Sk >= 0, "block_select: negative size");
  SHRIMP_REQUIRE(a->Hk >= 1 && a->H >= a->Hk && a->H % a->Hk == 0, "block_select: %d query heads for %d key heads",
                 a->H, a->Hk);
  SHRIMP_REQUIRE(a->D >= 1 && a->D <= MAX_D, "block_select: head dim %d outside [1, %d]", a->D, MAX_D);
  SHRIMP_REQUIRE(a->block >= 1 && a->block <= MAX_KEYS && a->Sk <= MAX_KEYS,
                 "block_select: block of %d keys of %d", a->block, a->Sk);
  SHRIMP_REQUIRE(a->topk >= 1 && a->topk <= MAX_TOPK, "block_select: topk %d outside [1, %d]", a->topk,
                 MAX_TOPK);
  const int64_t nb = ((int64_t)a->Sk + a->block - 1) / a->block;
  SHRIMP_REQUIRE(nb <= MAX_BLOCKS, "block_select: %lld blocks, at most %d", (long long)nb, MAX_BLOCKS);
  if (a->B == 0 || a->Sq == 0) return SHRIMP_OK;
  SHRIMP_REQUIRE(a->q && a->q_lens && a->k_lens && a->sel && (a->means || nb == 0),
                 "block_select: null pointer");
  SHRIMP_REQUIRE(reinterpret_cast<uintptr_t>(a->means) % 16 == 0,
                 "block_select: means must start on a 16-byte boundary");
  const int64_t rows = mul_sat({a->B, a->Hk, a->Sq});
  SHRIMP_REQUIRE(rows <= INT32_MAX && a->Sq <= MAX_KEYS, "block_select: %lld queries", (long long)rows);
  SelectParams p{a->q, a->means, a->q_lens, a->k_lens, a->sel, a->q_sb, a->q_sh, a->q_sn,
                 a->B, a->H, a->Hk, a->Sq, a->Sk, a->D, (int)nb, a->block, a->topk, a->H / a->Hk,
                 (a->Sq + 15) / 16, 0, row_vec(4, a->q, a->q_sb, a->q_sh, a->q_sn, a->D, dt_size(a->dt))};
  p.chunk = nb < 128 ? (int)(nb + 15) / 16 * 16 : 128;
  // A tile of 16 queries takes a product's time however few of them there are.
  const bool by_row = a->Sq <= 2;
  const size_t row_lds = (MAX_D + nb) * 8;
  const size_t tile_lds = (size_t)16 * (a->topk + p.chunk) * 8 + (size_t)16 * a->topk * 16;
  hipStream_t st = as_stream(stream);
  if (a->dt == SHRIMP_DT_F32)
    select_launch<float>(p, rows, row_lds, tile_lds, by_row, st);
  else if (a->dt == SHRIMP_DT_F16)
    select_launch<_Float16>(p, rows, row_lds, tile_lds, by_row, st);
  else
    select_launch<__bf16>(p, rows, row_lds, tile_lds, by_row, st);
  return check_launch("block_select");
}
