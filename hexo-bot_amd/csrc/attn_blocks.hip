// Attention of every query over its own blocks of keys.
//
//   out[b, h, i] = sum_j p_j v_j,  p = softmax_j(q . k_j / sqrt(d)),  j over the keys
//   below k_lens[b] of the blocks that sel[b, h / G, i] names (each once);
//   lse[b, h, i] = log sum_j exp(q . k_j / sqrt(d)). A row without a key: 0 and -inf.
//
// Neighbouring queries choose different blocks, so no tile of queries shares its
// keys. The chunk kernel turns the choice round: a wave owns up to 64 rows (queries x
// the G heads of a key head) with their output accumulators in LDS; its workgroup
// goes through the keys 64 at a time, read once from memory while the ones before are
// worked on, and for each block a wave gathers those of its rows that chose it, 16 to
// a matrix product. (Where LDS holds the accumulators twice, two waves share the rows and
// each takes half of the 64 keys; their halves are joined at the end.) Every (row, block)
// pair is computed once, nothing leaves the chip in between, and a row meets its blocks in
// ascending order alone, so among launches of one shape its bits depend on its own inputs
// only (and, with blocks of 16 or 32, on whether a block beside its own holds numbers that
// are not finite). Products stay transposed (S^T = K Q^T, O^T = V^T P^T): a lane's
// scores are already its part of the next product's operand; V^T's operands are put
// together from 4 keys x EPL dimensions per lane with byte permutes.
//
// Softmax in base 2 around the running maximum, statistics and accumulators in fp32;
// a weight enters its product as the sum of two numbers of the type of V (one alone put the
// error against float64 at 2.1e-3 of the result's norm in bf16 and that of dq at 2.5e-3;
// two at 1.7e-3, the rounding of the result).
#include <type_traits>

#include "capi.hpp"
#include "common.hpp"

namespace shrimp {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int STAGE = 64;   // keys in LDS at a time
constexpr int WINDOW = 64;  // blocks whose row masks a wave holds at a time, one per lane

// How a chunk workgroup divides: RUNS runs of up to R rows (one bit each in a 64-bit mask),
// and TEAMS waves per run, each with its part of a stage's keys and accumulators of its own.
// R is what a compute unit's LDS holds for one workgroup, at D = 32 for three.
template <int RUNS_, int TEAMS_, int R_>
struct Shape {
  static constexpr int RUNS = RUNS_, TEAMS = TEAMS_, R = R_, WAVES = RUNS * TEAMS;
};
template <int D>
struct NarrowShape : Shape<4, 1, D == 128 ? 48 : 64> {};
template <>
struct NarrowShape<64> : Shape<4, 2, 64> {};
typedef Shape<8, 1, 56> WideShape;  // at D = 64

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  static SHRIMP_DEV f32x4 k32(u32x4 a, u32x4 b, f32x4 c) { return mfma16x16x32(a, b, c); }
  static SHRIMP_DEV f32x4 k16(u32x2 a, u32x2 b, f32x4 c) { return mfma16x16x16(a, b, c); }
  static SHRIMP_DEV unsigned pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  // x as the sum of two numbers, four at a time. The high part is cut below |x|, so the
  // low part is neither zero nor of the other sign, and an infinity stays one under both.
  static SHRIMP_DEV void split(const float (&x)[4], u32x2& hi, u32x2& lo) {
    unsigned t[4];
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = __float_as_uint(x[i] * (1.f - 0x1p-16f));
      r[i] = x[i] - __uint_as_float(t[i] & 0xFFFF0000u);
    }
    hi = u32x2{__builtin_amdgcn_perm(t[1], t[0], 0x07060302u), __builtin_amdgcn_perm(t[3], t[2], 0x07060302u)};
    lo = u32x2{pack(r[0], r[1]), pack(r[2], r[3])};
  }
};
template <>
struct Mma<_Float16> {
  static SHRIMP_DEV f32x4 k32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static SHRIMP_DEV f32x4 k16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  static SHRIMP_DEV unsigned pack(float lo, float hi) {
    const f16x2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(unsigned, v);
  }
  static SHRIMP_DEV void split(const float (&x)[4], u32x2& hi, u32x2& lo) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const auto h = __builtin_amdgcn_cvt_pkrtz(x[i] * (1.f - 0x1p-13f), x[i + 1] * (1.f - 0x1p-13f));
      hi[i / 2] = __builtin_bit_cast(unsigned, h);
      lo[i / 2] = pack(x[i] - (float)h[0], x[i + 1] - (float)h[1]);
    }
  }
};

struct BlocksParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_sb, k_sb, v_sb;
  int q_sh, q_sn, k_sh, k_sn, v_sh, v_sn;  // below 2^31: an offset is one 32 x 32 bit product
  const int32_t* sel;
  const int32_t* q_lens;
  const int32_t* k_lens;
  uint16_t* out;
  float* lse;
  int B, H, Hk, Sq, Sk, d, block, topk;
  int group;    // query heads per key head
  unsigned recip; // r / group = r recip >> 16 for r < 64
  int queries;  // queries per run
  int chunks;   // runs of queries per (sequence, key head)
  bool wide;    // WideShape
  int groups;   // chunk workgroups per (sequence, key head)
  int stage;    // keys per stage: 2^shared whole blocks, or an equal part of one
  int shared;
  int by_xcd;   // a key head's chunks stay on one XCD
  float scale2; // log2(e) / sqrt(d)
};

// The waves of one (sequence, key head) read the same keys: with by_xcd the blocks that
// one XCD receives (every eighth) take whole key heads, so these stay in its L2.
SHRIMP_DEV bool place_chunk(const BlocksParams& p, int chunks, int64_t& bh, int& chunk) {
  const int64_t id = blockIdx.x, pairs = (int64_t)p.B * p.Hk;
  if (p.by_xcd) {
    const int64_t slot = id >> 3;
    bh = slot / chunks * 8 + (id & 7);
    chunk = (int)(slot % chunks);
  } else {
    bh = id / chunks;
    chunk = (int)(id % chunks);
  }
  return bh < pairs;
}

SHRIMP_DEV unsigned perm(unsigned hi, unsigned lo, unsigned sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}
constexpr unsigned SEL_LO = 0x05040100u, SEL_HI = 0x07060302u;

// Rows of 16-bit elements read in 32-bit words.
template <int W>
using Words = unsigned __attribute__((ext_vector_type(W)));

// KT tiles of 16 keys from key0 as the A operand of S^T = K Q^T: lane (lr, lg) has
// dimensions 32 ks + 8 lg .. + 7 of key 16 kt + lr; zero past the keys and past d.
template <int D, int KT>
SHRIMP_DEV void load_rows(const uint16_t* base, int sn, int key0, int len, int d, int lr, int lg,
                          u32x4 (&f)[KT][D / 32]) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int key = key0 + kt * 16 + lr;
    const uint16_t* row = base + (int64_t)key * sn + lg * 8;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)
      f[kt][ks] = key < len && ks * 32 + lg * 8 < d ? *reinterpret_cast<const u32x4*>(row + ks * 32)
                                                    : u32x4{0, 0, 0, 0};
  }
}

// The same keys' rows for a transposed operand: lane (lr, lg) reads, of keys
// 16 kt + 4 lg + j (j < 4), the EPL = D / 16 dimensions EPL lr .. of each.
template <int D, int KT>
struct Turned {
  static constexpr int EPL = D / 16, W = EPL / 2;
  Words<W> raw[KT][4];

  SHRIMP_DEV void load(const uint16_t* base, int sn, int key0, int len, int d, int lr, int lg) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + kt * 16 + lg * 4 + j;
        const bool ok = key < len && lr * EPL < d;
        raw[kt][j] = ok ? *reinterpret_cast<const Words<W>*>(base + (int64_t)key * sn + lr * EPL)
                        : (Words<W>)0u;
      }
  }
  // Element e of the lane's dimensions, keys 4 lg .. + 3 of tile kt, as two words.
  SHRIMP_DEV u32x2 four(int kt, int e) const {
    const unsigned s = e & 1 ? SEL_HI : SEL_LO;
    const int w = e >> 1;
    return u32x2{perm(raw[kt][1][w], raw[kt][0][w], s), perm(raw[kt][3][w], raw[kt][2][w], s)};
  }
};

// acc[e] += (dimension-major A of these keys) x (their weights of 16 rows, hi + lo); the order
// of the keys inside a product is that of the lanes' weights, the same on both sides.
template <typename T, int D, int KT>
SHRIMP_DEV void weigh(const Turned<D, KT>& v, const u32x2 (&hi)[KT], const u32x2 (&lo)[KT],
                      f32x4 (&acc)[D / 16]) {
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    if constexpr (KT == 1) {
      const u32x2 a = v.four(0, e);
      acc[e] = Mma<T>::k16(a, hi[0], acc[e]);
      acc[e] = Mma<T>::k16(a, lo[0], acc[e]);
    } else {
#pragma unroll
      for (int kt = 0; kt < KT; kt += 2) {
        const u32x2 a = v.four(kt, e), b = v.four(kt + 1, e);
        const u32x4 ab{a[0], a[1], b[0], b[1]};
        acc[e] = Mma<T>::k32(ab, u32x4{hi[kt][0], hi[kt][1], hi[kt + 1][0], hi[kt + 1][1]}, acc[e]);
        acc[e] = Mma<T>::k32(ab, u32x4{lo[kt][0], lo[kt][1], lo[kt + 1][0], lo[kt + 1][1]}, acc[e]);
      }
    }
  }
}

// What the scores of KT tiles start from: -inf for the keys past the sequence (their
// rows were read as zeros), so that no select stands between a product and its readers.
// (A branch there is more than slow: hipcc 7.2 left out the wait states that a VALU read
// of a product's result needs where a branch jumps to the read, and maxima came out wrong.)
template <int KT>
SHRIMP_DEV void score_start(int key0, int len, int lg, f32x4 (&c)[KT]) {
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[kt][i] = key0 + kt * 16 + lg * 4 + i < len ? 0.f : -INFINITY;
}

// One step of the softmax of 16 rows (row lr, keys 16 kt + 4 lg + i at the lane): from
// scores s and the row's (m, l) the weights hi + lo in T, the factor for what came before,
// and the new (m, l).
template <typename T, int KT>
SHRIMP_DEV float soft_step(const f32x4 (&s)[KT], float scale2, float& m, float& l, u32x2 (&hi)[KT],
                           u32x2 (&lo)[KT]) {
  float mx = s[0][0];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kt][i]);
  const float top = fmaxf(m, max_groups_swap(mx) * scale2);
  const float off = top == -INFINITY ? 0.f : top;  // no key yet: weights 0, not exp(nan)
  float sum = 0.f;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], scale2, -off));
      sum += w[i];
    }
    Mma<T>::split(w, hi[kt], lo[kt]);
  }
  const float alpha = __builtin_amdgcn_exp2f(m - off);
  l = fmaf(l, alpha, sum_groups_swap(sum));
  m = top;
  return alpha;
}

// Row r < 64 of a run of queries: query r / group, head r % group.
SHRIMP_DEV int row_query(const BlocksParams& p, int r) { return (int)((unsigned)r * p.recip >> 16); }

// 16-byte pieces of a row of d elements as a product's operand (lane group lg), zeros
// where `on` is false and past d.
template <int D>
SHRIMP_DEV void load_row(const uint16_t* row, bool on, int d, int lg, u32x4 (&f)[D / 32]) {
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
    f[ks] = on && ks * 32 + lg * 8 < d ? *reinterpret_cast<const u32x4*>(row + ks * 32 + lg * 8)
                                       : u32x4{0, 0, 0, 0};
}

// The same without zeros: past d a piece of the row's own again, for a product whose other
// operand is zero there. (No branch stands around a load that the next products wait for.)
template <int D>
SHRIMP_DEV void load_any(const uint16_t* row, int d, int lg, u32x4 (&f)[D / 32]) {
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
    f[ks] = *reinterpret_cast<const u32x4*>(row + min(ks * 32 + lg * 8, d - 8));
}

template <int D>
constexpr int row_floats() {
  return D + 4;  // rows 16 bytes apart in the banks
}

// ---- chunk kernel ------------------------------------------------------------------------

struct GradParams {
  const uint16_t* g;
  const float* g_lse;  // or null
  int64_t g_sb;
  int g_sh, g_sn;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float2* stat;     // (B, H, Sq): lse log2(e) (+inf: no key), delta
  uint64_t* masks;  // (B, Hk, NB, chunks): row masks of the dq kernel's waves
  float scale;
  int nb, segments; // blocks; runs of keys per (sequence, key head)
};

// What p and ds are multiplied by before they are split in fp16 numbers, whose smallest step is
// 2^-24: over thousands of keys both come near that order (4096 keys, incoming gradients of
// 2^-6: dq and dk were 2.6e-3 off in the 2-norm, now 2.1e-4, their rounding). p <= 1 stays
// below fp16's largest number; ds does up to 2000, past which the gradients of q and k
// stop being finite.
template <typename T>
struct Up {
  static constexpr bool HALF = std::is_same<T, _Float16>::value;
  static constexpr float P_LOG2 = HALF ? 15.f : 0.f, P = HALF ? 0x1p15f : 1.f, DS = HALF ? 0x1p6f : 1.f;
};

template <typename T>
SHRIMP_DEV float elem(unsigned word, int hi);
template <>
SHRIMP_DEV float elem<__bf16>(unsigned word, int hi) {
  return hi ? bf16_hi(word) : bf16_lo(word);
}
template <>
SHRIMP_DEV float elem<_Float16>(unsigned word, int hi) {
  return (float)__builtin_bit_cast(f16x2, word)[hi];
}

// LDS of a chunk workgroup, in this order.
template <int D, class S>
struct ChunkLds {
  static constexpr int R = S::R, RF = row_floats<D>(), WAVES = S::WAVES;
  static constexpr int RS = D + 8;                        // 16-bit elements of a staged row
  static constexpr int acc = 0;                           // [WAVES][R][RF] fp32, behind D of them float2 of the row
  static constexpr int mask = acc + WAVES * R * RF * 4;   // [RUNS][WINDOW] u64
  static constexpr int keys = mask + S::RUNS * WINDOW * 8;   // [2][STAGE][RS]
  static constexpr int start = keys + 2 * STAGE * RS * 2;  // [STAGE] fp32: 0, -inf past the keys
  static constexpr int large = start + STAGE * 4;          // [WAVES] words
  static constexpr int bytes = large + WAVES * 4;
  static_assert(bytes <= 160 * 1024, "a compute unit's LDS");
};

// The masks of blocks [w0, w0 + WINDOW): bit r of mask[block] = the wave's row r chose it.
SHRIMP_DEV void fill_masks(const BlocksParams& p, const int32_t* sel, int asking, int w0,
                           unsigned* mask, int lane) {
  mask[2 * lane] = mask[2 * lane + 1] = 0;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const uint64_t ones = (1ull << p.group) - 1;
  const int n = asking * p.topk;
  for (int j0 = lane; j0 < n; j0 += 64 * 8) {
    int s[8];  // eight entries in flight
#pragma unroll
    for (int u = 0; u < 8; ++u) s[u] = sel[min(j0 + u * 64, n - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * 64;
      const unsigned blk = (unsigned)s[u] - (unsigned)w0;
      if (j < n && s[u] >= w0 && blk < (unsigned)WINDOW) {
        const uint64_t bits = ones << (j / p.topk * p.group);
        if ((unsigned)bits) atomicOr(&mask[2 * blk], (unsigned)bits);
        if ((unsigned)(bits >> 32)) atomicOr(&mask[2 * blk + 1], (unsigned)(bits >> 32));
      }
    }
  }
}

// A point that x has arrived at: its load is waited for here, where the loads behind it can
// be counted, not at a use behind a branch or loop that makes the wait one for all.
template <int N>
SHRIMP_DEV void arrived(u32x4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// A bound on |x| of finite elements whose products stay finite: 2^56 for bf16, the largest
// number for fp16 (as bits without the sign).
template <typename T>
constexpr uint16_t large_bits() {
  return std::is_same<T, __bf16>::value ? (127 + 56) << 7 : 0x7C00;
}
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
SHRIMP_DEV u16x2 max_bits(u16x2 m, u32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7FFF7FFFu));
  return m;
}

SHRIMP_DEV uint64_t lane_u64(uint64_t v, int lane) {  // (lane: wave-uniform)
  return (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}

// The forward, and with BACK the gradient of q (see there). MULTI: stages of two or four
// blocks (of 32 or 16 keys).
template <typename T, int D, class S, bool BACK, bool MULTI>
__global__ __launch_bounds__(S::WAVES * 64, 1) void attn_blocks_kernel(const BlocksParams p,
                                                                      const GradParams gp) {
  extern __shared__ __align__(16) char lds[];
  using L = ChunkLds<D, S>;
  constexpr int R = L::R, RF = L::RF, RS = L::RS, RUNS = S::RUNS, TEAMS = S::TEAMS, WAVES = S::WAVES;
  constexpr int EPL = D / 16, KS = D / 32, W = EPL / 2, KT = STAGE / 16 / TEAMS;
  constexpr int LPR = D / 4;                                        // lanes of a row, four dimensions each
  constexpr int ALL = STAGE * (D / 8);                              // 16-byte pieces of a stage
  constexpr int PIECES = (ALL + WAVES * 64 - 1) / (WAVES * 64);
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4, wave = wave_id();
  const int run = wave % RUNS, team = TEAMS > 1 ? wave / RUNS : 0;  // (the teams of a run on one SIMD)
  float* acc_lds = reinterpret_cast<float*>(lds + L::acc) + wave * R * RF;
  auto stat_of = [&](int row) -> float2& { return *reinterpret_cast<float2*>(acc_lds + row * RF + D); };
  unsigned* mask_lds = reinterpret_cast<unsigned*>(lds + L::mask);
  uint16_t* k_lds = reinterpret_cast<uint16_t*>(lds + L::keys);
  uint16_t* v_lds = k_lds + STAGE * RS;
  float* start_lds = reinterpret_cast<float*>(lds + L::start);
  unsigned* large_lds = reinterpret_cast<unsigned*>(lds + L::large);
  int64_t bh;
  int grp;
  if (!place_chunk(p, p.groups, bh, grp)) return;
  const int b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  const int q_len = min(max(p.q_lens[b], 0), p.Sq), k_len = min(max(p.k_lens[b], 0), p.Sk);
  const int chunk = grp * RUNS + run;
  const int q0 = min(chunk * p.queries, p.Sq);
  const int queries = min(p.queries, p.Sq - q0);        // written
  const int asking = min(queries, max(q_len - q0, 0));  // with a choice
  const int live = (k_len + p.block - 1) / p.block;
  // rows of the wave: query q0 + r / G, head hk G + r % G
  const int first = min(q0, p.Sq - 1);  // (a row to read where the wave has none)
  const uint16_t* q = p.q + b * p.q_sb + (int64_t)(hk * p.group) * p.q_sh + (int64_t)first * p.q_sn;
  const uint16_t* g =
      BACK ? gp.g + b * gp.g_sb + (int64_t)(hk * p.group) * gp.g_sh + (int64_t)first * gp.g_sn : nullptr;
  const uint16_t* k = p.k + b * p.k_sb + (int64_t)hk * p.k_sh;
  const uint16_t* v = p.v + b * p.v_sb + (int64_t)hk * p.v_sh;
  const int32_t* sel = p.sel + (bh * p.Sq + q0) * p.topk;
  const int64_t out0 = ((int64_t)b * p.H + hk * p.group) * p.Sq + q0;  // of row 0

  for (int i = lane; i < R * D; i += 64) acc_lds[i / D * RF + i % D] = 0.f;
  if constexpr (BACK) {
    for (int r0 = 0; r0 < queries * p.group; r0 += 64 / LPR) {
      const int r = r0 + lane / LPR, c = lane % LPR;
      const bool on = r < queries * p.group;
      const int query = on ? row_query(p, r) : 0, head = on ? r - query * p.group : 0;
      const int64_t o = out0 + (int64_t)head * p.Sq + query;
      float delta = 0.f;
      if (on && c * 4 < p.d) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p.out + o * p.d + c * 4);
        const u32x2 y = *reinterpret_cast<const u32x2*>(g + (int64_t)head * gp.g_sh + (int64_t)query * gp.g_sn + c * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) delta = fmaf(elem<T>(x[e >> 1], e & 1), elem<T>(y[e >> 1], e & 1), delta);
      }
      for (int m = 1; m < LPR; m <<= 1) delta += xor_shfl(delta, m);
      if (on && c == 0) {
        if (gp.g_lse) delta -= gp.g_lse[o];
        const float lse = p.lse[o];
        const float2 st = {lse == -INFINITY ? INFINITY : lse * LOG2E, delta};
        stat_of(r) = st;
        if (team == 0) gp.stat[o] = st;
      }
    }
  } else {
    if (lane < R) stat_of(lane) = float2{-INFINITY, 0.f};  // maximum, sum
  }

  // Stage of keys from key0: requested into registers, put into LDS by `store`. Requests go
  // out without a condition (keys and dimensions past the end: the last ones again), so
  // that later waits can count them; the zeros are put in on the way to LDS.
  u32x4 kr[PIECES], vr[PIECES];
  auto request = [&](int key0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = tid + i * WAVES * 64, row = min(key0 + at / (D / 8), k_len - 1);
      const int c = min(at % (D / 8) * 8, p.d - 8);
      kr[i] = *reinterpret_cast<const u32x4*>(k + (int64_t)row * p.k_sn + c);
      vr[i] = *reinterpret_cast<const u32x4*>(v + (int64_t)row * p.v_sn + c);
    }
  };
  auto store = [&](int key0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = tid + i * WAVES * 64, row = at / (D / 8), c = at % (D / 8);
      const bool keep = row < p.stage && key0 + row < k_len && c * 8 < p.d;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        kr[i][w] = keep ? kr[i][w] : 0;
        vr[i][w] = keep ? vr[i][w] : 0;
      }
      if (ALL % (WAVES * 64) == 0 || at < ALL) {
        *reinterpret_cast<u32x4*>(k_lds + row * RS + c * 8) = kr[i];
        *reinterpret_cast<u32x4*>(v_lds + row * RS + c * 8) = vr[i];
      }
    }
    if (tid < STAGE) start_lds[tid] = tid < p.stage && key0 + tid < k_len ? 0.f : -INFINITY;
    if constexpr (MULTI) {
      u16x2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < PIECES; ++i) m = max_bits(max_bits(m, kr[i]), vr[i]);
      const uint64_t some = __ballot(m[0] >= large_bits<T>() || m[1] >= large_bits<T>());
      if (lane == 0) large_lds[wave] = some != 0;
    }
  };

  __syncthreads();
  const int shared = MULTI ? p.shared : 0, per_stage = 1 << shared;  // blocks of a stage
  const int tile_shift = 2 - shared;                                   // of its 16-key tiles per block
  const int per_team = max(per_stage / TEAMS, 1);
  const int block0 = per_stage > 1 ? team * per_team : 0;  // the team's first block of a stage
  static_assert(KT * TEAMS == 4, "a stage of four tiles");
  for (int w0 = 0; w0 < live; w0 += WINDOW) {
    if (team == 0) fill_masks(p, sel, asking, w0, mask_lds + run * 2 * WINDOW, lane);
    __syncthreads();
    const bool here = w0 + lane < live;
    uint64_t any = 0, mine = 0;
#pragma unroll
    for (int w = 0; w < RUNS; ++w) {
      const uint64_t m = here ? reinterpret_cast<const uint64_t*>(mask_lds)[w * WINDOW + lane] : 0;
      any |= m;
      if (w == run) mine = m;
    }
    if constexpr (BACK)
      if (here && team == 0 && chunk < p.chunks) gp.masks[(bh * gp.nb + w0 + lane) * p.chunks + chunk] = mine;
    uint64_t todo = __ballot(any != 0);
    const uint64_t stage_bits = (1u << per_stage) - 1;
    int at = 0, key0 = 0;  // first block (of the window) and first key of a stage with chosen blocks
    auto first_of = [&]() {
      at = __builtin_ctzll(todo) >> shared << shared;
      key0 = (w0 + at) * p.block;
    };
    if (todo == 0) {
      __syncthreads();  // the masks are read
      continue;
    }
    // to the stage behind (at, key0): of the same block, or of the next chosen one; false
    // behind the last, which is then left as it is
    auto advance = [&]() {
      if (p.stage < p.block && key0 + p.stage < min((w0 + at + 1) * p.block, k_len)) {
        key0 += p.stage;
        return true;
      }
      todo &= ~(stage_bits << at);
      if (todo == 0) return false;
      first_of();
      return true;
    };
    // the wave's rows that chose one of its blocks of the stage, and which of them; their
    // list: lane j has the j-th row (the others behind them)
    constexpr int M = MULTI ? 4 / TEAMS : 1;
    auto choice = [&](uint64_t (&mask)[M]) {
      uint64_t rows = 0;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        mask[i] = i < per_team ? lane_u64(mine, min(at + block0 + i, WINDOW - 1)) : 0;
        rows |= mask[i];
      }
      const int from = team * KT * 16;  // its first key of the stage
      return from < p.stage && key0 + from < k_len ? rows : 0;
    };
    auto list = [&](uint64_t of, int& count) {
      count = __popcll(of);
      const bool in = of >> lane & 1;
      const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(of >> 32),
                                                   __builtin_amdgcn_mbcnt_lo((unsigned)of, 0));
      return __builtin_amdgcn_ds_permute((in ? before : count + lane - before) << 2, lane);
    };
    struct Tile {  // 16 rows of a list: the lane's row and its pieces
      int row;
      bool on;
      u32x4 q[KS], g[BACK ? KS : 1];
    };
    auto gather = [&](int row_at, int count, int t, Tile& x) {
      x.on = t + lr < count;
      const int listed = __builtin_amdgcn_ds_bpermute((t + lr) << 2, row_at);
      x.row = x.on ? listed : 0;
      const int query = row_query(p, x.row), head = x.row - query * p.group;
      load_any<D>(q + (int64_t)head * p.q_sh + (int64_t)query * p.q_sn, p.d, lg, x.q);
      if constexpr (BACK) load_any<D>(g + (int64_t)head * gp.g_sh + (int64_t)query * gp.g_sn, p.d, lg, x.g);
    };

    // Pipeline: while a stage is worked on, the next one's keys are on their way into
    // registers, and its first rows too.
    first_of();
    request(key0);
    uint64_t mask[M];
    int count;
    Tile tile;
    uint64_t rows = choice(mask);
    int row_at = list(rows, count);
    gather(row_at, count, 0, tile);
    store(key0);
    bool more = advance();
    request(key0);
    __syncthreads();
    for (;;) {
      uint64_t next_mask[M];
      int next_count;
      Tile next;
      const uint64_t next_rows = choice(next_mask);
      const int next_at = list(next_rows, next_count);
      arrived(tile.q);
      if constexpr (BACK) arrived(tile.g);
      gather(next_at, next_count, 0, next);
      if (rows != 0) {
        // The blocks of a stage share their products, where a row that did not choose one has
        // scores of -inf and weights of 0; keys or values that are not finite, or large
        // enough for scores that are not, would reach it all the same (0 times infinity),
        // so such a stage goes block by block.
        unsigned large = 0;
        if constexpr (MULTI) {
#pragma unroll
          for (int w = 0; w < WAVES; ++w) large |= large_lds[w];
        }
        const int passes = MULTI && __builtin_amdgcn_readfirstlane((int)large) ? per_team : 1;
        for (int pass = 0; pass < passes; ++pass) {
          if (MULTI && passes > 1) {
            uint64_t only = mask[0];
#pragma unroll
            for (int i = 1; i < M; ++i) only = pass == i ? mask[i] : only;
            if (only == 0) continue;
            row_at = list(only, count);
            gather(row_at, count, 0, tile);
            arrived(tile.q);
            if constexpr (BACK) arrived(tile.g);
          }
          u32x4 kf[KT][KS], vf[KT][KS];
          Turned<D, KT> turned;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const int from = ((team * KT + kt) * 16 + lr) * RS + ks * 32 + lg * 8;
              kf[kt][ks] = *reinterpret_cast<const u32x4*>(k_lds + from);
              if constexpr (BACK) vf[kt][ks] = *reinterpret_cast<const u32x4*>(v_lds + from);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              turned.raw[kt][j] = *reinterpret_cast<const Words<W>*>((BACK ? k_lds : v_lds) +
                                                                    ((team * KT + kt) * 16 + lg * 4 + j) * RS + lr * EPL);
          }
          if (MULTI && passes > 1) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
              if (kt >> tile_shift != pass) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                  kf[kt][ks] = u32x4{0, 0, 0, 0};
                  if constexpr (BACK) vf[kt][ks] = u32x4{0, 0, 0, 0};
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) turned.raw[kt][j] = (Words<W>)0u;
              }
          }
          for (int t = 0;;) {
            float2 st = stat_of(tile.row);
            float* to = acc_lds + tile.row * RF + lg * EPL * 4;
            f32x4 acc[EPL];
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] = *reinterpret_cast<const f32x4*>(to + e * 4);
            f32x4 s[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[kt] = *reinterpret_cast<const f32x4*>(start_lds + (team * KT + kt) * 16 + lg * 4);
            if constexpr (MULTI) {
              // bit i: the row chose block i of the stage (and the pass is for it)
              unsigned chose = 0;
#pragma unroll
              for (int i = 0; i < M; ++i) chose |= (unsigned)(mask[i] >> tile.row & 1) << i;
              if (passes > 1) chose &= 1u << pass;
#pragma unroll
              for (int kt = 0; kt < KT; ++kt) {
                const bool none = !(chose >> (kt >> tile_shift) & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[kt][i] = none ? -INFINITY : s[kt][i];
              }
            }
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) s[kt] = Mma<T>::k32(kf[kt][ks], tile.q[ks], s[kt]);
            u32x2 hi[KT], lo[KT];
            if constexpr (BACK) {
#pragma unroll
              for (int kt = 0; kt < KT; ++kt) {
                f32x4 dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) dp = Mma<T>::k32(vf[kt][ks], tile.g[ks], dp);
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  w[i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], p.scale2, -st.x)) * (gp.scale * Up<T>::DS) * (dp[i] - st.y);
                Mma<T>::split(w, hi[kt], lo[kt]);
              }
            } else {
              const float alpha = soft_step<T, KT>(s, p.scale2, st.x, st.y, hi, lo);
#pragma unroll
              for (int e = 0; e < EPL; ++e) acc[e] *= alpha;
            }
            weigh<T, D, KT>(turned, hi, lo, acc);
            if (tile.on) {
#pragma unroll
              for (int e = 0; e < EPL; ++e) *reinterpret_cast<f32x4*>(to + e * 4) = acc[e];
              if (!BACK && lg == 0) stat_of(tile.row) = st;
            }
            // (the rows' state is read again by other lanes of the wave)
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            t += 16;
            if (t >= count) break;
            gather(row_at, count, t, tile);
            arrived(tile.q);
            if constexpr (BACK) arrived(tile.g);
          }
        }
      }
      __syncthreads();  // the stage is done with
      if (!more) break;
      store(key0);
#pragma unroll
      for (int i = 0; i < M; ++i) mask[i] = next_mask[i];
      rows = next_rows;
      row_at = next_at;
      count = next_count;
      tile = next;
      more = advance();
      request(key0);
      __syncthreads();
    }
  }

  // The teams' rows joined, around the larger maximum, in team order; each team writes its
  // part of them. (Behind the last window's barrier; without a window all is as it began.)
  const float* acc0 = reinterpret_cast<const float*>(lds + L::acc) + run * R * RF;
  const float* acc1 = acc0 + (TEAMS - 1) * RUNS * R * RF;
  for (int r0 = team * (64 / LPR); r0 < queries * p.group; r0 += TEAMS * (64 / LPR)) {
    const int r = r0 + lane / LPR, c = lane % LPR;
    if (r >= queries * p.group) continue;
    const int query = row_query(p, r), head = r - query * p.group;
    const int64_t o = out0 + (int64_t)head * p.Sq + query;
    float2 st = *reinterpret_cast<const float2*>(acc0 + r * RF + D);
    float mul0 = BACK ? 1.f / Up<T>::DS : 1.f, mul1 = mul0;
    if constexpr (!BACK) {
      if constexpr (TEAMS > 1) {
        const float2 so = *reinterpret_cast<const float2*>(acc1 + r * RF + D);
        const float top = fmaxf(st.x, so.x), off = top == -INFINITY ? 0.f : top;
        mul0 = __builtin_amdgcn_exp2f(st.x - off);
        mul1 = __builtin_amdgcn_exp2f(so.x - off);
        st = float2{top, fmaf(st.y, mul0, so.y * mul1)};
      }
      const float inv = st.y == 0.f ? 0.f : 1.f / st.y;
      mul0 *= inv, mul1 *= inv;
    }
    if (c * 4 < p.d) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // dimension 4 c + e is element dim % EPL of the product's row dim / EPL = 4 lg + i
        const int dim = c * 4 + e, rr = dim / EPL, ee = dim % EPL;
        const int from = r * RF + ((rr >> 2) * EPL + ee) * 4 + (rr & 3);
        x[e] = TEAMS > 1 ? fmaf(acc0[from], mul0, acc1[from] * mul1) : acc0[from] * mul0;
      }
      *reinterpret_cast<u32x2*>((BACK ? gp.dq : p.out) + o * p.d + c * 4) =
          u32x2{Mma<T>::pack(x[0], x[1]), Mma<T>::pack(x[2], x[3])};
    }
    if (!BACK && c == 0) p.lse[o] = st.y == 0.f ? -INFINITY : (st.x + __builtin_amdgcn_logf(st.y)) * LN2;
  }
}

// ---- few queries: a workgroup per query, its blocks dealt to the waves ----------------------

constexpr int QW = 8;  // waves

template <typename T, int D, int KT>
__global__ __launch_bounds__(QW * 64) void attn_blocks_query_kernel(const BlocksParams p) {
  constexpr int EPL = D / 16, KS = D / 32, RF = row_floats<D>();
  __shared__ float o_lds[QW][16 * RF];
  __shared__ float m_lds[QW][16], l_lds[QW][16];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4, wave = wave_id();
  const int64_t bh = blockIdx.x / p.Sq;
  const int i = (int)(blockIdx.x - bh * p.Sq);
  const int b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  const int q_len = min(max(p.q_lens[b], 0), p.Sq), k_len = min(max(p.k_lens[b], 0), p.Sk);
  const int live = i < q_len ? (k_len + p.block - 1) / p.block : 0;
  // lane t: entry t of the choice (topk <= 64), -1 where nothing is to be read
  int mine = lane < p.topk ? p.sel[(bh * p.Sq + i) * p.topk + lane] : -1;
  if (mine >= live) mine = -1;
  const uint16_t* k = p.k + b * p.k_sb + (int64_t)hk * p.k_sh;
  const uint16_t* v = p.v + b * p.v_sb + (int64_t)hk * p.v_sh;

  for (int g0 = 0; g0 < p.group; g0 += 16) {  // heads of the key head, 16 rows
    const int head = hk * p.group + g0 + lr;
    const bool on = g0 + lr < p.group;
    const uint16_t* q = p.q + b * p.q_sb + (int64_t)head * p.q_sh + (int64_t)i * p.q_sn;
    u32x4 qf[KS];
    load_row<D>(q, on, p.d, lg, qf);
    float m = -INFINITY, l = 0.f;
    f32x4 acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t = wave; t < p.topk; t += QW) {
      const int blk = __builtin_amdgcn_readlane(mine, t);
      if (blk < 0 || __builtin_ctzll(__ballot(mine == blk)) != t) continue;  // absent, or named before
      const int start = blk * p.block;
      for (int key0 = start; key0 < min(start + p.block, k_len); key0 += KT * 16) {
        u32x4 kf[KT][KS];
        load_rows<D, KT>(k, p.k_sn, key0, k_len, p.d, lr, lg, kf);
        Turned<D, KT> vf;
        vf.load(v, p.v_sn, key0, k_len, p.d, lr, lg);
        f32x4 s[KT];
        score_start<KT>(key0, k_len, lg, s);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[kt] = Mma<T>::k32(kf[kt][ks], qf[ks], s[kt]);
        u32x2 hi[KT], lo[KT];
        const float alpha = soft_step<T, KT>(s, p.scale2, m, l, hi, lo);
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] *= alpha;
        weigh<T, D, KT>(vf, hi, lo, acc);
      }
    }
    // join: every wave's rows around its own maximum, added in wave order
#pragma unroll
    for (int e = 0; e < EPL; ++e)
      *reinterpret_cast<f32x4*>(&o_lds[wave][lr * RF + (lg * EPL + e) * 4]) = acc[e];
    if (lg == 0) {
      m_lds[wave][lr] = m;
      l_lds[wave][lr] = l;
    }
    __syncthreads();
    const int rows = min(16, p.group - g0);
    for (int x = threadIdx.x; x < rows * (D / 4); x += QW * 64) {
      const int r = x / (D / 4), c = x % (D / 4);
      float top = -INFINITY;
      for (int w = 0; w < QW; ++w) top = fmaxf(top, m_lds[w][r]);
      const float off = top == -INFINITY ? 0.f : top;
      float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < QW; ++w) {
        const float f = __builtin_amdgcn_exp2f(m_lds[w][r] - off);
        sum = fmaf(l_lds[w][r], f, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dim = c * 4 + e, rr = dim / EPL, ee = dim % EPL;
          y[e] = fmaf(o_lds[w][r * RF + ((rr >> 2) * EPL + ee) * 4 + (rr & 3)], f, y[e]);
        }
      }
      const int64_t o = ((int64_t)b * p.H + hk * p.group + g0 + r) * p.Sq + i;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (c * 4 < p.d)
        *reinterpret_cast<u32x2*>(p.out + o * p.d + c * 4) =
            u32x2{Mma<T>::pack(y[0] * inv, y[1] * inv), Mma<T>::pack(y[2] * inv, y[3] * inv)};
      if (c == 0) p.lse[o] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
    }
    __syncthreads();
  }
}

// ---- gradients ----------------------------------------------------------------------------------
//
// With p = exp(s - lse), delta_i = sum_d g_id out_id - g_lse_i and
// ds_ij = p_ij (sum_d g_id v_jd - delta_i) / sqrt(d):
//   dq_i = sum_j ds_ij k_j,   dk_j = sum_i ds_ij q_i,   dv_j = sum_i p_ij g_i,
// the sums over a shared key head's queries of all its heads. Two kernels, each
// computing the scores again: dq in the chunk kernel (BACK), which
// also leaves every block's row masks and every row's (lse, delta) behind; dk and dv
// with a workgroup per run of keys, which gathers the rows of those masks, 32 to
// a product, and keeps both accumulators in registers. Every sum has one order, so
// gradients repeat bit for bit. p and ds are the sum of two numbers of the operands' type.

constexpr int GW = 4;  // waves of a workgroup at most

// One workgroup: KT tiles of 16 keys of one block. Its waves take every GW-th word of the
// block's row masks (a word: the rows of one wave of the dq kernel), 64 words at a time, list their
// rows in LDS and go through them 32 at a time; at the end the waves' sums are added in
// wave order.
template <typename T, int D, int KT>
__global__ __launch_bounds__(GW * 64) void attn_blocks_dkv_kernel(const BlocksParams p, const GradParams gp) {
  constexpr int EPL = D / 16, KS = D / 32, W = EPL / 2;
  // the lists, and at the end the sums: KT 16 keys x D dimensions x 2
  extern __shared__ char lds[];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4, wave = wave_id();
  const int waves = blockDim.x >> 6;
  uint16_t* list = reinterpret_cast<uint16_t*>(lds) + wave * (64 * 64);
  int64_t bh;
  int seg;
  if (!place_chunk(p, gp.segments, bh, seg)) return;
  const int b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  const int k_len = min(max(p.k_lens[b], 0), p.Sk);
  const int key0 = seg * KT * 16, blk = key0 / p.block;
  const uint16_t* q = p.q + b * p.q_sb + (int64_t)(hk * p.group) * p.q_sh;
  const uint16_t* g = gp.g + b * gp.g_sb + (int64_t)(hk * p.group) * gp.g_sh;
  const float2* stat = gp.stat + ((int64_t)b * p.H + hk * p.group) * p.Sq;

  f32x4 dk[KT][EPL], dv[KT][EPL];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int e = 0; e < EPL; ++e) dk[kt][e] = dv[kt][e] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (key0 < k_len) {
    u32x4 kf[KT][KS], vf[KT][KS];
    load_rows<D, KT>(p.k + b * p.k_sb + (int64_t)hk * p.k_sh, p.k_sn, key0, k_len, p.d, lr, lg, kf);
    load_rows<D, KT>(p.v + b * p.v_sb + (int64_t)hk * p.v_sh, p.v_sn, key0, k_len, p.d, lr, lg, vf);
    f32x4 start_at[KT];  // the lane's key (column lr of each tile)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const float c = key0 + kt * 16 + lr < k_len ? 0.f : -INFINITY;
      start_at[kt] = f32x4{c, c, c, c};
    }
    const uint64_t* masks = gp.masks + (bh * gp.nb + blk) * p.chunks;
    for (int c0 = 0; c0 < p.chunks; c0 += 64 * waves) {
      // list entries: lane of the word, row of its chunk
      const int word = c0 + lane * waves + wave;
      uint64_t m = word < p.chunks ? masks[word] : 0;
      int at = __popcll(m);
      const int mine = at;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_up(at, s, 64);
        if (lane >= s) at += o;
      }
      const int count = __shfl(at, 63, 64);
      at -= mine;
      while (m) {
        list[at++] = (uint16_t)(lane << 6 | __builtin_ctzll(m));
        m &= m - 1;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      // 32 rows of the list, twice: as they lie for the scores (row 16 rt + lr), and as the
      // turned operands of the gradients (rows 16 rt + 4 lg + j). Past the list its last
      // row again, with a weight of 0.
      auto locate = [&](int i, int& query, int& head) {
        const int e = list[min(i, count - 1)], r = e & 63;
        const int qi = row_query(p, r);
        query = (c0 + (e >> 6) * waves + wave) * p.queries + qi;
        head = r - qi * p.group;
      };
      struct Rows {
        u32x4 q[2][KS], g[2][KS];
      };
      auto load = [&](int t, Rows& x) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          int query, head;
          locate(t + rt * 16 + lr, query, head);
          load_any<D>(q + (int64_t)head * p.q_sh + (int64_t)query * p.q_sn, p.d, lg, x.q[rt]);
          load_any<D>(g + (int64_t)head * gp.g_sh + (int64_t)query * gp.g_sn, p.d, lg, x.g[rt]);
        }
      };
      for (int t = 0; t < count; t += 32) {
        Rows now;
        load(t, now);
        Words<W> qt[2][4], gt[2][4];
        float2 st[2][4];
        const int c = min(lr * EPL, p.d - EPL);
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = t + rt * 16 + lg * 4 + j;
            int query, head;
            locate(i, query, head);
            st[rt][j] = stat[(int64_t)head * p.Sq + query];
            st[rt][j].x = i < count ? st[rt][j].x - Up<T>::P_LOG2 : INFINITY;
            qt[rt][j] = *reinterpret_cast<const Words<W>*>(q + (int64_t)head * p.q_sh + (int64_t)query * p.q_sn + c);
            gt[rt][j] = *reinterpret_cast<const Words<W>*>(g + (int64_t)head * gp.g_sh + (int64_t)query * gp.g_sn + c);
          }
        const auto &qf = now.q, &gf = now.g;
        auto turn = [&](const Words<W> (&x)[2][4], int e) {
          const unsigned s = e & 1 ? SEL_HI : SEL_LO;
          const int w = e >> 1;
          return u32x4{perm(x[0][1][w], x[0][0][w], s), perm(x[0][3][w], x[0][2][w], s),
                       perm(x[1][1][w], x[1][0][w], s), perm(x[1][3][w], x[1][2][w], s)};
        };
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          u32x2 ph[2], pl[2], dh[2], dl[2];
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            f32x4 s = start_at[kt], dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = Mma<T>::k32(qf[rt][ks], kf[kt][ks], s);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dp = Mma<T>::k32(gf[rt][ks], vf[kt][ks], dp);
            float w[4], x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.scale2, -st[rt][i].x));
              x[i] = w[i] * (gp.scale * (Up<T>::DS / Up<T>::P)) * (dp[i] - st[rt][i].y);
            }
            Mma<T>::split(w, ph[rt], pl[rt]);
            Mma<T>::split(x, dh[rt], dl[rt]);
          }
#pragma unroll
          for (int e = 0; e < EPL; ++e) {
            const u32x4 ga = turn(gt, e), qa = turn(qt, e);
            dv[kt][e] = Mma<T>::k32(ga, u32x4{ph[0][0], ph[0][1], ph[1][0], ph[1][1]}, dv[kt][e]);
            dk[kt][e] = Mma<T>::k32(qa, u32x4{dh[0][0], dh[0][1], dh[1][0], dh[1][1]}, dk[kt][e]);
            dv[kt][e] = Mma<T>::k32(ga, u32x4{pl[0][0], pl[0][1], pl[1][0], pl[1][1]}, dv[kt][e]);
            dk[kt][e] = Mma<T>::k32(qa, u32x4{dl[0][0], dl[0][1], dl[1][0], dl[1][1]}, dk[kt][e]);
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }

  // sums of the waves, in their order: [tensor][key][RF], per key lane group, e, i
  constexpr int RF = row_floats<D>();
  float* sum = reinterpret_cast<float*>(lds);
  for (int w = 0; w < waves; ++w) {
    __syncthreads();
    if (wave != w) continue;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        f32x4* a = reinterpret_cast<f32x4*>(sum + (kt * 16 + lr) * RF + (lg * EPL + e) * 4);
        f32x4* c = reinterpret_cast<f32x4*>(sum + (KT * 16 + kt * 16 + lr) * RF + (lg * EPL + e) * 4);
        *a = w ? *a + dk[kt][e] : dk[kt][e];
        *c = w ? *c + dv[kt][e] : dv[kt][e];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * KT * 16 * (D / 4); i += blockDim.x) {
    const int c = i % (D / 4), row = i / (D / 4), key = key0 + row % (KT * 16);
    if (c * 4 >= p.d || key >= p.Sk) continue;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int dim = c * 4 + e, rr = dim / EPL, ee = dim % EPL;
      x[e] = sum[row * RF + ((rr >> 2) * EPL + ee) * 4 + (rr & 3)] * (row < KT * 16 ? 1.f / Up<T>::DS : 1.f / Up<T>::P);
    }
    uint16_t* out = (row < KT * 16 ? gp.dk : gp.dv) + (bh * p.Sk + key) * p.d + c * 4;
    *reinterpret_cast<u32x2*>(out) = u32x2{Mma<T>::pack(x[0], x[1]), Mma<T>::pack(x[2], x[3])};
  }
}

// ---- host ------------------------------------------------------------------------------------

// Few enough queries that a workgroup for each (its tile holding the G heads alone)
// beats waves that go through every block for 64 rows.
constexpr int FEW_QUERIES = 8;

int check_blocks(const shrimp_attn_blocks_args* a, bool back, const char* what) {
  SHRIMP_REQUIRE(a != nullptr, "%s: null arguments", what);
  SHRIMP_REQUIRE(a->dt == SHRIMP_DT_BF16 || a->dt == SHRIMP_DT_F16, "%s: element type %d", what, a->dt);
  SHRIMP_REQUIRE(a->B >= 0 && a->H >= 0 && a->Sq >= 0 && a->Sk >= 0, "%s: negative size", what);
  SHRIMP_REQUIRE(a->Hk >= 1 && a->H % a->Hk == 0 && a->H / a->Hk <= SHRIMP_BLOCK_MAX_GROUP,
                 "%s: %d query heads for %d key heads (at most %d each)", what, a->H, a->Hk,
                 SHRIMP_BLOCK_MAX_GROUP);
  SHRIMP_REQUIRE(a->d >= 8 && a->d <= SHRIMP_BLOCK_MAX_D && a->d % 8 == 0,
                 "%s: head dim %d is not a multiple of 8 in [8, %d]", what, a->d, SHRIMP_BLOCK_MAX_D);
  SHRIMP_REQUIRE(a->block >= 16 && a->block % 16 == 0 && a->block <= (1 << 20),
                 "%s: blocks of %d keys, a multiple of 16 expected", what, a->block);
  SHRIMP_REQUIRE(a->topk >= 1 && a->topk <= SHRIMP_BLOCK_MAX_TOPK, "%s: topk %d outside [1, %d]", what,
                 a->topk, SHRIMP_BLOCK_MAX_TOPK);
  SHRIMP_REQUIRE(a->Sq <= (1 << 30) && a->Sk <= (1 << 30), "%s: Sq=%d, Sk=%d", what, a->Sq, a->Sk);
  SHRIMP_REQUIRE(a->scale > 0.f, "%s: scale must be positive", what);
  auto aligned = [](const void* base, int64_t sb, int64_t sh, int64_t sn) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && sb % 8 == 0 && sh % 8 == 0 && sn % 8 == 0 &&
           strides_ok({sh, sn});
  };
  const bool rows = a->B > 0 && a->H > 0 && a->Sq > 0, keys = a->B > 0 && a->Sk > 0 && (rows || back);
  SHRIMP_REQUIRE(!rows || (a->q && a->sel && a->q_lens && a->k_lens && a->out && a->lse),
                 "%s: null pointer", what);
  SHRIMP_REQUIRE(!keys || (a->k && a->v && a->k_lens), "%s: null k, v or k_lens", what);
  SHRIMP_REQUIRE(!rows || (aligned(a->q, a->q_sb, a->q_sh, a->q_sn) && aligned(a->out, 0, 0, 0)),
                 "%s: rows must start on 16-byte boundaries, strides be below 2^31", what);
  SHRIMP_REQUIRE(!keys || (aligned(a->k, a->k_sb, a->k_sh, a->k_sn) && aligned(a->v, a->v_sb, a->v_sh, a->v_sn)),
                 "%s: rows must start on 16-byte boundaries, strides be below 2^31", what);
  return SHRIMP_OK;
}

// Keys that a wave of the other two kernels scores at once (16 KT): the most of 64, 32 and
// 16 that divide a block.
int key_step(int block) { return block % 64 == 0 ? 64 : block % 32 == 0 ? 32 : 16; }

BlocksParams blocks_params(const shrimp_attn_blocks_args* a) {
  BlocksParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.q_sb = a->q_sb, p.q_sh = (int)a->q_sh, p.q_sn = (int)a->q_sn;
  p.k_sb = a->k_sb, p.k_sh = (int)a->k_sh, p.k_sn = (int)a->k_sn;
  p.v_sb = a->v_sb, p.v_sh = (int)a->v_sh, p.v_sn = (int)a->v_sn;
  p.sel = a->sel;
  p.q_lens = a->q_lens;
  p.k_lens = a->k_lens;
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  p.B = a->B, p.H = a->H, p.Hk = a->Hk, p.Sq = a->Sq, p.Sk = a->Sk;
  p.d = a->d, p.block = a->block, p.topk = a->topk;
  p.group = a->H / a->Hk;
  p.recip = p.group > 0 ? (65536u + p.group - 1) / p.group : 0;
  const int64_t pairs = (int64_t)a->B * a->Hk;
  // At D = 64 the wide shape serves 1.75 times the rows at a time, but takes 1.37 times as
  // long for a workgroup: whichever ends first on 256 compute units. 8 heads of 8100 queries,
  // 16 blocks of 64: narrow 188 us, wide 261; the same with 64 heads 1516 and 1306.
  auto groups = [&](int runs, int rows) {
    const int64_t most = (int64_t)runs * (p.group > 0 ? rows / p.group : rows);
    return (a->Sq + most - 1) / most;
  };
  int runs = 4, rows = a->d > 64 ? NarrowShape<128>::R : NarrowShape<64>::R;
  if (a->d > 32 && a->d <= 64) {
    auto rounds = [&](int64_t n) { return (mul_sat({pairs, n}) - 1) / 256 + 1; };
    p.wide = rounds(groups(WideShape::RUNS, WideShape::R)) / 8.0 < rounds(groups(runs, rows)) / 11.0;
    if (p.wide) runs = WideShape::RUNS, rows = WideShape::R;
  }
  p.groups = (int)groups(runs, rows);
  // the queries dealt evenly to the runs of all workgroups
  const int64_t all = (int64_t)p.groups * runs;
  p.queries = all > 0 ? (int)((a->Sq + all - 1) / all) : 1;
  p.chunks = (a->Sq + p.queries - 1) / p.queries;
  // whole blocks of up to 64 keys together, or the largest equal part of a longer block
  p.stage = 16;
  p.shared = a->block == 16 ? 2 : a->block == 32 ? 1 : 0;
  if (a->block <= STAGE)
    p.stage = a->block << p.shared;
  else
    for (int keys = STAGE; keys > 16; keys -= 16)
      if (a->block % keys == 0) {
        p.stage = keys;
        break;
      }
  p.by_xcd = pairs % 8 == 0 || pairs >= 64;
  p.scale2 = a->scale * LOG2E;
  return p;
}

template <typename T, int D, class S, bool BACK>
int launch_shape(const BlocksParams& p, const GradParams& gp, unsigned blocks, hipStream_t st) {
  constexpr int bytes = ChunkLds<D, S>::bytes;
  SHRIMP_REQUIRE(bytes <= max_lds_per_block(), "attn_blocks: %d bytes of LDS, %d available", bytes,
                 max_lds_per_block());
  const dim3 grid(blocks), threads(S::WAVES * 64);
  if (p.shared)
    hipLaunchKernelGGL((attn_blocks_kernel<T, D, S, BACK, true>), grid, threads, bytes, st, p, gp);
  else
    hipLaunchKernelGGL((attn_blocks_kernel<T, D, S, BACK, false>), grid, threads, bytes, st, p, gp);
  return SHRIMP_OK;
}

template <typename T, int D, bool BACK>
int launch_chunk(const BlocksParams& p, const GradParams& gp, unsigned blocks, hipStream_t st) {
  if constexpr (D == 64)
    if (p.wide) return launch_shape<T, D, WideShape, BACK>(p, gp, blocks, st);
  return launch_shape<T, D, NarrowShape<D>, BACK>(p, gp, blocks, st);
}

template <typename T, int D, int KT>
int launch_forward(const BlocksParams& p, hipStream_t st) {
  if (p.Sq <= FEW_QUERIES) {
    const int64_t n = mul_sat({p.B, p.Hk, p.Sq});
    SHRIMP_REQUIRE(n <= INT32_MAX, "attn_blocks: %lld queries", (long long)n);
    hipLaunchKernelGGL((attn_blocks_query_kernel<T, D, KT>), dim3((unsigned)n), dim3(QW * 64), 0, st, p);
    return SHRIMP_OK;
  }
  const int64_t pairs = (int64_t)p.B * p.Hk;
  const int64_t n = mul_sat({p.by_xcd ? (pairs + 7) / 8 * 8 : pairs, p.groups});
  SHRIMP_REQUIRE(n <= INT32_MAX, "attn_blocks: %lld groups of queries", (long long)n);
  return launch_chunk<T, D, false>(p, GradParams{}, (unsigned)n, st);
}

template <typename T, int D>
int launch_forward_kt(const BlocksParams& p, hipStream_t st) {
  if (key_step(p.block) == 64) return launch_forward<T, D, 4>(p, st);
  if (key_step(p.block) == 32) return launch_forward<T, D, 2>(p, st);
  return launch_forward<T, D, 1>(p, st);
}

template <typename T>
int launch_forward_d(const BlocksParams& p, hipStream_t st) {
  if (p.d <= 32) return launch_forward_kt<T, 32>(p, st);
  if (p.d <= 64) return launch_forward_kt<T, 64>(p, st);
  return launch_forward_kt<T, 128>(p, st);
}

int64_t grad_stat_bytes(const shrimp_attn_blocks_args* a) {
  return mul_sat({a->B, a->H, a->Sq, 8});
}
int64_t grad_mask_bytes(const shrimp_attn_blocks_args* a) {
  const BlocksParams p = blocks_params(a);
  return mul_sat({a->B, a->Hk, ((int64_t)a->Sk + a->block - 1) / a->block, p.chunks, 8});
}

// Tiles of 16 keys that a workgroup of the dk / dv kernel takes: every row is gathered once
// for all of them, but their two accumulators are registers. At D = 64 32 keys leave two
// waves per SIMD (2 x 8 heads x 4096 in pairs, 8 blocks of 64: 84 us, 64 keys 92); at
// D = 128 there is one either way (16 heads x 8192, 16 blocks of 64, the whole backward:
// 1717 us, with 16 keys 2049).
template <int D, int KT>
constexpr int key_tiles() {
  return D >= 64 && KT == 4 ? 2 : KT;
}

template <typename T, int D, int KT>
int launch_backward(const BlocksParams& p, GradParams gp, hipStream_t st) {
  constexpr int KG = key_tiles<D, KT>();
  const int64_t pairs = (int64_t)p.B * p.Hk, sets = p.by_xcd ? (pairs + 7) / 8 * 8 : pairs;
  const int64_t n = mul_sat({sets, p.groups});
  gp.segments = (p.Sk + KG * 16 - 1) / (KG * 16);
  const int64_t m = mul_sat({sets, gp.segments});
  SHRIMP_REQUIRE(n <= INT32_MAX && m <= INT32_MAX, "attn_blocks_backward: %lld chunks of queries, %lld of keys",
                 (long long)n, (long long)m);
  if (n > 0) {
    const int rc = launch_chunk<T, D, true>(p, gp, (unsigned)n, st);
    if (rc != SHRIMP_OK) return rc;
  }
  if (m > 0) {
    // waves by the rows that a block has on average: tiles of 32 that stay full
    const int64_t rows = (int64_t)p.Sq * p.group * p.topk / (gp.nb > 0 ? gp.nb : 1);
    const int waves = rows >= 256 ? GW : rows >= 128 ? 2 : 1;
    const size_t list = (size_t)waves * 64 * 64 * 2, sum = (size_t)2 * KG * 16 * row_floats<D>() * 4;
    hipLaunchKernelGGL((attn_blocks_dkv_kernel<T, D, KG>), dim3((unsigned)m), dim3(waves * 64),
                       list > sum ? list : sum, st, p, gp);
  }
  return SHRIMP_OK;
}

template <typename T, int D>
int launch_backward_kt(const BlocksParams& p, const GradParams& gp, hipStream_t st) {
  if (key_step(p.block) == 64) return launch_backward<T, D, 4>(p, gp, st);
  if (key_step(p.block) == 32) return launch_backward<T, D, 2>(p, gp, st);
  return launch_backward<T, D, 1>(p, gp, st);
}

template <typename T>
int launch_backward_d(const BlocksParams& p, const GradParams& gp, hipStream_t st) {
  if (p.d <= 32) return launch_backward_kt<T, 32>(p, gp, st);
  if (p.d <= 64) return launch_backward_kt<T, 64>(p, gp, st);
  return launch_backward_kt<T, 128>(p, gp, st);
}

}  // namespace
}  // namespace shrimp

extern "C" int shrimp_attn_blocks(const shrimp_attn_blocks_args* a, void* stream) {
  using namespace shrimp;
  const int rc = check_blocks(a, false, "attn_blocks");
  if (rc != SHRIMP_OK) return rc;
  if (a->B == 0 || a->H == 0 || a->Sq == 0) return SHRIMP_OK;
  const BlocksParams p = blocks_params(a);
  const int e = a->dt == SHRIMP_DT_F16 ? launch_forward_d<_Float16>(p, as_stream(stream))
                                       : launch_forward_d<__bf16>(p, as_stream(stream));
  if (e != SHRIMP_OK) return e;
  return check_launch("attn_blocks");
}

extern "C" int64_t shrimp_attn_blocks_workspace(const shrimp_attn_blocks_args* a) {
  using namespace shrimp;
  if (check_blocks(a, true, "attn_blocks_workspace") != SHRIMP_OK) return -1;
  const int64_t stat = grad_stat_bytes(a), mask = grad_mask_bytes(a);
  return stat > INT64_MAX - mask ? INT64_MAX : stat + mask;
}

extern "C" int shrimp_attn_blocks_backward(const shrimp_attn_blocks_args* a,
                                           const shrimp_attn_blocks_grads* g, void* stream) {
  using namespace shrimp;
  const int rc = check_blocks(a, true, "attn_blocks_backward");
  if (rc != SHRIMP_OK) return rc;
  SHRIMP_REQUIRE(g != nullptr, "attn_blocks_backward: null gradients");
  if (a->B == 0) return SHRIMP_OK;
  const bool rows = a->H > 0 && a->Sq > 0;
  SHRIMP_REQUIRE(!rows || (g->g && g->dq), "attn_blocks_backward: null gradient of out or q");
  SHRIMP_REQUIRE(a->Sk == 0 || (g->dk && g->dv), "attn_blocks_backward: null gradient of k or v");
  SHRIMP_REQUIRE(reinterpret_cast<uintptr_t>(g->g) % 16 == 0 && g->g_sb % 8 == 0 && g->g_sh % 8 == 0 &&
                     g->g_sn % 8 == 0 && strides_ok({g->g_sh, g->g_sn}) && reinterpret_cast<uintptr_t>(g->dq) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(g->dk) % 16 == 0 && reinterpret_cast<uintptr_t>(g->dv) % 16 == 0,
                 "attn_blocks_backward: gradients must start on 16-byte boundaries");
  const int64_t stat = grad_stat_bytes(a), mask = grad_mask_bytes(a);
  SHRIMP_REQUIRE(g->workspace_bytes >= stat && g->workspace_bytes - stat >= mask &&
                     (g->workspace || stat + mask == 0) && reinterpret_cast<uintptr_t>(g->workspace) % 8 == 0,
                 "attn_blocks_backward: workspace of %lld bytes, %lld + %lld needed",
                 (long long)g->workspace_bytes, (long long)stat, (long long)mask);
  BlocksParams p = blocks_params(a);
  if (!rows) p.groups = p.chunks = 0;  // (no heads: the keys' gradients are zero)
  GradParams gp{};
  gp.g = static_cast<const uint16_t*>(g->g);
  gp.g_lse = g->g_lse;
  gp.g_sb = g->g_sb, gp.g_sh = (int)g->g_sh, gp.g_sn = (int)g->g_sn;
  gp.dq = static_cast<uint16_t*>(g->dq);
  gp.dk = static_cast<uint16_t*>(g->dk);
  gp.dv = static_cast<uint16_t*>(g->dv);
  gp.stat = static_cast<float2*>(g->workspace);
  gp.masks = reinterpret_cast<uint64_t*>(static_cast<char*>(g->workspace) + stat);
  gp.scale = a->scale;
  gp.nb = (a->Sk + a->block - 1) / a->block;
  const int e = a->dt == SHRIMP_DT_F16 ? launch_backward_d<_Float16>(p, gp, as_stream(stream))
                                       : launch_backward_d<__bf16>(p, gp, as_stream(stream));
  if (e != SHRIMP_OK) return e;
  return check_launch("attn_blocks_backward");
}
