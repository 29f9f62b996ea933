// Rotation of head dimensions by positions on several axes, alone and after an
// RMS norm of every query and key head, and the gradients of both.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps), n_d = x_d r w_d      (norm form only)
//   theta_p = pos[axis(p)] freqs[p]                        (P pairs, sections of axes)
//   (a, b) -> (a cos theta - b sin theta, b cos theta + a sin theta)
// Pair p is dimensions (p, P + p), or (2 p, 2 p + 1) interleaved; the D - 2 P
// dimensions behind the pairs pass. The rotation's gradient is its inverse; with
// u = R^T g the norm's are dw_d = sum u_d x_d r and
//   dx_d = r (u_d w_d - x_d r^2 mean_e(u_e w_e x_e)).
//
// Bound: HBM, one read of every input and one write of every output. A thread
// keeps one unit (V pairs, two vector accesses of up to 16 bytes) of one token and
// goes through its heads of q and then of k, four at a time in flight, so an
// angle is worked out once for all the heads that share it: in float64 (a position
// of 400000 at frequency 1 has lost 2^-6 rad in fp32), reduced to +-pi/4 there, then
// Taylor polynomials in fp32. Threads of a wave take a head's units first, then
// heads or tokens, whichever lie beside them in memory, until a wave reads runs of
// 256 bytes.
#include "capi.hpp"
#include "common.hpp"

namespace shrimp {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_AXES = SHRIMP_ROPE_MAX_AXES;
constexpr int MAX_D = 256;
// Elements of an access: 8 bytes of 16-bit elements beat 16, whose units need twice
// the registers (backward of 512 boards' q and k, 16 heads of 16: 75 against 112 us;
// 2 x 8190 x 40 heads of 128: 125 against 143).
constexpr int VEC = 4;

struct RopeTensor {
  const void* x;
  const void* g;  // backward: gradient of the output
  const void* w;  // norm weight, or null
  void* out;
  float* part;    // backward: [block][D] partial weight gradients
  int64_t x_sb, x_sh, x_sn, g_sb, g_sh, g_sn;
  int heads, groups;
};

struct RopeParams {
  RopeTensor t[2];
  const void* pos;
  const void* freqs;
  int64_t p_sb, p_sn, p_sa;
  int pos_dt, freq_f64, w_dt;
  int axes, cut[MAX_AXES - 1];  // pair at which axis i + 1 begins
  float eps, sign, inv_d;
  int tokens, S, D, P;
  int lanes, head_lanes;  // lanes per head, heads across lanes
  int groups_per_block;   // head groups (of q, then of k) per blockIdx.y
  int q_rows;             // backward: blockIdx.y below takes q alone, the others k alone
  int interleaved;
};

template <typename T, int V>
using Vec = T __attribute__((ext_vector_type(V)));

SHRIMP_DEV float load_weight(const void* w, int dt, int i) {
  if (dt == SHRIMP_DT_F32) return static_cast<const float*>(w)[i];
  if (dt == SHRIMP_DT_F16) return (float)static_cast<const _Float16*>(w)[i];
  return (float)static_cast<const __bf16*>(w)[i];
}

SHRIMP_DEV double load_pos(const void* p, int dt, int64_t i) {
  if (dt == SHRIMP_DT_I32) return (double)static_cast<const int32_t*>(p)[i];
  if (dt == SHRIMP_DT_I64) return (double)static_cast<const int64_t*>(p)[i];
  return (double)static_cast<const float*>(p)[i];
}

// cos and sin of t: t - n pi/2 in float64 (pi/2 as two numbers), then the Taylor
// polynomials, whose first dropped terms at pi/4 are 1.8e-9 and 1.1e-10.
SHRIMP_DEV void cos_sin(double t, float& c, float& s) {
  const double n = __builtin_rint(t * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489661923, t);
  r = __builtin_fma(-n, 6.123233995736766036e-17, r);
  const int quad = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  const float x = (float)r, x2 = x * x;
  float ps = fmaf(x2, 1.f / 362880, -1.f / 5040);
  ps = fmaf(x2, ps, 1.f / 120);
  ps = fmaf(x2, ps, -1.f / 6);
  ps = fmaf(x * x2, ps, x);
  float pc = fmaf(x2, -1.f / 3628800, 1.f / 40320);
  pc = fmaf(x2, pc, -1.f / 720);
  pc = fmaf(x2, pc, 1.f / 24);
  pc = fmaf(x2, pc, -0.5f);
  pc = fmaf(x2, pc, 1.f);
  const float cc = (quad & 1) ? ps : pc, ss = (quad & 1) ? pc : ps;
  c = (quad == 1 || quad == 2) ? -cc : cc;
  s = (quad >= 2) ? -ss : ss;
}

// Sum over aligned groups of `lanes` lanes (a power of two up to 64).
SHRIMP_DEV float lanes_sum(float v, int lanes) {
  for (int m = 1; m < lanes; m <<= 1) v += xor_shfl(v, m);
  return v;
}

// F: groups of heads loaded together, while the F before them are worked on.
template <typename T, int V, int F, bool NORM, bool BACK>
__global__ __launch_bounds__(THREADS) void rope_kernel(const RopeParams p) {
  constexpr int NU = V == 1 ? 2 : 1;  // units per lane: 128 units of one pair at D = 256
  __shared__ float shared[THREADS * 2 * V];  // angles, then the block's weight gradients
  const int tid = threadIdx.x;
  const int per_token = p.lanes * p.head_lanes;
  const int ul = tid & (p.lanes - 1);
  const int hl = (tid & (per_token - 1)) / p.lanes;
  const int per_block = THREADS / per_token;
  const int rot_units = p.P / V;

  // the unit's two accesses; they rotate into each other (rot) or pass. An odd
  // rest ends in one element (V = 1 only), and lanes past the units hold none.
  int off0[NU], off1[NU];
  bool n0[NU], n1[NU], rot[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = ul + i * 64;
    rot[i] = u < rot_units;
    off0[i] = rot[i] ? (p.interleaved ? 2 * u * V : u * V) : 2 * p.P + (u - rot_units) * 2 * V;
    off1[i] = rot[i] && !p.interleaved ? p.P + u * V : off0[i] + V;
    n0[i] = off0[i] + V <= p.D;
    n1[i] = off1[i] + V <= p.D;
  }

  const int q_groups = p.t[0].groups;
  // forward: a block's heads may be of q and of k, and share their angles; backward:
  // of one tensor, whose weight and its gradient take the registers of one
  constexpr int NT = BACK ? 1 : 2;
  const int of_k = BACK && (int)blockIdx.y >= p.q_rows;
  const int first = of_k ? q_groups + (blockIdx.y - p.q_rows) * p.groups_per_block
                         : blockIdx.y * p.groups_per_block;
  const int last = min(first + p.groups_per_block,
                       BACK && !of_k ? q_groups : q_groups + p.t[1].groups);
  const int64_t stride = (int64_t)gridDim.x * per_block;
  struct Place {  // one token: its rows' offsets in q and k, and its position
    int64_t x[NT], g[NT];
    int b, s;
    Vec<double, MAX_AXES> at;  // (an array would be indexed in memory)
    bool live;
  };
  auto locate = [&](int64_t tok) {
    Place w{};
    w.live = tok < p.tokens;
    const int i = w.live ? (int)tok : 0;
    w.b = i / p.S;
    w.s = i - w.b * p.S;
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const RopeTensor& t = p.t[BACK ? of_k : k];
      w.x[k] = w.b * t.x_sb + w.s * t.x_sn;
      if constexpr (BACK) w.g[k] = w.b * t.g_sb + w.s * t.g_sn;
    }
#pragma unroll
    for (int a = 0; a < MAX_AXES; ++a)
      w.at[a] = a < p.axes && p.P > 0
                    ? load_pos(p.pos, p.pos_dt, w.b * p.p_sb + w.s * p.p_sn + a * p.p_sa) : 0.0;
    return w;
  };
  struct Rows {
    Vec<T, V> x[F][NU][2], g[BACK ? F : 1][NU][2];
  };
  auto load = [&](int64_t xq, int64_t xk, int64_t gx, bool live, int g0, Rows& v) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const bool k = BACK ? of_k : g0 + f >= q_groups;
      const RopeTensor& t = p.t[k];
      const int head = (g0 + f - (k ? q_groups : 0)) * p.head_lanes + hl;
      const bool on = live && g0 + f < last && head < t.heads;
      const T* x = static_cast<const T*>(t.x) + (k ? xk : xq) + head * t.x_sh;
      const T* g = static_cast<const T*>(t.g) + gx + head * t.g_sh;
      const Vec<T, V> zero = (T)0.f;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        v.x[f][i][0] = on && n0[i] ? *reinterpret_cast<const Vec<T, V>*>(x + off0[i]) : zero;
        v.x[f][i][1] = on && n1[i] ? *reinterpret_cast<const Vec<T, V>*>(x + off1[i]) : zero;
        if constexpr (BACK) {
          v.g[f][i][0] = on && n0[i] ? *reinterpret_cast<const Vec<T, V>*>(g + off0[i]) : zero;
          v.g[f][i][1] = on && n1[i] ? *reinterpret_cast<const Vec<T, V>*>(g + off1[i]) : zero;
        }
      }
    }
  };

  int64_t base = (int64_t)blockIdx.x * per_block;
  Place now = locate(base + tid / per_token);
  Rows rows;
  load(now.x[0], now.x[NT - 1], now.g[0], now.live, first, rows);
  float wgt[NT][NU][2 * V], dw[NU][2 * V];
  if constexpr (NORM) {
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const void* w = p.t[BACK ? of_k : k].w;
          wgt[k][i][e] = w && n0[i] ? load_weight(w, p.w_dt, off0[i] + e) : 0.f;
          wgt[k][i][V + e] = w && n1[i] ? load_weight(w, p.w_dt, off1[i] + e) : 0.f;
          dw[i][e] = dw[i][V + e] = 0.f;
        }
  }

  for (; base < p.tokens; base += stride) {
    auto angle = [&](int pair, float& c, float& s) {
      double at = now.at[0];
#pragma unroll
      for (int a = 1; a < MAX_AXES; ++a) at = pair >= p.cut[a - 1] ? now.at[a] : at;
      const double f = p.freq_f64 ? static_cast<const double*>(p.freqs)[pair]
                                  : (double)static_cast<const float*>(p.freqs)[pair];
      cos_sin(at * f, c, s);
      s *= p.sign;
    };
    float cs[NU][V], sn[NU][V];
    if (p.head_lanes == 1) {
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          cs[i][e] = 1.f;
          sn[i][e] = 0.f;
          if (rot[i]) angle((ul + i * 64) * V + e, cs[i][e], sn[i][e]);
        }
    } else {
      // the lanes that hold a token's unit for several heads, all of one wave,
      // share its angles out
      const int slot = (tid / per_token * p.lanes + ul) * 2 * V;
      for (int e = hl; e < V; e += p.head_lanes) {
        float c = 1.f, s = 0.f;
        if (rot[0]) angle(ul * V + e, c, s);
        shared[slot + e] = c;
        shared[slot + V + e] = s;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int e = 0; e < V; ++e) {
        cs[0][e] = shared[slot + e];
        sn[0][e] = shared[slot + V + e];
        if constexpr (NU == 2) {  // more than one head: at most 32 units
          cs[1][e] = 1.f;
          sn[1][e] = 0.f;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    const Place next = locate(base + stride + tid / per_token);

    for (int g0 = first; g0 < last; g0 += F) {
      const Rows cur = rows;
      const bool end = g0 + F >= last;
      load(end ? next.x[0] : now.x[0], end ? next.x[NT - 1] : now.x[NT - 1],
           end ? next.g[0] : now.g[0], end ? next.live : now.live, end ? first : g0 + F, rows);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        if (g0 + f >= last) break;
        const bool k = BACK ? of_k : g0 + f >= q_groups;
        const RopeTensor& t = p.t[k];
        const int head = (g0 + f - (k ? q_groups : 0)) * p.head_lanes + hl;
        float y[NU][2 * V];  // what is rotated: x, x r w, or the gradient
        float r = 1.f;
        if constexpr (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) {
              const float v = (float)cur.x[f][i][e / V][e % V];
              ss = fmaf(v, v, ss);
            }
          r = rsqrtf(fmaf(lanes_sum(ss, p.lanes), p.inv_d, p.eps));
        }
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) {
            if constexpr (BACK)
              y[i][e] = (float)cur.g[f][i][e / V][e % V];
            else
              y[i][e] = (float)cur.x[f][i][e / V][e % V];
            if constexpr (NORM && !BACK) y[i][e] *= r * (k ? wgt[NT - 1][i][e] : wgt[0][i][e]);
          }
        // the gradient's rotation is the inverse; the sign of the sines says which
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          if (!rot[i]) continue;
          auto turn = [&](float& a, float& c, int e) {
            const float a0 = a, c0 = c;
            a = a0 * cs[i][e] - c0 * sn[i][e];
            c = c0 * cs[i][e] + a0 * sn[i][e];
          };
          if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < V; ++e) turn(y[i][2 * e], y[i][2 * e + 1], e);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) turn(y[i][e], y[i][V + e], e);
          }
        }
        if constexpr (BACK) {
          float dot = 0.f;
#pragma unroll
          for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) {
              const float v = (float)cur.x[f][i][e / V][e % V];
              dw[i][e] = fmaf(y[i][e], v * r, dw[i][e]);
              y[i][e] *= wgt[0][i][e];
              dot = fmaf(y[i][e], v, dot);
            }
          const float q = lanes_sum(dot, p.lanes) * p.inv_d * r * r;
#pragma unroll
          for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < 2 * V; ++e)
              y[i][e] = r * (y[i][e] - (float)cur.x[f][i][e / V][e % V] * q);
        }
        if (now.live && head < t.heads) {
          T* o = static_cast<T*>(t.out) + (((int64_t)now.b * t.heads + head) * p.S + now.s) * p.D;
#pragma unroll
          for (int i = 0; i < NU; ++i) {
            Vec<T, V> o0, o1;
#pragma unroll
            for (int e = 0; e < V; ++e) {
              o0[e] = (T)y[i][e];
              o1[e] = (T)y[i][V + e];
            }
            if (n0[i]) *reinterpret_cast<Vec<T, V>*>(o + off0[i]) = o0;
            if (n1[i]) *reinterpret_cast<Vec<T, V>*>(o + off1[i]) = o1;
          }
        }
      }
    }
    now = next;
  }

  if constexpr (BACK) {
    // the block's weight gradients: threads of one unit added in thread order
    const int block = (blockIdx.y - (of_k ? p.q_rows : 0)) * gridDim.x + blockIdx.x;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) shared[e * THREADS + tid] = dw[i][e];
      __syncthreads();
      for (int j = tid; j < p.lanes * 2 * V; j += THREADS) {
        const int e = j / p.lanes, l = j % p.lanes, u = l + i * 64;
        const bool r = u < rot_units;
        const int o0 = r ? (p.interleaved ? 2 * u * V : u * V) : 2 * p.P + (u - rot_units) * 2 * V;
        const int d = e < V ? o0 + e : (r && !p.interleaved ? p.P + u * V : o0 + V) + e - V;
        if (d >= p.D) continue;
        float sum = 0.f;
        for (int t = l; t < THREADS; t += p.lanes) sum += shared[e * THREADS + t];
        p.t[of_k].part[(int64_t)block * p.D + d] = sum;
      }
    }
  }
}

// Weight gradients from the blocks' partial sums, in float64 and in block order:
// workgroup (column block, tensor), 16 columns x 16 interleaved runs of blocks.
__global__ __launch_bounds__(THREADS) void rope_dw_kernel(const float* part_q, const float* part_k,
                                                          int blocks_q, int blocks_k, int D,
                                                          void* dw_q, void* dw_k, int dt) {
  __shared__ double acc[16][17];
  const float* part = blockIdx.y ? part_k : part_q;
  const int blocks = blockIdx.y ? blocks_k : blocks_q;
  void* dw = blockIdx.y ? dw_k : dw_q;
  const int c = threadIdx.x & 15, run = threadIdx.x >> 4, d = blockIdx.x * 16 + c;
  double sum = 0.0;
  if (d < D) {
#pragma unroll 8
    for (int i = run; i < blocks; i += 16) sum += (double)part[(int64_t)i * D + d];
  }
  acc[run][c] = sum;
  __syncthreads();
  if (run == 0 && d < D) {
    for (int i = 1; i < 16; ++i) sum += acc[i][c];
    if (dt == SHRIMP_DT_F32)
      static_cast<float*>(dw)[d] = (float)sum;
    else if (dt == SHRIMP_DT_F16)
      static_cast<_Float16*>(dw)[d] = (_Float16)(float)sum;
    else
      static_cast<__bf16*>(dw)[d] = (__bf16)(float)sum;
  }
}

int element_size(int dt) { return dt == SHRIMP_DT_F32 ? 4 : 2; }

int pow2_ceil(int n) {
  int v = 1;
  while (v < n) v <<= 1;
  return v;
}

struct RopePlan {
  RopeParams p;
  int vec, flight, grid_x, grid_y;
};

// Blocks of a launch per tensor: enough to fill the compute units, each with several
// tokens whose reads are in flight under the token before (and, backward, few enough
// that their partial weight gradients, 4 D bytes each, stay a small read).
constexpr int FULL_BLOCKS = 1024;

int plan_rope(const shrimp_rope_args* a, bool back, RopePlan* out, const char* what) {
  SHRIMP_REQUIRE(a != nullptr, "%s: null arguments", what);
  SHRIMP_REQUIRE(a->dt == SHRIMP_DT_BF16 || a->dt == SHRIMP_DT_F16 || a->dt == SHRIMP_DT_F32,
                 "%s: element type %d", what, a->dt);
  SHRIMP_REQUIRE(a->B >= 0 && a->S >= 0 && a->H >= 0 && a->Hk >= 0, "%s: negative size", what);
  SHRIMP_REQUIRE((int64_t)a->B * a->S <= INT32_MAX / 2, "%s: B * S = %lld tokens", what,
                 (long long)a->B * a->S);
  SHRIMP_REQUIRE(a->H <= 65536 && a->Hk <= 65536, "%s: H=%d, Hk=%d", what, a->H, a->Hk);
  SHRIMP_REQUIRE(a->D >= 1 && a->D <= MAX_D, "%s: head dim %d outside [1, %d]", what, a->D, MAX_D);
  SHRIMP_REQUIRE(a->axes >= 1 && a->axes <= MAX_AXES, "%s: %d axes", what, a->axes);
  int64_t pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    SHRIMP_REQUIRE(a->sections[i] >= 0, "%s: section %d holds %d pairs", what, i, a->sections[i]);
    pairs += a->sections[i];
  }
  SHRIMP_REQUIRE(2 * pairs <= a->D, "%s: %lld pairs in a head of %d dimensions", what,
                 (long long)pairs, a->D);
  const bool norm = a->q_w != nullptr || a->k_w != nullptr;
  const bool has_k = a->Hk > 0;
  if (norm) {
    SHRIMP_REQUIRE((a->q_w || a->H == 0) && (a->k_w || !has_k), "%s: a norm weight is missing", what);
    SHRIMP_REQUIRE(a->w_dt == SHRIMP_DT_BF16 || a->w_dt == SHRIMP_DT_F16 || a->w_dt == SHRIMP_DT_F32,
                   "%s: weight type %d", what, a->w_dt);
    SHRIMP_REQUIRE(a->eps > 0.f, "%s: eps must be positive", what);
  }
  SHRIMP_REQUIRE(!back || norm, "%s: the norm's weights are required", what);
  SHRIMP_REQUIRE(a->pos_dt == SHRIMP_DT_I32 || a->pos_dt == SHRIMP_DT_I64 || a->pos_dt == SHRIMP_DT_F32,
                 "%s: position type %d", what, a->pos_dt);
  const bool work = a->B > 0 && a->S > 0 && (a->H > 0 || has_k);
  if (work) {
    SHRIMP_REQUIRE(pairs == 0 || (a->pos && a->freqs), "%s: null positions or frequencies", what);
    SHRIMP_REQUIRE(a->H == 0 || (a->q && a->q_out && (!back || a->gq)), "%s: null q pointer", what);
    SHRIMP_REQUIRE(!has_k || (a->k && a->k_out && (!back || a->gk)), "%s: null k pointer", what);
  }

  const int es = element_size(a->dt);
  // wide accesses divide the sections, the rest and every address
  const int rest = a->D - 2 * (int)pairs;
  auto fits = [&](int v) {
    if (pairs % v || rest % (2 * v)) return false;
    auto ok = [&](const void* base, int64_t sb, int64_t sh, int64_t sn) {
      return reinterpret_cast<uintptr_t>(base) % (uintptr_t)(v * es) == 0 && sb % v == 0 &&
             sh % v == 0 && sn % v == 0;
    };
    return ok(a->q, a->q_sb, a->q_sh, a->q_sn) && ok(a->q_out, 0, 0, 0) &&
           ok(a->k, a->k_sb, a->k_sh, a->k_sn) && ok(a->k_out, 0, 0, 0) &&
           (!back || (ok(a->gq, a->gq_sb, a->gq_sh, a->gq_sn) &&
                      ok(a->gk, a->gk_sb, a->gk_sh, a->gk_sn)));
  };
  out->vec = fits(VEC) ? VEC : 1;

  RopeParams& p = out->p;
  p = RopeParams{};
  p.t[0] = RopeTensor{a->q, a->gq, a->q_w, a->q_out, nullptr, a->q_sb, a->q_sh, a->q_sn,
                      a->gq_sb, a->gq_sh, a->gq_sn, a->H, 0};
  p.t[1] = RopeTensor{a->k, a->gk, a->k_w, a->k_out, nullptr, a->k_sb, a->k_sh, a->k_sn,
                      a->gk_sb, a->gk_sh, a->gk_sn, a->Hk, 0};
  p.pos = a->pos;
  p.freqs = a->freqs;
  p.p_sb = a->p_sb;
  p.p_sn = a->p_sn;
  p.p_sa = a->p_sa;
  p.pos_dt = a->pos_dt;
  p.freq_f64 = a->freq_f64;
  p.w_dt = a->w_dt;
  p.axes = a->axes;
  int cut = 0;
  for (int i = 0; i < MAX_AXES - 1; ++i) {
    cut += i < a->axes ? a->sections[i] : 0;
    p.cut[i] = i + 1 < a->axes ? cut : MAX_D;
  }
  p.eps = a->eps;
  p.sign = (a->inverse != 0) != back ? -1.f : 1.f;
  p.tokens = a->B * a->S;
  p.S = a->S;
  p.D = a->D;
  p.inv_d = 1.f / (float)a->D;
  p.P = (int)pairs;
  p.interleaved = a->interleaved != 0;
  const int units = (int)pairs / out->vec + (rest + 2 * out->vec - 1) / (2 * out->vec);
  p.lanes = pow2_ceil(units < 64 ? units : 64);
  // heads beside each other in memory (a token's row): across lanes until a read is 256 bytes
  p.head_lanes = 1;
  const int heads = a->H > a->Hk ? a->H : a->Hk;
  const int64_t sh = a->H > 0 ? a->q_sh : a->k_sh, sn = a->H > 0 ? a->q_sn : a->k_sn;
  if (sh < sn)
    while (p.head_lanes * a->D * es < 256 && p.head_lanes < heads && p.head_lanes * p.lanes < 64)
      p.head_lanes *= 2;
  const int per_block = THREADS / (p.lanes * p.head_lanes);
  const int64_t blocks = ((int64_t)p.tokens + per_block - 1) / per_block;
  const int64_t full = FULL_BLOCKS;
  out->grid_x = (int)(blocks > full ? full : blocks);
  p.t[0].groups = (a->H + p.head_lanes - 1) / p.head_lanes;
  p.t[1].groups = (a->Hk + p.head_lanes - 1) / p.head_lanes;
  const int groups = p.t[0].groups + p.t[1].groups;
  int split = 1;
  if (blocks > 0 && blocks < full) split = (int)((full + blocks - 1) / blocks);
  if (split > groups) split = groups;
  p.groups_per_block = groups > 0 ? (groups + split - 1) / split : 0;
  auto rows = [&](int n) { return n > 0 ? (n + p.groups_per_block - 1) / p.groups_per_block : 0; };
  p.q_rows = rows(p.t[0].groups);
  out->grid_y = back ? p.q_rows + rows(p.t[1].groups) : rows(groups);
  out->flight = p.groups_per_block > 1 && !back ? 2 : 1;
  return SHRIMP_OK;
}

template <typename T, int V, bool NORM, bool BACK>
void launch(const RopePlan& pl, hipStream_t st) {
  const dim3 grid(pl.grid_x, pl.grid_y), block(THREADS);
  if (pl.flight == 1)
    hipLaunchKernelGGL((rope_kernel<T, V, 1, NORM, BACK>), grid, block, 0, st, pl.p);
  else
    hipLaunchKernelGGL((rope_kernel<T, V, BACK ? 1 : 2, NORM, BACK>), grid, block, 0, st, pl.p);
}

template <bool NORM, bool BACK>
void launch_any(const RopePlan& pl, int dt, hipStream_t st) {
  const bool wide = pl.vec == VEC;
  if (dt == SHRIMP_DT_F32)
    wide ? launch<float, VEC, NORM, BACK>(pl, st) : launch<float, 1, NORM, BACK>(pl, st);
  else if (dt == SHRIMP_DT_F16)
    wide ? launch<_Float16, VEC, NORM, BACK>(pl, st) : launch<_Float16, 1, NORM, BACK>(pl, st);
  else
    wide ? launch<__bf16, VEC, NORM, BACK>(pl, st) : launch<__bf16, 1, NORM, BACK>(pl, st);
}

}  // namespace
}  // namespace shrimp

extern "C" int shrimp_rope(const shrimp_rope_args* a, void* stream) {
  using namespace shrimp;
  RopePlan pl;
  const int rc = plan_rope(a, false, &pl, "rope");
  if (rc != SHRIMP_OK) return rc;
  if (pl.grid_x == 0 || pl.grid_y == 0) return SHRIMP_OK;
  if (a->q_w || a->k_w)
    launch_any<true, false>(pl, a->dt, as_stream(stream));
  else
    launch_any<false, false>(pl, a->dt, as_stream(stream));
  return check_launch("rope");
}

extern "C" int64_t shrimp_qk_norm_rope_workspace(const shrimp_rope_args* a) {
  using namespace shrimp;
  RopePlan pl;
  if (plan_rope(a, true, &pl, "qk_norm_rope_workspace") != SHRIMP_OK) return -1;
  return (int64_t)pl.grid_x * pl.grid_y * a->D * 4;
}

extern "C" int shrimp_qk_norm_rope_backward(const shrimp_rope_args* a, void* dw_q, void* dw_k,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace shrimp;
  RopePlan pl;
  const int rc = plan_rope(a, true, &pl, "qk_norm_rope_backward");
  if (rc != SHRIMP_OK) return rc;
  SHRIMP_REQUIRE(dw_q && dw_k, "qk_norm_rope_backward: null weight gradient");
  const int blocks[2] = {pl.grid_x * pl.p.q_rows, pl.grid_x * (pl.grid_y - pl.p.q_rows)};
  const int64_t need = (int64_t)(blocks[0] + blocks[1]) * a->D * 4;
  SHRIMP_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
                 "qk_norm_rope_backward: workspace of %lld bytes, %lld needed",
                 (long long)workspace_bytes, (long long)need);
  pl.p.t[0].part = static_cast<float*>(workspace);
  pl.p.t[1].part = need ? static_cast<float*>(workspace) + (int64_t)blocks[0] * a->D : nullptr;
  if (need > 0) {
    launch_any<true, true>(pl, a->dt, as_stream(stream));
    const int e = check_launch("qk_norm_rope_backward");
    if (e != SHRIMP_OK) return e;
  }
  hipLaunchKernelGGL(rope_dw_kernel, dim3((a->D + 15) / 16, 2), dim3(THREADS), 0, as_stream(stream),
                     pl.p.t[0].part, pl.p.t[1].part, blocks[0], blocks[1], a->D, dw_q, dw_k, a->w_dt);
  return check_launch("qk_norm_rope_backward");
}
