// Norm of every query and key head, and the position rotation, in one pass; and its gradients.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w                     (w: one weight per entry, shared by the heads)
//   y = rotation of the pairs (a, b) of the first R entries of n by the token's angles: (a c - b s, b c + a s)
//   pairs: (i, i + R/2), or (2 i, 2 i + 1) when interleaved; the entries from R on pass through
//
//   backward: g = the pairs of dy rotated back: (a c + b s, b c - a s);  dw = sum over rows of g x r
//             dx = r (g w) - x r^3 mean(g w x)
//
// Memory-bound: every row is read once and written once (backward: x and dy read, dx written).  All
// sums are fp32; the results are rounded once, to the type of the tensors.
//
// A row belongs to a group of lanes of one warp, and a lane holds both members of each of its pairs, so
// the rotation needs no exchange and the row sums are one shuffle tree.  The group walks several heads
// of ONE token with the lane's angles and weights in registers: fetched per row they would be as much
// traffic as the row itself.  Two forms:
//   vectors  two 16-byte vectors of the row per lane (vectors j and j + R/2 entries; neighbouring ones
//            when the pairs are neighbours): D a multiple of a vector, R of two (of one), 16-byte rows
//   pairs    every other shape and alignment: single entries, consecutive pairs in consecutive lanes
#include "common.cuh"
#include "ptx.cuh"

namespace kcg {

namespace {

constexpr int RN_THREADS = 256;

struct RopeParams {
  const void* x[2];               // queries, keys
  const void* dy[2];              // backward: gradients of the outputs
  void* y[2];                     // outputs (backward: gradients of x)
  long long xs[2][3], ds[2][3], ys[2][3];   // strides: batch, head, row (elements)
  const void* w[2];               // may be null: weights of one
  int w_f32;
  const float *cs, *sn;           // [table_rows, R / 2]
  long long table_rows;
  const void* pos;                // null: token s is at position s
  int pos64;
  long long pos_sb, pos_ss;
  int B, S, D, R, heads[2];
  int interleaved;
  float eps, inv_d;
  int chunk[2], chunks[2];        // heads a group walks; how many such runs a token has
  unsigned units[2];              // B * S * chunks
  int ctas[2];                    // backward: CTAs of each tensor
  float* part;                    // backward: [ctas][D] partial weight gradients; null when none is wanted
  int* status;
  unsigned long long y_extent[2], part_extent, dw_extent; // bounds-checking build
  unsigned long long* bounds_detail;
};

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4 v, float2 (&f)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
  }
  __device__ static uint4 pack(const float2 (&f)[4]) {
    return make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                      pack_bf16x2(f[3].x, f[3].y));
  }
  __device__ static float one(const __nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 round(float v) { return __float2bfloat16(v); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4 v, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  __device__ static uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
  __device__ static float one(const float v) { return v; }
  __device__ static float round(float v) { return v; }
};

// Both weights as fp32 in shared memory, ones where there is none.
__device__ __forceinline__ void stage_weights(const RopeParams& p, float (&w)[2][256]) {
  for (int i = threadIdx.x; i < 2 * p.D; i += RN_THREADS) {
    const int t = i >= p.D, k = i - t * p.D;
    float v = 1.f;
    if (p.w[t]) v = p.w_f32 ? static_cast<const float*>(p.w[t])[k] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.w[t])[k]);
    w[t][k] = v;
  }
}

// A group's work: some heads of one token of one of the tensors.
struct Unit {
  int type, b, s, h_first, n_heads;
  // every group of a warp takes part in its rounds (shuffles inside); one past the end has no heads
  __device__ Unit(const RopeParams& p, unsigned u, bool live, int fixed_type) {
    type = fixed_type;
    if (type < 0) {
      type = u >= p.units[0] ? 1 : 0;
      if (type) u -= p.units[0];
    }
    // consecutive groups take consecutive tokens: their rows of a head are neighbours in the output
    const unsigned tokens = static_cast<unsigned>(p.B) * p.S, run = u / tokens, token = u - run * tokens;
    h_first = static_cast<int>(run) * p.chunk[type];
    b = static_cast<int>(token / p.S);
    s = static_cast<int>(token - static_cast<unsigned>(b) * p.S);
    n_heads = live ? min(p.chunk[type], p.heads[type] - h_first) : 0;
  }
  __device__ long long offset(const long long (&st)[3]) const { return b * st[0] + h_first * st[1] + s * st[2]; }
};

// Row of the tables for token (b, s), or -1: a position outside the tables is recorded in the status
// word, and its rotated entries come out as NaN.
__device__ __forceinline__ long long table_row(const RopeParams& p, int b, int s) {
  long long at = s;
  if (p.pos) {
    const long long i = b * p.pos_sb + s * p.pos_ss;
    at = p.pos64 ? static_cast<const long long*>(p.pos)[i] : static_cast<const int*>(p.pos)[i];
  }
  if (at >= 0 && at < p.table_rows) return at;
  atomicCAS(p.status, 0, static_cast<int>(DEV_BAD_POSITION));
  return -1;
}

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

__device__ __forceinline__ float2 swap2(float2 v) { return make_float2(v.y, v.x); }

// The vector form: LPR lanes per row, two vectors per lane.  The rows on their way wait in shared memory, in
// slots that one thread alone writes (asynchronous copies) and reads, DEPTH rows deep for every group: that
// many registers would leave too few warps, and too few bytes in flight for the memory's latency (gradients
// at 4 x 4096 x 40 x 128 in bf16: one row ahead in registers 3.9 TB/s, three in shared memory
// 5.6).  The arithmetic is in pairs of entries (packed fp32), the angles and weights multiplied into the
// lane's constants once per token:
//   y_a = r (a * ca + mate_a * sa), with the mate of a vector's entries in the lane's other vector, or
//   (neighbours) the other entry of the pair.
constexpr int rope_rows(bool bwd) { return bwd ? 1 : 2; }     // rows of a group that are computed together
constexpr int rope_depth(bool bwd) { return bwd ? 3 : 2; }    // times as many are on their way
constexpr int rope_slots(bool bwd) { return bwd ? 4 : 2; }    // vectors of a row per lane: x, and dy
template <typename T, int LPR, bool IL, bool BWD>
__global__ void __launch_bounds__(RN_THREADS, 2) rope_vec_kernel(const __grid_constant__ RopeParams p) {
  constexpr int N = Vec<T>::N, P = N / 2;
  constexpr unsigned GROUPS = RN_THREADS / LPR;
  constexpr int U = rope_rows(BWD), DEPTH = rope_depth(BWD), SLOTS = rope_slots(BWD);
  __shared__ __align__(16) float weights[2][256];
  __shared__ float red[BWD ? RN_THREADS / 32 : 1][BWD ? 256 : 1];
  extern __shared__ __align__(16) uint4 rows[];             // [DEPTH][U][SLOTS][RN_THREADS]
  const uint32_t slot0 = smem_u32(rows) + threadIdx.x * 16;
  if (BWD) griddep_launch_dependents();
  const int gl = threadIdx.x % LPR;
  const unsigned group = threadIdx.x / LPR;
  const int nv = p.D / N;
  // the lane's vectors
  const int hp = IL ? 0 : p.R / (2 * N);
  const bool mates = gl < hp;
  const int va = IL || mates ? gl : 2 * hp + 2 * (gl - hp);
  const int vb = IL ? gl + LPR : mates ? gl + hp : va + 1;
  const bool has_a = va < nv, has_b = vb < nv;
  // whether the lane's vectors are rotated (R is a multiple of a vector)
  const bool rot_a = has_a && (IL ? va * N < p.R : mates), rot_b = has_b && (IL ? vb * N < p.R : mates);
  float2 acc_a[P], acc_b[P];
  if (BWD) {
#pragma unroll
    for (int i = 0; i < P; ++i) acc_a[i] = acc_b[i] = make_float2(0.f, 0.f);
  }
  const int cta_type = BWD ? (static_cast<int>(blockIdx.x) >= p.ctas[0] ? 1 : 0) : -1;
  const unsigned end = BWD ? p.units[cta_type] : p.units[0] + p.units[1];
  const unsigned cta = blockIdx.x - (BWD && cta_type ? p.ctas[0] : 0);
  const unsigned step = (BWD ? p.ctas[cta_type] : gridDim.x) * GROUPS;
  const int rounds = BWD ? p.chunk[cta_type] : max(p.chunk[0], p.chunk[1]);
  unsigned u0 = cta * GROUPS;
  if (u0 >= end) return;
  // Where a unit's rows are, and the rows of one round: U heads.
  struct Where {
    int type, n_heads;
    long long tr;
    const T *x, *dy;
    long long y0;
  };
  auto place = [&](unsigned u) {
    const bool live = u + group < end;
    const Unit un(p, live ? u + group : end - 1, live, cta_type);
    Where w;
    w.type = un.type;
    w.n_heads = un.n_heads;
    w.tr = table_row(p, un.b, un.s);
    w.x = static_cast<const T*>(p.x[un.type]) + un.offset(p.xs[un.type]);
    w.dy = BWD ? static_cast<const T*>(p.dy[un.type]) + un.offset(p.ds[un.type]) : nullptr;
    w.y0 = un.offset(p.ys[un.type]);
    return w;
  };
  // the row that is asked for next: of unit ui, head hi of the run
  unsigned ui = u0;
  int hi = 0, to = 0;
  Where wi = place(u0);
  auto request = [&]() {
    if (ui < end) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool on = hi + k < wi.n_heads;
        const T* xr = wi.x + (hi + k) * p.xs[wi.type][1];
        const uint32_t at = slot0 + (to * U + k) * (SLOTS * RN_THREADS * 16);
        cp_async16(at, on && has_a ? xr + va * N : wi.x, on && has_a);
        cp_async16(at + RN_THREADS * 16, on && has_b ? xr + vb * N : wi.x, on && has_b);
        if (BWD) {
          const T* dr = wi.dy + (hi + k) * p.ds[wi.type][1];
          cp_async16(at + 2 * RN_THREADS * 16, on && has_a ? dr + va * N : wi.dy, on && has_a);
          cp_async16(at + 3 * RN_THREADS * 16, on && has_b ? dr + vb * N : wi.dy, on && has_b);
        }
      }
      hi += U;
      if (hi >= rounds) {
        hi = 0;
        ui += step;
        if (ui < end) wi = place(ui);
      }
    }
    cp_async_commit();     // (an empty group past the end, so that the count stays)
    to = to + 1 == DEPTH ? 0 : to + 1;
  };
  Where un = wi;
#pragma unroll
  for (int k = 0; k < DEPTH - 1; ++k) request();
  stage_weights(p, weights);
  __syncthreads();
  int from = 0;
  for (;;) {
    const int type = un.type;
    const long long yh = p.ys[type][1];
    // the lane's constants; backward: ca, sa hold the angles alone, cb, sb the weights
    float2 ca[P], sa[P], cb[P], sb[P];
    {
      const long long tr = un.tr;
      // angle of pair i of the lane: half-split, entry i of a with entry i of b; neighbours, first the P
      // pairs of a, then those of b
      float2 c[P], sn[P];
      const float* ct = p.cs + tr * (p.R / 2) + va * (IL ? P : N);
      const float* st = p.sn + tr * (p.R / 2) + va * (IL ? P : N);
      const float bad = __int_as_float(0x7FC00000);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const bool rot = IL ? (2 * i < P ? rot_a : rot_b) : mates;
        c[i] = rot ? make_float2(bad, bad) : make_float2(1.f, 1.f);
        sn[i] = rot ? make_float2(bad, bad) : make_float2(0.f, 0.f);
        if (rot && tr >= 0) {
          const int at = IL && 2 * i >= P ? (vb - va) * P + 2 * i - P : 2 * i;
          c[i] = __ldg(reinterpret_cast<const float2*>(ct + at));
          sn[i] = __ldg(reinterpret_cast<const float2*>(st + at));
        }
      }
      float2 wa[P], wb[P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        wa[i] = wb[i] = make_float2(0.f, 0.f);
        if (has_a) wa[i] = *reinterpret_cast<const float2*>(&weights[type][va * N + 2 * i]);
        if (has_b) wb[i] = *reinterpret_cast<const float2*>(&weights[type][vb * N + 2 * i]);
      }
      auto at = [](const float2 (&v)[P], int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; };
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (BWD) {
          ca[i] = c[i];
          sa[i] = sn[i];
          cb[i] = wa[i];
          sb[i] = wb[i];
        } else if (IL) {
          const float c0 = at(c, i), s0 = at(sn, i), c1 = at(c, P + i), s1 = at(sn, P + i);
          ca[i] = make_float2(c0 * wa[i].x, c0 * wa[i].y);
          sa[i] = make_float2(-s0 * wa[i].y, s0 * wa[i].x);
          cb[i] = make_float2(c1 * wb[i].x, c1 * wb[i].y);
          sb[i] = make_float2(-s1 * wb[i].y, s1 * wb[i].x);
        } else {
          ca[i] = mul2(c[i], wa[i]);
          sa[i] = mul2(make_float2(-sn[i].x, -sn[i].y), wb[i]);
          cb[i] = mul2(c[i], wb[i]);
          sb[i] = mul2(sn[i], wa[i]);
        }
      }
    }
    const bool more = u0 + step < end;
    Where next = un;
    if (more) next = place(u0 + step);
    if (more && next.tr >= 0) {     // the next token's angles, out of the way of its first row
      prefetch_l1(p.cs + next.tr * (p.R / 2) + (rot_a ? va * (IL ? P : N) : 0));
      prefetch_l1(p.sn + next.tr * (p.R / 2) + (rot_a ? va * (IL ? P : N) : 0));
    }
    for (int h0 = 0; h0 < rounds; h0 += U) {
      request();
      cp_async_wait<DEPTH - 1>();
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool on = h0 + k < un.n_heads;
        const uint32_t at = slot0 + (from * U + k) * (SLOTS * RN_THREADS * 16);
        const uint4 xa = ld_shared_v4(at), xb = ld_shared_v4(at + RN_THREADS * 16);
        float2 a[P], bb[P], s2 = make_float2(0.f, 0.f);
        Vec<T>::unpack(xa, a);
        Vec<T>::unpack(xb, bb);
#pragma unroll
        for (int i = 0; i < P; ++i) s2 = fma2(bb[i], bb[i], fma2(a[i], a[i], s2));
        const float ms = group_sum<LPR>(s2.x + s2.y) * p.inv_d + p.eps;
        const float r = on ? rsqrtf(ms) : 0.f;     // (a row of zeros with an eps of zero would be 0 * inf)
        const float2 r2 = make_float2(r, r);
        float2 oa[P], ob[P];
        if (!BWD) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            oa[i] = mul2(fma2(IL ? swap2(a[i]) : bb[i], sa[i], mul2(a[i], ca[i])), r2);
            ob[i] = mul2(fma2(IL ? swap2(bb[i]) : a[i], sb[i], mul2(bb[i], cb[i])), r2);
          }
        } else {
          float2 ga[P], gb[P], d2 = make_float2(0.f, 0.f);
          Vec<T>::unpack(ld_shared_v4(at + 2 * RN_THREADS * 16), ga);
          Vec<T>::unpack(ld_shared_v4(at + 3 * RN_THREADS * 16), gb);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 f = ga[i], g = gb[i];
            if (IL) {
              // pair i's angle: entry i of the first half of c and sn for a, of the second for b
              const float cA = i & 1 ? ca[i / 2].y : ca[i / 2].x, sA = i & 1 ? sa[i / 2].y : sa[i / 2].x;
              const float cB = (P + i) & 1 ? ca[(P + i) / 2].y : ca[(P + i) / 2].x, sB = (P + i) & 1 ? sa[(P + i) / 2].y : sa[(P + i) / 2].x;
              ga[i] = fma2(make_float2(f.y, -f.x), make_float2(sA, sA), mul2(f, make_float2(cA, cA)));
              gb[i] = fma2(make_float2(g.y, -g.x), make_float2(sB, sB), mul2(g, make_float2(cB, cB)));
            } else {
              ga[i] = fma2(g, sa[i], mul2(f, ca[i]));
              gb[i] = fma2(make_float2(-f.x, -f.y), sa[i], mul2(g, ca[i]));
            }
            // rows past the run are zeros: they add nothing
            acc_a[i] = fma2(ga[i], mul2(a[i], r2), acc_a[i]);
            acc_b[i] = fma2(gb[i], mul2(bb[i], r2), acc_b[i]);
            ga[i] = mul2(ga[i], cb[i]);
            gb[i] = mul2(gb[i], sb[i]);
            d2 = fma2(gb[i], bb[i], fma2(ga[i], a[i], d2));
          }
          // x r^3 mean(g w x): the factors in an order that neither overflows nor vanishes for tiny rows
          const float m = -group_sum<LPR>((d2.x + d2.y) * r) * p.inv_d;
          const float2 m2 = make_float2(m, m);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            oa[i] = mul2(fma2(mul2(a[i], r2), m2, ga[i]), r2);
            ob[i] = mul2(fma2(mul2(bb[i], r2), m2, gb[i]), r2);
          }
        }
        if (on) {
          const long long to_row = un.y0 + (h0 + k) * yh;
          T* yr = static_cast<T*>(p.y[type]) + to_row;
          if (has_a && bounds_ok((to_row + va * N) * sizeof(T), 16, p.y_extent[type], p.status, p.bounds_detail))
            *reinterpret_cast<uint4*>(yr + va * N) = Vec<T>::pack(oa);
          if (has_b && bounds_ok((to_row + vb * N) * sizeof(T), 16, p.y_extent[type], p.status, p.bounds_detail))
            *reinterpret_cast<uint4*>(yr + vb * N) = Vec<T>::pack(ob);
        }
      }
      from = from + 1 == DEPTH ? 0 : from + 1;
    }
    if (!more) break;
    un = next;
    u0 += step;
  }
  if (BWD && p.part) {
    // lanes of equal place in their group, then the warps, in a fixed order
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        acc_a[i].x += __shfl_xor_sync(0xFFFFFFFFu, acc_a[i].x, o);
        acc_a[i].y += __shfl_xor_sync(0xFFFFFFFFu, acc_a[i].y, o);
        acc_b[i].x += __shfl_xor_sync(0xFFFFFFFFu, acc_b[i].x, o);
        acc_b[i].y += __shfl_xor_sync(0xFFFFFFFFu, acc_b[i].y, o);
      }
    }
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) < LPR) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (has_a) red[warp][va * N + 2 * i] = acc_a[i].x, red[warp][va * N + 2 * i + 1] = acc_a[i].y;
        if (has_b) red[warp][vb * N + 2 * i] = acc_b[i].x, red[warp][vb * N + 2 * i + 1] = acc_b[i].y;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += RN_THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < RN_THREADS / 32; ++k) sum += red[k][i];
      const long long at = static_cast<long long>(blockIdx.x) * p.D + i;
      if (bounds_ok(at * 4, 4, p.part_extent, p.status, p.bounds_detail)) p.part[at] = sum;
    }
  }
}

// The pair form: LPR lanes per row, pairs gl, gl + LPR, .. of the row per lane (first the rotated ones,
// then the rest of the row two by two), single entries.  Bound by the latency of its 2- or 4-byte loads, with no rows
// on their way but the two at hand: 2 x 8000 tokens x 32 heads x 96, 38 rotated, bf16 69 us (2.85 TB/s), gradients 177 us
// (1.67 TB/s).
template <typename T, int LPR, int NP, bool BWD, int U>
__global__ void __launch_bounds__(RN_THREADS, 2) rope_pair_kernel(const __grid_constant__ RopeParams p) {
  constexpr unsigned GROUPS = RN_THREADS / LPR;
  __shared__ float weights[2][256];
  __shared__ float red[BWD ? RN_THREADS / 32 : 1][BWD ? 256 : 1];
  if (BWD) griddep_launch_dependents();
  const int gl = threadIdx.x % LPR;
  const unsigned group = threadIdx.x / LPR;
  const int half = p.R / 2;
  int ea[NP], eb[NP];    // the pairs' entries; -1: none
  float acc_a[NP], acc_b[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int pr = gl + i * LPR;
    const bool split = pr < half && !p.interleaved;
    ea[i] = pr < p.D / 2 ? (split ? pr : 2 * pr) : -1;
    eb[i] = split ? pr + half : 2 * pr + 1;
    acc_a[i] = acc_b[i] = 0.f;
  }
  stage_weights(p, weights);
  __syncthreads();
  const int cta_type = BWD ? (static_cast<int>(blockIdx.x) >= p.ctas[0] ? 1 : 0) : -1;
  const unsigned end = BWD ? p.units[cta_type] : p.units[0] + p.units[1];
  const unsigned cta = blockIdx.x - (BWD && cta_type ? p.ctas[0] : 0);
  const unsigned step = (BWD ? p.ctas[cta_type] : gridDim.x) * GROUPS;
  const int rounds = BWD ? p.chunk[cta_type] : max(p.chunk[0], p.chunk[1]);
  for (unsigned u0 = cta * GROUPS; u0 < end; u0 += step) {
    const bool live = u0 + group < end;
    const Unit un(p, live ? u0 + group : end - 1, live, cta_type);
    const int type = un.type;
    const long long xh = p.xs[type][1], dh = p.ds[type][1], yh = p.ys[type][1];
    const T* x = static_cast<const T*>(p.x[type]) + un.offset(p.xs[type]);
    const T* dy = BWD ? static_cast<const T*>(p.dy[type]) + un.offset(p.ds[type]) : nullptr;
    const long long y0 = un.offset(p.ys[type]);
    float c[NP], sn[NP], wa[NP], wb[NP];
    const long long tr = table_row(p, un.b, un.s);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      c[i] = 1.f, sn[i] = 0.f, wa[i] = wb[i] = 0.f;
      const int pr = gl + i * LPR;
      if (pr < half) {
        c[i] = sn[i] = __int_as_float(0x7FC00000);
        if (tr >= 0) {
          c[i] = __ldg(p.cs + tr * half + pr);
          sn[i] = __ldg(p.sn + tr * half + pr);
        }
      }
      if (ea[i] >= 0) {
        wa[i] = weights[type][ea[i]];
        wb[i] = weights[type][eb[i]];
      }
    }
    for (int h0 = 0; h0 < rounds; h0 += U) {
      float a[U][NP], bb[U][NP], ga[BWD ? U : 1][NP], gb[BWD ? U : 1][NP];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool on = h0 + k < un.n_heads;
        const T* xr = x + (h0 + k) * xh;
        const T* dr = dy + (h0 + k) * dh;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          a[k][i] = bb[k][i] = 0.f;
          if (BWD) ga[k][i] = gb[k][i] = 0.f;
          if (on && ea[i] >= 0) {
            a[k][i] = Vec<T>::one(xr[ea[i]]);
            bb[k][i] = Vec<T>::one(xr[eb[i]]);
            if (BWD) {
              ga[k][i] = Vec<T>::one(dr[ea[i]]);
              gb[k][i] = Vec<T>::one(dr[eb[i]]);
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool on = h0 + k < un.n_heads;
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) ss = fmaf(a[k][i], a[k][i], fmaf(bb[k][i], bb[k][i], ss));
        const float ms = group_sum<LPR>(ss) * p.inv_d + p.eps;
        const float r = on ? rsqrtf(ms) : 0.f;
        float oa[NP], ob[NP];
        if (!BWD) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float f = a[k][i] * wa[i], g = bb[k][i] * wb[i];
            oa[i] = r * (f * c[i] - g * sn[i]);
            ob[i] = r * (g * c[i] + f * sn[i]);
          }
        } else {
          float dot = 0.f;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float f = ga[k][i] * c[i] + gb[k][i] * sn[i], g = gb[k][i] * c[i] - ga[k][i] * sn[i];
            // rows past the run are zeros: they add nothing
            acc_a[i] = fmaf(f, a[k][i] * r, acc_a[i]);
            acc_b[i] = fmaf(g, bb[k][i] * r, acc_b[i]);
            oa[i] = f * wa[i];
            ob[i] = g * wb[i];
            dot = fmaf(oa[i], a[k][i], fmaf(ob[i], bb[k][i], dot));
          }
          const float m = group_sum<LPR>(dot * r) * p.inv_d;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            oa[i] = r * (oa[i] - (a[k][i] * r) * m);
            ob[i] = r * (ob[i] - (bb[k][i] * r) * m);
          }
        }
        if (on) {
          const long long at = y0 + (h0 + k) * yh;
          T* yr = static_cast<T*>(p.y[type]) + at;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            if (ea[i] < 0) continue;
            if (bounds_ok((at + ea[i]) * sizeof(T), sizeof(T), p.y_extent[type], p.status, p.bounds_detail)) yr[ea[i]] = Vec<T>::round(oa[i]);
            if (bounds_ok((at + eb[i]) * sizeof(T), sizeof(T), p.y_extent[type], p.status, p.bounds_detail)) yr[eb[i]] = Vec<T>::round(ob[i]);
          }
        }
      }
    }
  }
  if (BWD && p.part) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        acc_a[i] += __shfl_xor_sync(0xFFFFFFFFu, acc_a[i], o);
        acc_b[i] += __shfl_xor_sync(0xFFFFFFFFu, acc_b[i], o);
      }
      if ((threadIdx.x & 31) < LPR && ea[i] >= 0) {
        red[threadIdx.x >> 5][ea[i]] = acc_a[i];
        red[threadIdx.x >> 5][eb[i]] = acc_b[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += RN_THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < RN_THREADS / 32; ++k) sum += red[k][i];
      const long long at = static_cast<long long>(blockIdx.x) * p.D + i;
      if (bounds_ok(at * 4, 4, p.part_extent, p.status, p.bounds_detail)) p.part[at] = sum;
    }
  }
}

// dw[i] = sum of the CTAs' partial sums, in a fixed order (zero where there are none: no key heads): 32 columns per
// CTA, a warp per 32nd row.  Its launch overlaps the kernel before it.
__global__ void __launch_bounds__(1024) rope_weight_sum_kernel(const __grid_constant__ RopeParams p, float* dw0, float* dw1) {
  __shared__ float red[32][33];
  float* dw = blockIdx.y ? dw1 : dw0;
  if (!dw) return;
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane, D = p.D;
  const int n = p.ctas[blockIdx.y];
  const long long first = (blockIdx.y ? static_cast<long long>(p.ctas[0]) * D : 0) + col;
  griddep_wait();
  float sum = 0.f;
  if (col < D) {
#pragma unroll 4
    for (int i = sub; i < n; i += 32) {
      const long long at = first + static_cast<long long>(i) * D;
      if (bounds_ok(at * 4, 4, p.part_extent, p.status, p.bounds_detail)) sum += p.part[at];
    }
  }
  red[sub][lane] = sum;
  __syncthreads();
  if (sub == 0 && col < D) {
#pragma unroll
    for (int k = 1; k < 32; ++k) sum += red[k][lane];
    if (bounds_ok(col * 4, 4, p.dw_extent, p.status, p.bounds_detail)) dw[col] = sum;
  }
}

bool row_vectors(const HeadView& v, int es) {
  if (!v.base) return true;
  if (!aligned16(v.base)) return false;
  const int64_t s[3] = {v.sr, v.sh, v.sb};
  const int n[3] = {v.S, v.H, v.B};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && s[i] * es % 16) return false;
  return true;
}

// CTAs that the backward pass may use for each tensor: at most two per SM over both (what is resident), so that the
// partial weight gradients stay few.  A function of the shape alone (the workspace query has no pointers).
void bwd_ctas(const kcg_rope_desc* d, int& q, int& k) {
  const int most = 2 * 148;
  const long long heads = static_cast<long long>(d->H) + d->Hk;
  k = d->Hk ? static_cast<int>(most * static_cast<long long>(d->Hk) / heads) : 0;
  if (d->Hk && k < 1) k = 1;
  q = most - k;
}

template <typename T, int LPR, bool IL, bool BWD>
kcg_status_t go_vec(const RopeParams& p, unsigned grid, cudaStream_t stream) {
  constexpr int bytes = rope_depth(BWD) * rope_rows(BWD) * rope_slots(BWD) * RN_THREADS * 16;
  auto kern = rope_vec_kernel<T, LPR, IL, BWD>;
  static std::atomic<bool> allowed[64];
  const kcg_status_t st = allow_smem(kern, bytes, allowed);
  if (st == KCG_OK) kern<<<grid, RN_THREADS, bytes, stream>>>(p);
  return st;
}
template <typename T, bool IL, bool BWD>
kcg_status_t go_vec(const RopeParams& p, int lpr, unsigned grid, cudaStream_t stream) {
  switch (lpr) {
    case 4: return go_vec<T, 4, IL, BWD>(p, grid, stream);
    case 8: return go_vec<T, 8, IL, BWD>(p, grid, stream);
    case 16: return go_vec<T, 16, IL, BWD>(p, grid, stream);
    default: return go_vec<T, 32, IL, BWD>(p, grid, stream);
  }
}
template <typename T, bool BWD>
void go_pair(const RopeParams& p, unsigned grid, cudaStream_t stream) {
  constexpr int U = 2;
  switch ((p.D + 31) / 32) {   // lanes per row x pairs per lane >= D / 2
    case 1: return rope_pair_kernel<T, 16, 1, BWD, U><<<grid, RN_THREADS, 0, stream>>>(p);
    case 2: return rope_pair_kernel<T, 16, 2, BWD, U><<<grid, RN_THREADS, 0, stream>>>(p);
    case 3: return rope_pair_kernel<T, 16, 3, BWD, U><<<grid, RN_THREADS, 0, stream>>>(p);
    case 4: return rope_pair_kernel<T, 16, 4, BWD, U><<<grid, RN_THREADS, 0, stream>>>(p);
    case 5: case 6: return rope_pair_kernel<T, 32, 3, BWD, U><<<grid, RN_THREADS, 0, stream>>>(p);
    default: return rope_pair_kernel<T, 32, 4, BWD, U><<<grid, RN_THREADS, 0, stream>>>(p);
  }
}

template <typename T, bool BWD>
kcg_status_t launch_rope(RopeParams& p, const kcg_rope_desc* d, bool vectors, cudaStream_t stream) {
  constexpr int N = Vec<T>::N;
  const int nv = d->D / N;
  // the vector form: whole vectors, and both members of each pair in vectors of one lane
  const bool vec = vectors && d->D % N == 0 && (d->interleaved ? d->R % N == 0 : d->R % (2 * N) == 0);
  int lpr = 4;
  while (2 * lpr < nv) lpr *= 2;
  const int per_cta = RN_THREADS / (vec ? lpr : d->D <= 128 ? 16 : 32);
  const long long tokens = static_cast<long long>(d->B) * d->S, sms = device_sm_count();
  // Heads a group walks with one set of angles, at most 8.  Vector form: the length whose rounds over all groups
  // that the SMs hold (two CTAs each) take the fewest rows, a run counting one more for its start.  (3 x 777 tokens x
  // 16 heads of 80 in fp32: 4 heads 6.1 us, 8 heads 8.2; 1500 x 40 of 128 in bf16: 4 heads 8.4, 8 heads 6.9.)
  // Pair form: as long as every group still has work (backward, 2000 x 16 of 96: 2 heads 14.1 us, 4 heads 18.0).
  auto runs = [&](int t, int c) { return tokens * ((p.heads[t] + c - 1) / c); };
  auto rows = [&](int t, int c) {
    const long long units = BWD ? runs(t, c) : runs(0, c) + runs(1, c), groups = per_cta * (BWD ? p.ctas[t] : 2 * sms);
    constexpr int U = rope_rows(BWD);
    return (units + groups - 1) / groups * ((c + U - 1) / U * U + 1);
  };
  for (int t = 0; t < 2; ++t) {
    int chunk = 1;
    if (!p.heads[t]) {
      // (no such tensor)
    } else if (vec) {
      for (int c = 2; c <= 8; c *= 2)
        if (rows(t, c) < rows(t, chunk)) chunk = c;
    } else {
      while (chunk < 8 && tokens * (p.heads[0] + p.heads[1]) / (2 * chunk) >= sms * 2 * per_cta) chunk *= 2;
    }
    if (chunk > p.heads[t]) chunk = p.heads[t] ? p.heads[t] : 1;
    const int chunks = p.heads[t] ? (p.heads[t] + chunk - 1) / chunk : 0;
    if (tokens * chunks > 0x3FFFFFFFll) return KCG_BAD_SHAPE;
    p.chunk[t] = chunk;
    p.chunks[t] = chunks;
    p.units[t] = static_cast<unsigned>(tokens * chunks);
  }
  unsigned grid;
  if (BWD) {
    for (int t = 0; t < 2; ++t) {
      const unsigned want = (p.units[t] + per_cta - 1) / per_cta;
      if (static_cast<unsigned>(p.ctas[t]) > want) p.ctas[t] = static_cast<int>(want);
    }
    grid = static_cast<unsigned>(p.ctas[0] + p.ctas[1]);
  } else {
    const long long want = (static_cast<long long>(p.units[0]) + p.units[1] + per_cta - 1) / per_cta, most = (vec ? 2 : 16) * sms;
    grid = static_cast<unsigned>(want < most ? want : most);
  }
  kcg_status_t st = KCG_OK;
  if (!vec) go_pair<T, BWD>(p, grid, stream);
  else st = d->interleaved ? go_vec<T, true, BWD>(p, lpr, grid, stream) : go_vec<T, false, BWD>(p, lpr, grid, stream);
  if (st != KCG_OK) return st;
  g_launches.fetch_add(1);
  KCG_CUDA_TRY(cudaGetLastError());
  return KCG_OK;
}

kcg_status_t check_desc(const kcg_rope_desc* d) {
  if (!d) return KCG_BAD_ARGUMENT;
  if (d->B <= 0 || d->S <= 0 || d->H <= 0 || d->Hk < 0) return KCG_BAD_SHAPE;
  if (d->D <= 0 || d->D > 256 || d->D % 2 || d->R <= 0 || d->R > d->D || d->R % 2) return KCG_BAD_SHAPE;
  if (d->table_rows <= 0) return KCG_BAD_SHAPE;
  if (d->dtype != KCG_F32 && d->dtype != KCG_BF16) return KCG_UNSUPPORTED;
  if (d->dtype_w != KCG_F32 && d->dtype_w != KCG_BF16) return KCG_UNSUPPORTED;
  if (d->pos_bits != 32 && d->pos_bits != 64) return KCG_UNSUPPORTED;
  if (!(d->eps >= 0.f) || d->eps > 3.0e38f) return KCG_BAD_ARGUMENT;
  return KCG_OK;
}

// Fills what both directions share; x, dy, y: queries and keys.  An output's used strides must be
// positive: with one of zero, rows would fall on one another.
kcg_status_t fill(const kcg_rope_desc* d, const void* const (&x)[2], const int64_t* const (&xs)[2], const void* const (&dy)[2],
                  const int64_t* const (&ds)[2], void* const (&y)[2], const int64_t* const (&ys)[2], const void* const (&w)[2],
                  const void* cs, const void* sn, const void* pos, RopeParams& p, bool& vectors) {
  const int es = d->dtype == KCG_F32 ? 4 : 2, ws = d->dtype_w == KCG_F32 ? 4 : 2;
  if (!x[0] || !y[0] || !cs || !sn || (d->Hk && (!x[1] || !y[1]))) return KCG_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(cs) | reinterpret_cast<uintptr_t>(sn)) & 3u) return KCG_BAD_ALIGN;
  if (pos && reinterpret_cast<uintptr_t>(pos) % (d->pos_bits / 8)) return KCG_BAD_ALIGN;
  vectors = aligned16(cs) && aligned16(sn);
  for (int t = 0; t < 2; ++t) {
    const int heads = t ? d->Hk : d->H;
    p.heads[t] = heads;
    p.x[t] = x[t], p.dy[t] = dy[t], p.y[t] = y[t], p.w[t] = heads ? w[t] : nullptr;
    p.y_extent[t] = 0;
    if (!heads) continue;
    if (reinterpret_cast<uintptr_t>(w[t]) % ws) return KCG_BAD_ALIGN;
    const void* ptr[3] = {x[t], dy[t], y[t]};
    const int64_t* str[3] = {xs[t], ds[t], ys[t]};
    long long* into[3] = {p.xs[t], p.ds[t], p.ys[t]};
    for (int k = 0; k < 3; ++k) {
      if (!ptr[k]) continue;
      if (reinterpret_cast<uintptr_t>(ptr[k]) % es) return KCG_BAD_ALIGN;
      const int n[3] = {d->B, heads, d->S};
      for (int i = 0; i < 3; ++i) {
        into[k][i] = n[i] == 1 ? 0 : str[k][i];
        if (n[i] > 1 && (str[k][i] < 0 || (k == 2 && str[k][i] == 0))) return KCG_BAD_SHAPE;
      }
      const HeadView v{ptr[k], d->B, heads, d->S, d->D, into[k][0], into[k][1], into[k][2]};
      vectors = vectors && row_vectors(v, es);
      if (k == 2) p.y_extent[t] = head_view_extent(v, es);
    }
  }
  // An output is written while other groups of lanes still read: it may be the very view that its own rows are read
  // from (a row is read before it is written, by the same lanes), and may overlap nothing else.
  auto view = [&](const void* at, const long long (&s)[3], int t) { return HeadView{at, d->B, p.heads[t], d->S, d->D, s[0], s[1], s[2]}; };
  for (int t = 0; t < 2; ++t) {
    if (!p.heads[t]) continue;
    const HeadRegion out(view(p.y[t], p.ys[t], t), es);
    for (int u = 0; u < 2; ++u) {
      if (!p.heads[u]) continue;
      const void* in[2] = {p.x[u], p.dy[u]};
      const long long(*st[2])[3] = {&p.xs[u], &p.ds[u]};
      for (int k = 0; k < 2; ++k) {
        if (!in[k]) continue;
        const long long(&s)[3] = *st[k];
        const bool same = u == t && in[k] == p.y[t] && s[0] == p.ys[t][0] && s[1] == p.ys[t][1] && s[2] == p.ys[t][2];
        if (!same && views_overlap(out, HeadRegion(view(in[k], s, u), es))) return KCG_BAD_ARGUMENT;
      }
    }
    if (t && p.heads[0] && views_overlap(out, HeadRegion(view(p.y[0], p.ys[0], 0), es))) return KCG_BAD_ARGUMENT;
  }
  p.w_f32 = d->dtype_w == KCG_F32;
  p.cs = static_cast<const float*>(cs);
  p.sn = static_cast<const float*>(sn);
  p.table_rows = d->table_rows;
  p.pos = pos;
  p.pos64 = d->pos_bits == 64;
  p.pos_sb = d->B == 1 ? 0 : d->pos[0];
  p.pos_ss = d->S == 1 ? 0 : d->pos[1];
  if (pos && (p.pos_sb < 0 || p.pos_ss < 0)) return KCG_BAD_SHAPE;
  p.B = d->B, p.S = d->S, p.D = d->D, p.R = d->R;
  p.interleaved = d->interleaved ? 1 : 0;
  p.eps = d->eps;
  p.inv_d = 1.f / static_cast<float>(d->D);
  p.part = nullptr;
  p.ctas[0] = p.ctas[1] = 0;
  p.part_extent = qk_norm_rope_bwd_workspace_impl(d);
  p.dw_extent = 4ull * d->D;
  if (const unsigned long long cap = debug_extent_limit())
    for (unsigned long long* e : {&p.y_extent[0], &p.y_extent[1], &p.part_extent, &p.dw_extent}) *e = *e < cap ? *e : cap;
  p.bounds_detail = nullptr;
  debug_bounds_detail_ptr(&p.bounds_detail);
  return device_status_ptr(&p.status);
}

}  // namespace

kcg_status_t qk_norm_rope_impl(const kcg_rope_desc* d, const void* q, const void* k, const void* wq, const void* wk,
                               const void* cs, const void* sn, const void* pos, void* q_out, void* k_out,
                               cudaStream_t stream) {
  kcg_status_t st = check_desc(d);
  if (st != KCG_OK) return st;
  RopeParams p;
  bool vectors;
  st = fill(d, {q, k}, {d->q, d->k}, {nullptr, nullptr}, {d->q, d->k}, {q_out, k_out}, {d->q_out, d->k_out}, {wq, wk}, cs, sn,
            pos, p, vectors);
  if (st != KCG_OK) return st;
  return d->dtype == KCG_F32 ? launch_rope<float, false>(p, d, vectors, stream)
                             : launch_rope<__nv_bfloat16, false>(p, d, vectors, stream);
}

size_t qk_norm_rope_bwd_workspace_impl(const kcg_rope_desc* d) {
  if (check_desc(d) != KCG_OK) return 0;
  int q, k;
  bwd_ctas(d, q, k);
  return static_cast<size_t>(q + k) * d->D * sizeof(float);
}

kcg_status_t qk_norm_rope_bwd_impl(const kcg_rope_desc* d, const void* dq_out, const void* dk_out, const void* q, const void* k,
                                   const void* wq, const void* wk, const void* cs, const void* sn, const void* pos, void* dq,
                                   void* dk, float* dwq, float* dwk, void* ws, size_t ws_bytes, cudaStream_t stream) {
  kcg_status_t st = check_desc(d);
  if (st != KCG_OK) return st;
  if (!dq_out || (d->Hk && !dk_out)) return KCG_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(dwq) | reinterpret_cast<uintptr_t>(dwk)) & 3u) return KCG_BAD_ALIGN;
  RopeParams p;
  bool vectors;
  st = fill(d, {q, k}, {d->q, d->k}, {dq_out, dk_out}, {d->q_out, d->k_out}, {dq, dk}, {d->d_q, d->d_k}, {wq, wk}, cs, sn, pos,
            p, vectors);
  if (st != KCG_OK) return st;
  const bool sums = dwq || dwk;
  if (sums) {
    if (!ws || ws_bytes < qk_norm_rope_bwd_workspace_impl(d) || !aligned16(ws)) return KCG_BAD_WORKSPACE;
    p.part = static_cast<float*>(ws);
  }
  bwd_ctas(d, p.ctas[0], p.ctas[1]);
  st = d->dtype == KCG_F32 ? launch_rope<float, true>(p, d, vectors, stream)
                           : launch_rope<__nv_bfloat16, true>(p, d, vectors, stream);
  if (st != KCG_OK || !sums) return st;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>((d->D + 31) / 32), 2);
  cfg.blockDim = dim3(1024);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KCG_CUDA_TRY(cudaLaunchKernelEx(&cfg, rope_weight_sum_kernel, p, dwq, dwk));
  g_launches.fetch_add(1);
  return KCG_OK;
}

}  // namespace kcg
