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
// A row belongs to a group of lanes of one warp.  In the vector path a lane holds two 16-byte vectors
// of the row, chosen so that both members of each of its pairs are its own (vectors j and j + R/2
// entries; any two when the pairs are neighbours), so the rotation needs no exchange, and the row sums
// are one shuffle tree.  The group walks several heads of ONE token with the lane's angles and weights
// in registers: read per row, the tables would be as much traffic as the row itself.  Rows whose size,
// alignment or R does not split that way take a second kernel, one row at a time, that
// exchanges the pairs through shared memory.
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
  float eps;
  int chunk[2], chunks[2];        // heads a group walks; how many such runs a token has
  long long units[2];             // B * S * chunks
  int ctas[2];                    // backward: CTAs of each tensor
  float* part;                    // backward: [ctas][D] partial weight gradients; null when none is wanted
  int* status;
  unsigned long long y_extent[2]; // bounds-checking build
  unsigned long long* bounds_detail;
};

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ static uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ static float one(const __nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 round(float v) { return __float2bfloat16(v); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  __device__ static float one(const float v) { return v; }
  __device__ static float round(float v) { return v; }
};

__device__ __forceinline__ float weight_at(const RopeParams& p, int which, int i) {
  if (!p.w[which]) return 1.f;
  return p.w_f32 ? static_cast<const float*>(p.w[which])[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.w[which])[i]);
}

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

// Vector path: LPR lanes per row, two vectors per lane.  BWD: the gradients.  U rows are in flight.
template <typename T, int LPR, bool IL, bool BWD>
__global__ void __launch_bounds__(RN_THREADS) rope_vec_kernel(const RopeParams p) {
  constexpr int N = Vec<T>::N;
  constexpr int GROUPS = RN_THREADS / LPR;
  constexpr int U = BWD ? 2 : 4;
  __shared__ float red[BWD ? RN_THREADS / 32 : 1][BWD ? 256 : 1];
  const int gl = threadIdx.x % LPR;
  const int group = threadIdx.x / LPR;
  const int nv = p.D / N;
  // the lane's vectors
  const int hp = IL ? 0 : p.R / (2 * N);
  const bool mates = gl < hp;
  const int va = mates ? gl : 2 * hp + 2 * (gl - hp);
  const int vb = mates ? gl + hp : va + 1;
  const bool has_a = va < nv, has_b = vb < nv;
  // whether the lane's vectors are rotated (R is a multiple of a vector)
  const bool rot_a = IL ? va * N < p.R : mates, rot_b = IL ? vb * N < p.R : mates;
  float acc_a[N], acc_b[N];
  if (BWD) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc_a[i] = acc_b[i] = 0.f;
  }
  const long long total = BWD ? 0 : p.units[0] + p.units[1];
  const int cta_type = BWD && static_cast<int>(blockIdx.x) >= p.ctas[0] ? 1 : 0;
  const long long end = BWD ? p.units[cta_type] : total;
  const long long cta = BWD ? static_cast<long long>(blockIdx.x) - (cta_type ? p.ctas[0] : 0) : blockIdx.x;
  const long long step = static_cast<long long>(BWD ? p.ctas[cta_type] : gridDim.x) * GROUPS;
  // the same for every lane of the warp, whichever tensor its group is at: there are shuffles inside
  const int rounds = BWD ? p.chunk[cta_type] : max(p.chunk[0], p.chunk[1]);
  int loaded_type = -1;
  float wa[N], wb[N];
  // every lane of a warp makes the same number of rounds (shuffles inside); units past the end idle
  for (long long u0 = cta * GROUPS; u0 < end; u0 += step) {
    const long long uu = u0 + group;
    const bool live = uu < end;
    long long u = live ? uu : end - 1;
    int type = cta_type;
    if (!BWD && u >= p.units[0]) {
      type = 1;
      u -= p.units[0];
    }
    const long long token = u / p.chunks[type];
    const int h_first = static_cast<int>(u - token * p.chunks[type]) * p.chunk[type];
    const int b = static_cast<int>(token / p.S), s = static_cast<int>(token - static_cast<long long>(b) * p.S);
    const int h_end = min(h_first + p.chunk[type], p.heads[type]);
    if (type != loaded_type) {
      loaded_type = type;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        wa[i] = has_a ? weight_at(p, type, va * N + i) : 0.f;
        wb[i] = has_b ? weight_at(p, type, vb * N + i) : 0.f;
      }
    }
    // angles: half-split, pair i of the lane = (a_i, b_i); neighbours, pairs 0.. of a then those of b
    float c[N], sn[N];
    {
      const long long tr = table_row(p, b, s);
      const float* ct = p.cs + tr * (p.R / 2);
      const float* st = p.sn + tr * (p.R / 2);
      const float bad = __int_as_float(0x7FC00000);
      if (IL) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool rot = i < N / 2 ? rot_a && has_a : rot_b && has_b;
          const int at = i < N / 2 ? va * (N / 2) + i : vb * (N / 2) + i - N / 2;
          c[i] = rot ? (tr >= 0 ? ct[at] : bad) : 1.f;
          sn[i] = rot ? (tr >= 0 ? st[at] : bad) : 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          float4 c4 = make_float4(bad, bad, bad, bad), s4 = c4;
          if (mates && tr >= 0) {
            c4 = *reinterpret_cast<const float4*>(ct + va * N + i);
            s4 = *reinterpret_cast<const float4*>(st + va * N + i);
          }
          c[i] = c4.x, c[i + 1] = c4.y, c[i + 2] = c4.z, c[i + 3] = c4.w;
          sn[i] = s4.x, sn[i + 1] = s4.y, sn[i + 2] = s4.z, sn[i + 3] = s4.w;
        }
      }
    }
    const T* x = static_cast<const T*>(p.x[type]) + b * p.xs[type][0] + s * p.xs[type][2];
    const T* dy = BWD ? static_cast<const T*>(p.dy[type]) + b * p.ds[type][0] + s * p.ds[type][2] : nullptr;
    const long long y0 = b * p.ys[type][0] + s * p.ys[type][2];
    for (int h0 = 0; h0 < rounds; h0 += U) {
      uint4 xv[U][2], dv[BWD ? U : 1][2];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int h = h_first + h0 + k;
        const bool on = live && h0 + k < p.chunk[type] && h < h_end;
        xv[k][0] = xv[k][1] = make_uint4(0u, 0u, 0u, 0u);
        if (BWD) dv[k][0] = dv[k][1] = make_uint4(0u, 0u, 0u, 0u);
        if (on) {
          const T* xr = x + h * p.xs[type][1];
          if (has_a) xv[k][0] = *reinterpret_cast<const uint4*>(xr + va * N);
          if (has_b) xv[k][1] = *reinterpret_cast<const uint4*>(xr + vb * N);
          if (BWD) {
            const T* dr = dy + h * p.ds[type][1];
            if (has_a) dv[k][0] = *reinterpret_cast<const uint4*>(dr + va * N);
            if (has_b) dv[k][1] = *reinterpret_cast<const uint4*>(dr + vb * N);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int h = h_first + h0 + k;
        const bool on = live && h0 + k < p.chunk[type] && h < h_end;
        float a[N], bb[N], ss = 0.f;
        Vec<T>::unpack(xv[k][0], a);
        Vec<T>::unpack(xv[k][1], bb);
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(a[i], a[i], fmaf(bb[i], bb[i], ss));
        ss = group_sum<LPR>(ss);
        const float r = rsqrtf(ss / p.D + p.eps);
        float oa[N], ob[N];
        if (!BWD) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            oa[i] = a[i] * r * wa[i];
            ob[i] = bb[i] * r * wb[i];
          }
          if (IL) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              const float a0 = oa[2 * i], a1 = oa[2 * i + 1], b0 = ob[2 * i], b1 = ob[2 * i + 1];
              if (rot_a) oa[2 * i] = a0 * c[i] - a1 * sn[i], oa[2 * i + 1] = a1 * c[i] + a0 * sn[i];
              if (rot_b) ob[2 * i] = b0 * c[N / 2 + i] - b1 * sn[N / 2 + i], ob[2 * i + 1] = b1 * c[N / 2 + i] + b0 * sn[N / 2 + i];
            }
          } else if (mates) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float f = oa[i], g = ob[i];
              oa[i] = f * c[i] - g * sn[i];
              ob[i] = g * c[i] + f * sn[i];
            }
          }
        } else {
          float ga[N], gb[N], dot = 0.f;
          Vec<T>::unpack(dv[k][0], ga);
          Vec<T>::unpack(dv[k][1], gb);
          if (IL) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              const float a0 = ga[2 * i], a1 = ga[2 * i + 1], b0 = gb[2 * i], b1 = gb[2 * i + 1];
              if (rot_a) ga[2 * i] = a0 * c[i] + a1 * sn[i], ga[2 * i + 1] = a1 * c[i] - a0 * sn[i];
              if (rot_b) gb[2 * i] = b0 * c[N / 2 + i] + b1 * sn[N / 2 + i], gb[2 * i + 1] = b1 * c[N / 2 + i] - b0 * sn[N / 2 + i];
            }
          } else if (mates) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float f = ga[i], g = gb[i];
              ga[i] = f * c[i] + g * sn[i];
              gb[i] = g * c[i] - f * sn[i];
            }
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (on) {
              acc_a[i] = fmaf(ga[i] * r, a[i], acc_a[i]);
              acc_b[i] = fmaf(gb[i] * r, bb[i], acc_b[i]);
            }
            ga[i] *= wa[i];
            gb[i] *= wb[i];
            dot = fmaf(ga[i], a[i], fmaf(gb[i], bb[i], dot));
          }
          // x r^3 mean(g w x): the factors in an order that neither overflows nor vanishes for tiny rows
          const float m = group_sum<LPR>(dot * r) / p.D;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            oa[i] = r * (ga[i] - (a[i] * r) * m);
            ob[i] = r * (gb[i] - (bb[i] * r) * m);
          }
        }
        if (on) {
          const long long at = y0 + h * p.ys[type][1];
          T* yr = static_cast<T*>(p.y[type]) + at;
          if (has_a && bounds_ok((at + va * N) * sizeof(T), 16, p.y_extent[type], p.status, p.bounds_detail))
            *reinterpret_cast<uint4*>(yr + va * N) = Vec<T>::pack(oa);
          if (has_b && bounds_ok((at + vb * N) * sizeof(T), 16, p.y_extent[type], p.status, p.bounds_detail))
            *reinterpret_cast<uint4*>(yr + vb * N) = Vec<T>::pack(ob);
        }
      }
    }
  }
  if (BWD && p.part) {
    // lanes of equal place in their group, then the warps, in a fixed order
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        acc_a[i] += __shfl_xor_sync(0xFFFFFFFFu, acc_a[i], o);
        acc_b[i] += __shfl_xor_sync(0xFFFFFFFFu, acc_b[i], o);
      }
    }
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) < LPR) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (has_a) red[warp][va * N + i] = acc_a[i];
        if (has_b) red[warp][vb * N + i] = acc_b[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += RN_THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < RN_THREADS / 32; ++k) sum += red[k][i];
      p.part[static_cast<long long>(blockIdx.x) * p.D + i] = sum;
    }
  }
}

// Any even D <= 256, any even R <= D, any alignment: a warp per row; VEC entries per access (16 bytes
// where the rows allow it), the pairs exchanged through shared memory.
template <typename T, int VEC, bool BWD>
__global__ void __launch_bounds__(RN_THREADS) rope_row_kernel(const RopeParams p) {
  constexpr int WARPS = RN_THREADS / 32;
  constexpr int PER = 256 / (32 * VEC) ? 256 / (32 * VEC) : 1;   // accesses per lane
  __shared__ float rows[WARPS][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* row = rows[warp];
  float acc[PER][VEC];
#pragma unroll
  for (int j = 0; j < PER; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[j][i] = 0.f;
  const int cta_type = BWD && static_cast<int>(blockIdx.x) >= p.ctas[0] ? 1 : 0;
  const long long end = BWD ? p.units[cta_type] : p.units[0] + p.units[1];
  const long long cta = BWD ? static_cast<long long>(blockIdx.x) - (cta_type ? p.ctas[0] : 0) : blockIdx.x;
  const long long step = static_cast<long long>(BWD ? p.ctas[cta_type] : gridDim.x) * WARPS;
  const int half = p.R / 2;
  // index of entry i's mate, of the pair's angle, and the sign of the mate's term in the forward rotation
  auto mate = [&](int i) { return p.interleaved ? i ^ 1 : (i < half ? i + half : i - half); };
  auto angle = [&](int i) { return p.interleaved ? i >> 1 : (i < half ? i : i - half); };
  auto first = [&](int i) { return p.interleaved ? !(i & 1) : i < half; };
  for (long long uu = cta * WARPS + warp; uu < end; uu += step) {
    long long u = uu;
    int type = cta_type;
    if (!BWD && u >= p.units[0]) {
      type = 1;
      u -= p.units[0];
    }
    // a unit is one row here (chunk = 1)
    const long long token = u / p.heads[type];
    const int h = static_cast<int>(u - token * p.heads[type]);
    const int b = static_cast<int>(token / p.S), s = static_cast<int>(token - static_cast<long long>(b) * p.S);
    const T* x = static_cast<const T*>(p.x[type]) + b * p.xs[type][0] + h * p.xs[type][1] + s * p.xs[type][2];
    const T* dy = BWD ? static_cast<const T*>(p.dy[type]) + b * p.ds[type][0] + h * p.ds[type][1] + s * p.ds[type][2] : nullptr;
    const long long y0 = b * p.ys[type][0] + h * p.ys[type][1] + s * p.ys[type][2];
    T* y = static_cast<T*>(p.y[type]) + y0;
    float xv[PER][VEC], ss = 0.f;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int at = (j * 32 + lane) * VEC;
      float other[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) xv[j][i] = other[i] = 0.f;
      if (at < p.D) {
        if constexpr (VEC == 1) {
          xv[j][0] = Vec<T>::one(x[at]);
          if (BWD) other[0] = Vec<T>::one(dy[at]);
        } else {
          Vec<T>::unpack(*reinterpret_cast<const uint4*>(x + at), xv[j]);
          if (BWD) Vec<T>::unpack(*reinterpret_cast<const uint4*>(dy + at), other);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) row[at + i] = BWD ? other[i] : xv[j][i] * weight_at(p, type, at + i);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(xv[j][i], xv[j][i], ss);
    }
    ss = group_sum<32>(ss);
    const float r = rsqrtf(ss / p.D + p.eps);
    const long long tr = table_row(p, b, s);
    __syncwarp();
    // forward: y = r * rotation of x w; backward: g = dy rotated back
    float out[PER][VEC], dot = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int e = (j * 32 + lane) * VEC + i;
        out[j][i] = 0.f;
        if (e >= p.D) continue;
        float v = row[e];
        if (e < p.R) {
          const float c = tr >= 0 ? p.cs[tr * half + angle(e)] : __int_as_float(0x7FC00000);
          const float sn = tr >= 0 ? p.sn[tr * half + angle(e)] : c;
          const float m = row[mate(e)] * sn;
          v = v * c + (first(e) == BWD ? m : -m);
        }
        if (BWD) {
          acc[j][i] = fmaf(v * r, xv[j][i], acc[j][i]);
          v *= weight_at(p, type, e);
          dot = fmaf(v, xv[j][i], dot);
          out[j][i] = v;
        } else {
          out[j][i] = r * v;
        }
      }
    if (BWD) {
      const float m = group_sum<32>(dot * r) / p.D;
#pragma unroll
      for (int j = 0; j < PER; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[j][i] = r * (out[j][i] - (xv[j][i] * r) * m);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int at = (j * 32 + lane) * VEC;
      if (at < p.D && bounds_ok((y0 + at) * sizeof(T), VEC * sizeof(T), p.y_extent[type], p.status, p.bounds_detail)) {
        if constexpr (VEC == 1)
          y[at] = Vec<T>::round(out[j][0]);
        else
          *reinterpret_cast<uint4*>(y + at) = Vec<T>::pack(out[j]);
      }
    }
  }
  if (BWD && p.part) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int e = (j * 32 + lane) * VEC + i;
        if (e < p.D) row[e] = acc[j][i];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += RN_THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) sum += rows[k][i];
      p.part[static_cast<long long>(blockIdx.x) * p.D + i] = sum;
    }
  }
}

// dw[i] = sum of the CTAs' partial sums, in a fixed order: 32 columns per CTA, 8 rows at a time.
__global__ void __launch_bounds__(256) rope_weight_sum_kernel(const float* part, int first, int count, int D, float* dw0,
                                                              int count1, float* dw1) {
  __shared__ float red[8][33];
  const int which = blockIdx.y;
  float* dw = which ? dw1 : dw0;
  if (!dw) return;
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), sub = threadIdx.x >> 5;
  const int begin = which ? first + count : first, n = which ? count1 : count;
  float sum = 0.f;
  if (col < D)
    for (int i = sub; i < n; i += 8) sum += part[static_cast<long long>(begin + i) * D + col];
  red[sub][threadIdx.x & 31] = sum;
  __syncthreads();
  if (sub == 0 && col < D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += red[k][threadIdx.x & 31];
    dw[col] = sum;
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

// CTAs that the backward pass may use for each tensor: at most four per SM over both, so that the
// partial weight gradients stay few.  A function of the shape alone (the workspace query has no pointers).
void bwd_ctas(const kcg_rope_desc* d, int& q, int& k) {
  const int most = 4 * 148;
  const long long heads = static_cast<long long>(d->H) + d->Hk;
  k = d->Hk ? static_cast<int>(most * static_cast<long long>(d->Hk) / heads) : 0;
  if (d->Hk && k < 1) k = 1;
  q = most - k;
}

template <typename T, int LPR, bool IL, bool BWD>
void go_vec(const RopeParams& p, unsigned grid, cudaStream_t stream) {
  rope_vec_kernel<T, LPR, IL, BWD><<<grid, RN_THREADS, 0, stream>>>(p);
}
template <typename T, bool IL, bool BWD>
void go_vec(const RopeParams& p, int lpr, unsigned grid, cudaStream_t stream) {
  switch (lpr) {
    case 4: return go_vec<T, 4, IL, BWD>(p, grid, stream);
    case 8: return go_vec<T, 8, IL, BWD>(p, grid, stream);
    case 16: return go_vec<T, 16, IL, BWD>(p, grid, stream);
    default: return go_vec<T, 32, IL, BWD>(p, grid, stream);
  }
}

template <typename T, bool BWD>
kcg_status_t launch_rope(RopeParams& p, const kcg_rope_desc* d, bool vectors, cudaStream_t stream) {
  constexpr int N = Vec<T>::N;
  const int nv = d->D / N;
  // the vector path: whole vectors, and both members of each pair in vectors of one lane
  const bool vec = vectors && d->D % N == 0 && (d->interleaved ? d->R % N == 0 : d->R % (2 * N) == 0);
  int lpr = 4;
  while (2 * lpr < nv) lpr *= 2;
  const int per_cta = vec ? RN_THREADS / lpr : RN_THREADS / 32;
  const long long tokens = static_cast<long long>(d->B) * d->S, sms = device_sm_count();
  for (int t = 0; t < 2; ++t) {
    // heads a group walks with one set of angles: as many as leave two groups' worth of work for
    // every group that the SMs hold (2048 threads each), at most 8
    int chunk = 1;
    if (vec)
      while (chunk < 8 && 2 * chunk <= p.heads[t] && tokens * p.heads[t] / (2 * chunk) >= sms * (2048 / RN_THREADS) * per_cta) chunk *= 2;
    p.chunk[t] = chunk;
    p.chunks[t] = p.heads[t] ? (p.heads[t] + chunk - 1) / chunk : 0;
    p.units[t] = tokens * p.chunks[t];
  }
  unsigned grid;
  if (BWD) {
    for (int t = 0; t < 2; ++t) {
      const long long want = (p.units[t] + per_cta - 1) / per_cta;
      if (p.ctas[t] > want) p.ctas[t] = static_cast<int>(want);
    }
    grid = static_cast<unsigned>(p.ctas[0] + p.ctas[1]);
  } else {
    const long long want = (p.units[0] + p.units[1] + per_cta - 1) / per_cta, most = 16 * sms;
    grid = static_cast<unsigned>(want < most ? want : most);
  }
  if (vec) {
    if (d->interleaved) go_vec<T, true, BWD>(p, lpr, grid, stream);
    else go_vec<T, false, BWD>(p, lpr, grid, stream);
  } else if (vectors && d->D % N == 0) {
    rope_row_kernel<T, N, BWD><<<grid, RN_THREADS, 0, stream>>>(p);
  } else {
    rope_row_kernel<T, 1, BWD><<<grid, RN_THREADS, 0, stream>>>(p);
  }
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
    p.x[t] = x[t], p.dy[t] = dy[t], p.y[t] = y[t], p.w[t] = w[t];
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
  p.part = nullptr;
  p.ctas[0] = p.ctas[1] = 0;
  if (const unsigned long long cap = debug_extent_limit())
    for (unsigned long long& e : p.y_extent) e = e < cap ? e : cap;
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
  const bool sums = dwq || (dwk && d->Hk);
  if (sums) {
    if (!ws || ws_bytes < qk_norm_rope_bwd_workspace_impl(d) || !aligned16(ws)) return KCG_BAD_WORKSPACE;
    p.part = static_cast<float*>(ws);
  }
  bwd_ctas(d, p.ctas[0], p.ctas[1]);
  st = d->dtype == KCG_F32 ? launch_rope<float, true>(p, d, vectors, stream)
                           : launch_rope<__nv_bfloat16, true>(p, d, vectors, stream);
  if (st != KCG_OK || !sums) return st;
  rope_weight_sum_kernel<<<dim3(static_cast<unsigned>((d->D + 31) / 32), 2), 256, 0, stream>>>(
      p.part, 0, p.ctas[0], d->D, dwq, p.ctas[1], d->Hk ? dwk : nullptr);
  g_launches.fetch_add(1);
  KCG_CUDA_TRY(cudaGetLastError());
  return KCG_OK;
}

}  // namespace kcg
