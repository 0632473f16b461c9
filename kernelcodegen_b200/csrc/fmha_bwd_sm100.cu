// Gradients of O = softmax(scale * Q.K^T [causal]) . V on sm_100a.
//
//   P_ij  = exp(scale q_i.k_j - lse_i)            recomputed from the forward pass's lse, never stored
//   delta_i = dO_i.O_i,  dS_ij = P_ij (dO_i.v_j - delta_i)
//   dV_j = sum_i P_ij dO_i    dK_j = scale sum_i dS_ij q_i    dQ_i = scale sum_j dS_ij k_j
//
// dK and dV sum over queries, dQ over keys.  One sweep for all three needs dQ added up across CTAs
// (fp32 atomics whose order, and so whose rounding, differs from run to run, and a 32-bit dQ in
// memory that costs as much L2 traffic per tile as the tile's four operands).  Here a launch holds
// two kinds of work item instead, each of which owns what it writes:
//
//   kv item  128 keys of one key/value head; streams the query tiles of all its query heads:
//            S^T = K.Q^T, dP^T = V.dO^T, dV += P^T.dO, dK += dS^T.Q           (4 products a tile)
//   q item   128 queries of one query head; streams the key tiles:
//            S = Q.K^T, dP = dO.V^T, dQ += dS.K                               (3 products a tile)
//
// 7 products instead of 5, no atomics, no 32-bit gradient in memory, the same bits on every call.
//
// In both, P and dS are computed with the row of the ACCUMULATOR (one TMEM lane) in one thread's
// registers, written back to TMEM as bf16 over the columns they came from and used from there as the
// A operand of the accumulating products: nothing passes through shared memory but the TMA tiles,
// whose K-major form feeds S and dP and whose MN-major reading of the same bytes feeds dV, dK, dQ.
//
//   warp 0       TMA producer: two fixed tiles, then two streams (X, Y) of two stages each
//   warp 1       UMMA issuer
//   warps 4..11  P and dS: thread = accumulator row and one half of the tile's 128 columns
//
//             fixed A0, A1    stream X, Y    S = A0.X^T   dP = A1.Y^T   acc1 += dS.X   acc0 += P.Y
//   kv item   K, V            Q, dO          S^T          dP^T          dK             dV
//   q item    Q, dO           K, V           S            dP            dQ             -
//
// While the softmax warps turn S into P the tensor core works on the previous tile's acc1 product and
// this tile's dP; while they turn dP into dS it works on acc0 and the next tile's S.
#include "common.cuh"
#include "ptx.cuh"

namespace kcg {

namespace {

constexpr int BW_THREADS = 384;
constexpr int BT = 128;          // rows of every tile, and of a work item

struct BwdParams {
  void *dQ, *dK, *dV;
  long long q_sb, q_sh, q_sr, k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;   // strides of the gradients, elements
  const float* nlse;      // [B * H][sq_pad] -lse * log2(e); -inf for rows without a visible key and past Sq
  const float* ndelta;    // [B * H][sq_pad] -delta; 0 past Sq
  int H, Hkv, group;
  int Sq, Skv, sq_pad;
  int causal;
  float scale, scale_log2;
  int n_qt, n_kt;         // tiles of queries, of keys
  int kv_items;           // B * Hkv * n_kt; the q items follow
  int kv_group, kv_small; // order of the items, see item_of()
  int q_group, q_small;
  int* status;
  uint32_t spin;
  unsigned long long dq_extent, dk_extent, dv_extent;   // bounds-checking build
  unsigned long long* bounds_detail;
};

template <int D>
struct BwdCfg {
  static constexpr int TILE_BYTES = BT * D * 2;
  static constexpr int PANEL_BYTES = 128 * 128;       // 128 rows x 64 bf16
  static constexpr int DPANELS = D / 64;
  static constexpr int STAT_BYTES = 2 * BT * 4;       // -lse and -delta of a query tile
  static constexpr int SMEM_DATA = 6 * TILE_BYTES;    // A0, A1, X[2], Y[2]
  static constexpr int SMEM_TOTAL = SMEM_DATA + 2 * STAT_BYTES + 1024 /*ctrl*/ + 1024 /*align slack*/;
  static constexpr int TMEM_COLS = 512;
};

// Item index -> (head, tile).  The heads are walked in groups whose streamed tensors stay in L2;
// inside a group the tiles of all heads go together, `tile` counting from the longest.  Groups are
// equal up to one head: the first `small` hold one head fewer.
__device__ __forceinline__ void item_of(int idx, int tiles, int group, int small, int& head, int& tile) {
  int gsz = group - 1, g0 = 0;
  const int small_items = small * gsz * tiles;
  if (idx >= small_items) {
    idx -= small_items;
    gsz = group;
    g0 = small * (group - 1);
  }
  const int grp = idx / (gsz * tiles);
  const int rem = idx - grp * gsz * tiles;
  tile = rem / gsz;
  head = g0 + grp * gsz + (rem - tile * gsz);
}

// Shared between the two kinds of item.
struct BwdSmem {
  uint32_t a0, a1, x, y, stat;      // tiles; X, Y and stat have two stages
  uint32_t bar_fixed, bar_xfull, bar_xempty, bar_yfull, bar_yempty, bar_sfull, bar_pfull, bar_dpfull, bar_dsfull, bar_done;
};

// 2^x of pair k of a row: a share of the pairs (a fixed pattern, so that the two kinds of instruction
// interleave) takes the FMA-pipe polynomial, the rest the MUFU unit, which alone would need 1024 clocks
// for a 128 x 128 tile, as long as two of the tile's products.
constexpr int POLY_EIGHTHS = 3;
__device__ __forceinline__ float2 exp2_share(int k, float2 x) {
  if (((k * 5) & 7) < POLY_EIGHTHS) {
    x.x = fmaxf(x.x, -125.f);   // the polynomial's lower end: such a P is 2^-125, nothing in any sum
    x.y = fmaxf(x.y, -125.f);
    return ex2_quartic2(x);
  }
  x.x = ex2_approx(x.x);
  x.y = ex2_approx(x.y);
  return x;
}

// Two bf16 rows of 32 columns each from 64 floats: the A operand's form, two elements per TMEM column.
__device__ __forceinline__ void store_a_half(uint32_t taddr, const float2 (&v)[32]) {
  uint32_t pk[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) pk[i] = pack_bf16x2(v[i].x, v[i].y);
  tmem_st_32x32(taddr, pk);
}

template <int D, bool KV>
__device__ __forceinline__ void bwd_item(const CUtensorMap* tmA0, const CUtensorMap* tmA1, const CUtensorMap* tmX,
                                         const CUtensorMap* tmY, const BwdParams& p, int idx, const BwdSmem& sm,
                                         const float* stat_gen, uint32_t tmem_base, volatile int* abort_flag) {
  using Cfg = BwdCfg<D>;
  constexpr int TILE = Cfg::TILE_BYTES, PANEL = Cfg::PANEL_BYTES, DPANELS = Cfg::DPANELS;
  // S has two buffers where TMEM has room: S(i+1) is then computed ahead of everything of tile i
  constexpr int NS = (KV && D == 128) ? 1 : 2;
  constexpr uint32_t TM_S = 0, TM_DP = NS * 128, TM_ACC0 = TM_DP + 128, TM_ACC1 = KV ? TM_ACC0 + D : TM_ACC0;
  static_assert(TM_ACC1 + D <= 512, "TMEM columns");
  constexpr uint32_t IDESC_S = make_idesc(UMMA_FMT_BF16, BT, BT, 0, 0);
  constexpr uint32_t IDESC_ACC = make_idesc(UMMA_FMT_BF16, BT, D, 0, 1);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int shift = p.Skv - p.Sq;    // causal: query i sees keys j <= i + shift

  // the item: rows row0.. of head `head` of batch b; the tiles it streams: first..first+n_tiles-1 of
  // each of n_heads heads from head h0 on
  int head, tile, b, row0, first, n_tiles, h0, n_heads;
  if (KV) {
    item_of(idx, p.n_kt, p.kv_group, p.kv_small, head, tile);   // causal: key tile 0 is the longest
    b = head / p.Hkv;
    head -= b * p.Hkv;
    row0 = tile * BT;
    first = 0;
    if (p.causal) {
      const int q_min = row0 - shift;                           // the first query that sees a key of the tile
      first = q_min > 0 ? q_min / BT : 0;
    }
    n_tiles = p.n_qt > first ? p.n_qt - first : 0;
    h0 = head * p.group;
    n_heads = p.group;
  } else {
    item_of(idx, p.n_qt, p.q_group, p.q_small, head, tile);
    b = head / p.H;
    head -= b * p.H;
    if (p.causal) tile = p.n_qt - 1 - tile;
    row0 = tile * BT;
    first = 0;
    int end = p.Skv;
    if (p.causal) {
      const int lim = row0 + BT + shift;
      end = lim < end ? lim : end;
      if (end < 0) end = 0;
    }
    n_tiles = (end + BT - 1) / BT;
    h0 = head / p.group;
    n_heads = 1;
  }
  const int n_it = n_tiles * n_heads;

  if (warp == 0) {
    if (lane == 0 && n_it > 0) {
      // ------------------------------- TMA producer -------------------------------------------
      mbar_expect_tx(sm.bar_fixed, 2 * TILE);
#pragma unroll
      for (int dp = 0; dp < DPANELS; ++dp) {
        tma_load_4d(sm.a0 + dp * PANEL, tmA0, sm.bar_fixed, dp * 64, row0, head, b);
        tma_load_4d(sm.a1 + dp * PANEL, tmA1, sm.bar_fixed, dp * 64, row0, head, b);
      }
      bool ok = true;
      int armed = 0;
      int t = first, h = h0;
      for (int i = 0; i < n_it; ++i) {
        const int st = i & 1;
        const uint32_t par = ((i >> 1) & 1u) ^ 1u;
        ok = mbar_wait(sm.bar_xempty + 8 * st, par, abort_flag, p.status, DEV_TIMEOUT_PRODUCER, p.spin);
        if (!ok) break;
        mbar_expect_tx(sm.bar_xfull + 8 * st, TILE + (KV ? Cfg::STAT_BYTES : 0));
#pragma unroll
        for (int dp = 0; dp < DPANELS; ++dp)
          tma_load_4d(sm.x + st * TILE + dp * PANEL, tmX, sm.bar_xfull + 8 * st, dp * 64, t * BT, h, b);
        if (KV) {
          // written by the launch before this one; the tiles above are not
          if (i == 0) griddep_wait();
          const size_t at = (static_cast<size_t>(b) * p.H + h) * p.sq_pad + static_cast<size_t>(t) * BT;
          bulk_load(sm.stat + st * Cfg::STAT_BYTES, p.nlse + at, BT * 4, sm.bar_xfull + 8 * st);
          bulk_load(sm.stat + st * Cfg::STAT_BYTES + BT * 4, p.ndelta + at, BT * 4, sm.bar_xfull + 8 * st);
        }
        armed = i + 1;
        ok = mbar_wait(sm.bar_yempty + 8 * st, par, abort_flag, p.status, DEV_TIMEOUT_PRODUCER, p.spin);
        if (!ok) break;
        mbar_expect_tx(sm.bar_yfull + 8 * st, TILE);
#pragma unroll
        for (int dp = 0; dp < DPANELS; ++dp)
          tma_load_4d(sm.y + st * TILE + dp * PANEL, tmY, sm.bar_yfull + 8 * st, dp * 64, t * BT, h, b);
        if (++t == first + n_tiles) {
          t = first;
          ++h;
        }
      }
      if (!ok) {
        // copies in flight land before shared memory is released: the last two arms of each ring
        for (int i = armed > 2 ? armed - 2 : 0; i < armed; ++i)
          for (uint32_t it = 0; it < 65536u; ++it)
            if (mbar_try_wait(sm.bar_xfull + 8 * (i & 1), (i >> 1) & 1u) &&
                (i == armed - 1 || mbar_try_wait(sm.bar_yfull + 8 * (i & 1), (i >> 1) & 1u)))
              break;
        for (uint32_t it = 0; it < 65536u; ++it)
          if (mbar_try_wait(sm.bar_fixed, 0)) break;
      }
    }
  } else if (warp == 1) {
    if (n_it > 0) {
      // ------------------------------- UMMA issuer --------------------------------------------
      bool ok = true;
      auto wait_all = [&](uint32_t bar, uint32_t parity, int code) -> bool {
        return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, p.status, code, p.spin));
      };
      constexpr uint64_t TILE16 = TILE >> 4;
      const uint64_t a0_desc = make_smem_desc(sm.a0, 16, 1024), a1_desc = make_smem_desc(sm.a1, 16, 1024);
      const uint64_t x_desc = make_smem_desc(sm.x, 16, 1024), y_desc = make_smem_desc(sm.y, 16, 1024);
      const uint64_t xt_desc = make_smem_desc(sm.x, PANEL, 1024), yt_desc = make_smem_desc(sm.y, PANEL, 1024);
      // 128 x 128 += A . B^T over the head dimension, both K-major
      auto issue_ss = [&](uint32_t d_tmem, uint64_t ad, uint64_t bd, uint32_t bar) {
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint64_t off = static_cast<uint64_t>(((ks >> 2) * PANEL + (ks & 3) * 32) >> 4);
            umma_bf16_ss(d_tmem, ad + off, bd + off, IDESC_S, ks ? 1u : 0u);
          }
          umma_commit(bar);
        }
        __syncwarp();
      };
      // acc (+)= A . B over the tile's 128 rows: A in TMEM (the halves of the columns 64 apart), B MN-major
      auto issue_ts = [&](uint32_t d_tmem, uint32_t a_tmem, uint64_t bd, bool accumulate, uint32_t bar) {
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            umma_bf16_ts(d_tmem, a_tmem + 64 * (ks >> 2) + 8 * (ks & 3), bd + static_cast<uint64_t>((ks * 16 * 128) >> 4),
                         IDESC_ACC, (accumulate || ks) ? 1u : 0u);
          if (bar) umma_commit(bar);
        }
        __syncwarp();
      };
      auto issue_s = [&](int i) -> bool {
        if (!wait_all(sm.bar_xfull + 8 * (i & 1), (i >> 1) & 1u, DEV_TIMEOUT_MMA_FULL)) return false;
        tc_fence_after();
        issue_ss(tmem_base + TM_S + (NS == 2 ? (i & 1) * 128 : 0), a0_desc, x_desc + (i & 1) * TILE16,
                 sm.bar_sfull + 8 * (NS == 2 ? (i & 1) : 0));
        return true;
      };
      auto issue_dp = [&](int i) -> bool {
        if (!wait_all(sm.bar_yfull + 8 * (i & 1), (i >> 1) & 1u, DEV_TIMEOUT_MMA_FULL)) return false;
        tc_fence_after();
        issue_ss(tmem_base + TM_DP, a1_desc, y_desc + (i & 1) * TILE16, sm.bar_dpfull);
        // the last product that reads Y, except in a kv item, whose dV reads it once more
        if (!KV) {
          if (elect_one()) umma_commit(sm.bar_yempty + 8 * (i & 1));
          __syncwarp();
        }
        return true;
      };
      ok = wait_all(sm.bar_fixed, 0, DEV_TIMEOUT_Q) && issue_s(0) && issue_dp(0);
      for (int i = 0; i < n_it && ok; ++i) {
        const bool next = i + 1 < n_it;
        const uint32_t s_buf = tmem_base + TM_S + (NS == 2 ? (i & 1) * 128 : 0);
        if (NS == 2 && next && !(ok = issue_s(i + 1))) break;
        if (KV) {
          if (!(ok = wait_all(sm.bar_pfull, i & 1u, DEV_TIMEOUT_P))) break;
          tc_fence_after();
          issue_ts(tmem_base + TM_ACC0, s_buf, yt_desc + (i & 1) * TILE16, i > 0, sm.bar_yempty + 8 * (i & 1));
        }
        if (NS == 1 && next && !(ok = issue_s(i + 1))) break;
        if (!(ok = wait_all(sm.bar_dsfull, i & 1u, DEV_TIMEOUT_P))) break;
        tc_fence_after();
        issue_ts(tmem_base + TM_ACC1, tmem_base + TM_DP, xt_desc + (i & 1) * TILE16, i > 0, sm.bar_xempty + 8 * (i & 1));
        if (next && !(ok = issue_dp(i + 1))) break;
      }
      if (elect_one()) umma_commit(sm.bar_done);
      __syncwarp();
      if (!ok) {
        // products in flight finish before TMEM is freed
        for (uint32_t it = 0; it < 65536u; ++it)
          if (mbar_try_wait(sm.bar_done, 0)) break;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------- P and dS, then the output ----------------------------------
    const int half = (warp >> 2) - 1;          // columns 64 * half .. + 63 of every tile
    const int q = warp & 3;                    // TMEM lane quarter this warp may access
    const int r = q * 32 + lane;               // row inside the item
    const int row = row0 + r;
    const uint32_t t_lane = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t t_col = tmem_base + t_lane + 64 * half;
    const float c = p.scale_log2;
    float nl = 0.f, nd = 0.f;
    if (!KV && n_it > 0) {
      griddep_wait();
      const size_t at = (static_cast<size_t>(b) * p.H + head) * p.sq_pad + row;   // row < sq_pad
      nl = p.nlse[at];
      nd = p.ndelta[at];
    }
    bool ok = true;
    int t = first;
    for (int i = 0; i < n_it && ok; ++i) {
      // visible columns of this thread's half: [lo, hi)
      int lo = 0, hi = 64;
      bool mask;
      if (KV) {
        const int q0 = t * BT;
        mask = p.causal && row0 + BT - 1 > q0 + shift;
        lo = row - shift - q0 - 64 * half;     // query >= key - shift
        if (++t == first + n_tiles) t = first;
      } else {
        const int k0 = i * BT;
        int limit = p.Skv;
        if (p.causal) {
          const int l2 = row + shift + 1;
          limit = l2 < limit ? l2 : limit;
        }
        mask = k0 + BT > p.Skv || (p.causal && k0 + BT > row0 + shift + 1);
        hi = limit - k0 - 64 * half;
      }
      const uint32_t s_addr = t_col + TM_S + (NS == 2 ? (i & 1) * 128 : 0);
      const uint32_t s_bar = sm.bar_sfull + 8 * (NS == 2 ? (i & 1) : 0);
      const uint32_t s_par = NS == 2 ? (i >> 1) & 1u : i & 1u;
      const float* nl_s = stat_gen + (i & 1) * 2 * BT + 64 * half;
      if (KV) {
        // the statistics came by bulk copy on this barrier (long complete when S is)
        ok = mbar_wait(sm.bar_xfull + 8 * (i & 1), (i >> 1) & 1u, abort_flag, p.status, DEV_TIMEOUT_SOFTMAX, p.spin);
        if (!ok) break;
      }
      ok = mbar_wait(s_bar, s_par, abort_flag, p.status, DEV_TIMEOUT_SOFTMAX, p.spin);
      if (!ok) break;
      tc_fence_after();
      float2 pv[32];
      {
        uint32_t sr[2][32];
        tmem_ld_32x32(s_addr, sr[0]);
        tmem_ld_32x32(s_addr + 32, sr[1]);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float4 l4 = make_float4(nl, nl, nl, nl);
          if (KV) l4 = *reinterpret_cast<const float4*>(nl_s + 2 * k);
          const uint32_t* f = &sr[k >> 4][2 * (k & 15)];
          pv[k] = exp2_share(k, fma2(make_float2(__uint_as_float(f[0]), __uint_as_float(f[1])), make_float2(c, c), make_float2(l4.x, l4.y)));
          pv[k + 1] = exp2_share(k + 1, fma2(make_float2(__uint_as_float(f[2]), __uint_as_float(f[3])), make_float2(c, c), make_float2(l4.z, l4.w)));
        }
      }
      if (mask) {
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          if (2 * k < lo || 2 * k >= hi) pv[k].x = 0.f;
          if (2 * k + 1 < lo || 2 * k + 1 >= hi) pv[k].y = 0.f;
        }
      }
      if (KV) {
        store_a_half(s_addr, pv);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(sm.bar_pfull);
      }
      ok = mbar_wait(sm.bar_dpfull, i & 1u, abort_flag, p.status, DEV_TIMEOUT_PV, p.spin);
      if (!ok) break;
      tc_fence_after();
      {
        uint32_t dr[2][32];
        tmem_ld_32x32(t_col + TM_DP, dr[0]);
        tmem_ld_32x32(t_col + TM_DP + 32, dr[1]);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float4 d4 = make_float4(nd, nd, nd, nd);
          if (KV) d4 = *reinterpret_cast<const float4*>(nl_s + BT + 2 * k);
          const uint32_t* f = &dr[k >> 4][2 * (k & 15)];
          pv[k] = mul2(pv[k], add2(make_float2(__uint_as_float(f[0]), __uint_as_float(f[1])), make_float2(d4.x, d4.y)));
          pv[k + 1] = mul2(pv[k + 1], add2(make_float2(__uint_as_float(f[2]), __uint_as_float(f[3])), make_float2(d4.z, d4.w)));
        }
      }
      store_a_half(t_col + TM_DP, pv);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(sm.bar_dsfull);
    }
    if (ok && n_it > 0) {
      ok = mbar_wait(sm.bar_done, 0, abort_flag, p.status, DEV_TIMEOUT_EPILOGUE, p.spin);
      tc_fence_after();
    }
    // columns (D / 2) * half .. of the accumulators -> global, bf16; nothing visible: zeros
    const int rows = KV ? p.Skv : p.Sq;
    auto drain = [&](uint32_t acc, float f, void* out, size_t off, unsigned long long extent) {
#pragma unroll
      for (int c0 = 0; c0 < D / 2; c0 += 32) {
        uint32_t v[32];
        if (n_it > 0) {
          tmem_ld_32x32(tmem_base + t_lane + acc + (D / 2) * half + c0, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = 0u;
        }
        const size_t at = off + (D / 2) * half + c0;
        if (row < rows && bounds_ok(at * 2, 64, extent, p.status, p.bounds_detail)) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            auto f2 = [&](int e) { return pack_bf16x2(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f); };
            dst[k] = make_uint4(f2(8 * k), f2(8 * k + 2), f2(8 * k + 4), f2(8 * k + 6));
          }
        }
      }
    };
    if (ok) {
      if (KV) {
        drain(TM_ACC0, 1.f, p.dV, static_cast<size_t>(b) * p.v_sb + static_cast<size_t>(head) * p.v_sh + static_cast<size_t>(row) * p.v_sr, p.dv_extent);
        drain(TM_ACC1, p.scale, p.dK, static_cast<size_t>(b) * p.k_sb + static_cast<size_t>(head) * p.k_sh + static_cast<size_t>(row) * p.k_sr, p.dk_extent);
      } else {
        drain(TM_ACC1, p.scale, p.dQ, static_cast<size_t>(b) * p.q_sb + static_cast<size_t>(head) * p.q_sh + static_cast<size_t>(row) * p.q_sr, p.dq_extent);
      }
    }
    tc_fence_before();
  }
}

template <int D>
__global__ void __launch_bounds__(BW_THREADS, 1)
fmha_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                const __grid_constant__ BwdParams p) {
  using Cfg = BwdCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - raw);
  constexpr int TILE = Cfg::TILE_BYTES;
  const uint32_t ctrl_u = base + Cfg::SMEM_DATA + 2 * Cfg::STAT_BYTES;
  uint8_t* ctrl = gen + Cfg::SMEM_DATA + 2 * Cfg::STAT_BYTES;
  BwdSmem sm;
  sm.a0 = base;
  sm.a1 = base + TILE;
  sm.x = base + 2 * TILE;
  sm.y = base + 4 * TILE;
  sm.stat = base + Cfg::SMEM_DATA;
  sm.bar_fixed = ctrl_u;
  sm.bar_xfull = ctrl_u + 8;     // [2]
  sm.bar_xempty = ctrl_u + 24;   // [2]
  sm.bar_yfull = ctrl_u + 40;    // [2]
  sm.bar_yempty = ctrl_u + 56;   // [2]
  sm.bar_sfull = ctrl_u + 72;    // [2]
  sm.bar_pfull = ctrl_u + 88;
  sm.bar_dpfull = ctrl_u + 96;
  sm.bar_dsfull = ctrl_u + 104;
  sm.bar_done = ctrl_u + 112;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(ctrl + 128);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 132);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
    mbar_init(sm.bar_fixed, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(sm.bar_xfull + 8 * i, 1);
      mbar_init(sm.bar_xempty + 8 * i, 1);
      mbar_init(sm.bar_yfull + 8 * i, 1);
      mbar_init(sm.bar_yempty + 8 * i, 1);
      mbar_init(sm.bar_sfull + 8 * i, 1);
    }
    mbar_init(sm.bar_pfull, 256);
    mbar_init(sm.bar_dpfull, 1);
    mbar_init(sm.bar_dsfull, 256);
    mbar_init(sm.bar_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const float* stat_gen = reinterpret_cast<const float*>(gen + Cfg::SMEM_DATA);
  const int idx = static_cast<int>(blockIdx.x);
  if (idx < p.kv_items)
    bwd_item<D, true>(&tmK, &tmV, &tmQ, &tmDO, p, idx, sm, stat_gen, tmem_base, abort_flag);
  else
    bwd_item<D, false>(&tmQ, &tmDO, &tmK, &tmV, p, idx - p.kv_items, sm, stat_gen, tmem_base, abort_flag);
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// -lse * log2(e) and -delta of every row, laid out for 128-row tiles: [B * H][sq_pad].  D / 8 lanes
// per row, 16 bytes of O and of dO each; memory-bound (4 D bytes read per row).
struct StatParams {
  const __nv_bfloat16 *O, *dO;
  const float* lse;
  float *nlse, *ndelta;
  long long o_sb, o_sh, o_sr, g_sb, g_sh, g_sr;
  int H, Sq, sq_pad;
  long long rows;         // B * H * sq_pad
};

template <int D>
__global__ void __launch_bounds__(256) fmha_bwd_stat_kernel(const StatParams p) {
  griddep_launch_dependents();
  constexpr int LPR = D / 8;
  const int sub = threadIdx.x % LPR;
  const long long first = (blockIdx.x * 256ll + threadIdx.x) / LPR;
  const long long step = gridDim.x * 256ll / LPR;
  for (long long at = first; at < p.rows; at += step) {   // the lanes of a row leave together
    const long long bh = at / p.sq_pad;
    const int row = static_cast<int>(at - bh * p.sq_pad);
    const int b = static_cast<int>(bh / p.H), h = static_cast<int>(bh - static_cast<long long>(b) * p.H);
    float sum = 0.f, nl = -INFINITY;
    if (row < p.Sq) {
      const uint4 o = *reinterpret_cast<const uint4*>(p.O + b * p.o_sb + h * p.o_sh + row * p.o_sr + sub * 8);
      const uint4 g = *reinterpret_cast<const uint4*>(p.dO + b * p.g_sb + h * p.g_sh + row * p.g_sr + sub * 8);
      const uint32_t ow[4] = {o.x, o.y, o.z, o.w}, gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum = fmaf(__uint_as_float(ow[i] << 16), __uint_as_float(gw[i] << 16), sum);
        sum = fmaf(__uint_as_float(ow[i] & 0xFFFF0000u), __uint_as_float(gw[i] & 0xFFFF0000u), sum);
      }
      const float l = p.lse[bh * p.Sq + row];
      // a row without a visible key (lse = -inf) gets P = 0 like the rows past the end
      nl = l == -INFINITY ? -INFINITY : -l * 1.4426950408889634f;
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (sub == 0) {
      p.nlse[at] = nl;
      p.ndelta[at] = -sum;
    }
  }
}

inline size_t stat_pad(int Sq) { return (static_cast<size_t>(Sq) + BT - 1) / BT * BT; }

// Heads walked together: enough items for two waves of the SMs, at least 8 heads' worth, what the
// group streams within a third of the L2 (as in the forward kernel), all groups equal up to one head.
void item_groups(int heads, int tiles, long long stream_bytes, int& group, int& small) {
  const long long l2_heads = (40ll << 20) / (stream_bytes > 0 ? stream_bytes : 1);
  long long g = (2ll * device_sm_count() + tiles - 1) / tiles;
  if (g < 8) g = 8;
  if (g > l2_heads) g = l2_heads;
  if (g < 1) g = 1;
  if (g > heads) g = heads;
  const long long n_groups = (heads + g - 1) / g;
  g = (heads + n_groups - 1) / n_groups;
  group = static_cast<int>(g);
  small = static_cast<int>(g * n_groups - heads);
}

template <int D>
kcg_status_t launch_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                        const BwdParams& p, const StatParams& s, long long items, cudaStream_t stream) {
  using Cfg = BwdCfg<D>;
  static_assert(Cfg::SMEM_TOTAL <= 232448, "shared memory budget");
  auto kern = fmha_bwd_kernel<D>;
  static std::atomic<bool> allowed[64];
  const kcg_status_t st = allow_smem(kern, Cfg::SMEM_TOTAL, allowed);
  if (st != KCG_OK) return st;
  const long long want = (s.rows * (D / 8) + 255) / 256, most = 8ll * device_sm_count();
  fmha_bwd_stat_kernel<D><<<static_cast<unsigned>(want < most ? want : most), 256, 0, stream>>>(s);
  g_launches.fetch_add(1);
  KCG_CUDA_TRY(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(items));
  cfg.blockDim = dim3(BW_THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM_TOTAL;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KCG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, tdo, p));
  g_launches.fetch_add(1);
  return KCG_OK;
}

}  // namespace

size_t fmha_bwd_workspace_impl(const kcg_attn_desc* d) {
  if (attn_check_desc(d) != KCG_OK) return 0;
  return 2 * static_cast<size_t>(d->B) * d->H * stat_pad(d->Sq) * sizeof(float);
}

kcg_status_t fmha_bwd_launch_impl(const kcg_attn_desc* d, const void* dO, const void* Q, const void* K, const void* V,
                                  const void* O, const float* lse, void* dQ, void* dK, void* dV, void* ws,
                                  size_t ws_bytes, cudaStream_t stream) {
  kcg_status_t st = attn_check_desc(d);
  if (st != KCG_OK) return st;
  if (!dO || !Q || !K || !V || !O || !lse || !dQ || !dK || !dV) return KCG_BAD_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return KCG_BAD_ALIGN;
  auto view = [&](const void* x, int heads, int S, const int64_t* s) { return HeadView{x, d->B, heads, S, d->D, s[0], s[1], s[2]}; };
  const HeadView vq = view(Q, d->H, d->Sq, d->q), vk = view(K, d->Hkv, d->Skv, d->k), vv = view(V, d->Hkv, d->Skv, d->v),
                 vo = view(O, d->H, d->Sq, d->o), vdo = view(dO, d->H, d->Sq, d->d_o), vdq = view(dQ, d->H, d->Sq, d->d_q),
                 vdk = view(dK, d->Hkv, d->Skv, d->d_k), vdv = view(dV, d->Hkv, d->Skv, d->d_v);
  for (const HeadView* v : {&vq, &vk, &vv, &vo, &vdo, &vdq, &vdk, &vdv})
    if ((st = check_head_view(*v, 2)) != KCG_OK) return st;
  const size_t sq_pad = stat_pad(d->Sq), stat_rows = static_cast<size_t>(d->B) * d->H * sq_pad;
  if (!ws || ws_bytes < 2 * stat_rows * sizeof(float) || !aligned16(ws)) return KCG_BAD_WORKSPACE;
  BwdParams p;
  p.n_qt = static_cast<int>(sq_pad / BT);
  p.n_kt = static_cast<int>((static_cast<long long>(d->Skv) + BT - 1) / BT);
  const long long kv_items = static_cast<long long>(d->B) * d->Hkv * p.n_kt, q_items = static_cast<long long>(d->B) * d->H * p.n_qt;
  if (kv_items + q_items > 0x7FFFFFFFll || static_cast<long long>(d->H / d->Hkv) * p.n_qt > 0x7FFFFFFFll) return KCG_BAD_SHAPE;
  CUtensorMap tq, tk, tv, tdo;
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if ((st = encode_head_view(&tq, dt, 2, vq)) != KCG_OK) return st;
  if ((st = encode_head_view(&tk, dt, 2, vk)) != KCG_OK) return st;
  if ((st = encode_head_view(&tv, dt, 2, vv)) != KCG_OK) return st;
  if ((st = encode_head_view(&tdo, dt, 2, vdo)) != KCG_OK) return st;
  // the stride of an extent of one is never multiplied by anything but zero
  p.dQ = dQ, p.q_sb = d->d_q[0], p.q_sh = d->d_q[1], p.q_sr = d->d_q[2];
  p.dK = dK, p.k_sb = d->d_k[0], p.k_sh = d->d_k[1], p.k_sr = d->d_k[2];
  p.dV = dV, p.v_sb = d->d_v[0], p.v_sh = d->d_v[1], p.v_sr = d->d_v[2];
  StatParams s;
  s.O = static_cast<const __nv_bfloat16*>(O);
  s.dO = static_cast<const __nv_bfloat16*>(dO);
  s.lse = lse;
  s.nlse = static_cast<float*>(ws);
  s.ndelta = s.nlse + stat_rows;
  s.o_sb = d->o[0], s.o_sh = d->o[1], s.o_sr = d->o[2];
  s.g_sb = d->d_o[0], s.g_sh = d->d_o[1], s.g_sr = d->d_o[2];
  s.H = d->H;
  s.Sq = d->Sq;
  s.sq_pad = static_cast<int>(sq_pad);
  s.rows = static_cast<long long>(stat_rows);
  p.nlse = s.nlse;
  p.ndelta = s.ndelta;
  p.H = d->H;
  p.Hkv = d->Hkv;
  p.group = d->H / d->Hkv;
  p.Sq = d->Sq;
  p.Skv = d->Skv;
  p.sq_pad = s.sq_pad;
  p.causal = d->causal ? 1 : 0;
  p.scale = d->scale;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.kv_items = static_cast<int>(kv_items);
  item_groups(d->B * d->Hkv, p.n_kt, 4ll * p.group * d->Sq * d->D, p.kv_group, p.kv_small);
  item_groups(d->B * d->H, p.n_qt, 4ll * d->Skv * d->D / p.group, p.q_group, p.q_small);
  p.dq_extent = head_view_extent(vdq, 2);
  p.dk_extent = head_view_extent(vdk, 2);
  p.dv_extent = head_view_extent(vdv, 2);
  if (const unsigned long long cap = debug_extent_limit())
    for (unsigned long long* e : {&p.dq_extent, &p.dk_extent, &p.dv_extent}) *e = *e < cap ? *e : cap;
  p.bounds_detail = nullptr;
  debug_bounds_detail_ptr(&p.bounds_detail);
  if ((st = device_status_ptr(&p.status)) != KCG_OK) return st;
  const uint32_t spin = g_spin_limit.load();
  p.spin = spin ? spin : KCG_SPIN_LIMIT;
  const long long items = kv_items + q_items;
  if (d->D == 64) return launch_bwd<64>(tq, tk, tv, tdo, p, s, items, stream);
  return launch_bwd<128>(tq, tk, tv, tdo, p, s, items, stream);
}

}  // namespace kcg
