// Gradients of O = softmax(scale * Q.K^T [causal]) . V on sm_100a.
//
//   P_ij  = exp(scale q_i.k_j - lse_i)            recomputed from the forward pass's lse, never stored
//   delta_i = dO_i.O_i,  dS_ij = P_ij (dO_i.v_j - delta_i)
//   dV_j = sum_i P_ij dO_i    dK_j = scale sum_i dS_ij q_i    dQ_i = scale sum_j dS_ij k_j
//
// dK and dV sum over queries, dQ over keys.  One sweep for all three needs dQ added up across CTAs in a 32-bit buffer
// (64 KB of L2 traffic per 128 x 128 tile at D = 128, as much as the tile's four operands), by atomics whose order, and so
// whose rounding, differs from run to run, or in turns that CTAs wait for.  Here a launch holds
// two kinds of work item instead, each of which owns what it writes:
//
//   kv item  128 keys of one key/value head; streams the query tiles of all its query heads:
//            S^T = K.Q^T, dP^T = V.dO^T, dV += P^T.dO, dK += dS^T.Q           (4 products a tile)
//   q item   128 queries of one query head; streams the key tiles:
//            S = Q.K^T, dP = dO.V^T, dQ += dS.K                               (3 products a tile)
//
// 7 products instead of 5, no atomics, no 32-bit gradient in memory, the same bits on every call.  Where
// the items are too few to fill the SMs (few heads that many query heads share, short batches) an item is
// cut along its stream; the pieces' sums go to the workspace in fp32 and a small kernel adds them up in
// order.
//
// In both, P and dS are computed with the row of the ACCUMULATOR (one TMEM lane) in one thread's
// registers, written back to TMEM as bf16 and used from there as the A operand of the accumulating
// products: nothing passes through shared memory but the TMA tiles, whose K-major form feeds S and dP and
// whose MN-major reading of the same bytes feeds dV, dK, dQ.
//
//   warp 0       TMA producer: two fixed tiles, then two streams (X, Y) through rings
//   warp 1       UMMA issuer of S and dV
//   warp 2       UMMA issuer of dP and dK (dQ): an issuer is held up until the tensor core has all but about
//                four of its instructions behind it, so one warp's waits would leave gaps between products
//   warps 4..11  P and dS: thread = accumulator row and one half of the tile's columns
//
//             fixed A0, A1    stream X, Y    S = A0.X^T   dP = A1.Y^T   acc1 += dS.X   acc0 += P.Y
//   kv item   K, V            Q, dO          S^T          dP^T          dK             dV
//   q item    Q, dO           K, V           S            dP            dQ             -
//
// What sets the rest is latency: eight instructions of 128 x 128 x 16 take 512 clocks and 350 more until
// their barrier completes, a wait 80 even when the barrier has long completed, the exponentials of a
// 128 x 128 tile 640 at the least.  D = 64 leaves room for two CTAs per SM (streamed tiles of 64 rows, half
// of TMEM each), and each computes while the other waits.  At D = 128 one CTA has the SM: a q item gives
// S and dP back as soon as they are in registers and has two buffers for dS, so that S(i+1) and dP(i+1)
// run under the softmax of tile i; a kv item, whose four 128 x 128 fp32 buffers fill TMEM, holds P over S
// and dS over dP and hands P over in two halves, so that dV of the first runs under the exponentials of
// the second.  TMEM columns (BN = rows of a streamed tile: 128, or 64 at D = 64):
//
//   kv    S / P: BN    dP / dS: BN    dV: D    dK: D
//   q     S: BN        dP: BN         dQ: D    dS: 2 x BN / 2
//
// Measured (B200, bf16, causal, D = 128): 32 heads x 8192 1482 us, 927 TFLOP/s of 5 products (1298 of the 7 that
// run) in short bursts, 1700 to 1750 us in calls back to back for seconds, where the power limit holds cuBLAS's own
// bf16 products to 1384 TFLOP/s; 16 heads x 4096 209 us.  One issuer instead of two: 1615 and 228 us.
// D = 64, 2 x 32 heads x 4096 causal: 780 us, 440 TFLOP/s; one CTA per SM with 128-row tiles measures the same
// within the noise of the clocks.
#include "common.cuh"
#include "ptx.cuh"

namespace kcg {

namespace {

constexpr int BT = 128;          // rows of a work item
constexpr int SW = 8;            // softmax warps: two per TMEM lane quarter
constexpr int BW_THREADS = 128 + 32 * SW;

struct BwdParams {
  void *dQ, *dK, *dV;
  long long q_sb, q_sh, q_sr, k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;   // strides of the gradients, elements
  const float* nlse;      // [B * H][sq_pad] -lse * log2(e); -inf for rows without a visible key and past Sq
  const float* ndelta;    // [B * H][sq_pad] -delta; 0 past Sq
  int H, Hkv, group;
  int Sq, Skv, sq_pad;
  int causal;
  float scale, scale_log2;
  int n_qt, n_kt;         // items per head: 128-row tiles of queries, of keys
  int kv_items;           // B * Hkv * n_kt
  int kv_group, kv_small; // order of the items, see item_of()
  int q_group, q_small;
  int kv_split, q_split;  // pieces of every item; CTAs: kv_items * kv_split, then the q items' pieces
  float *part_q, *part_k, *part_v;   // [piece][batch * heads * tiles][D / 4][128 rows] of four columns, where there is more than one piece
  int bh, bhkv;           // batch * heads
  int* status;
  uint32_t spin;
  unsigned long long dq_extent, dk_extent, dv_extent;   // bounds-checking build
  unsigned long long stat_extent, part_q_extent, part_kv_extent;
  unsigned long long* bounds_detail;
};

template <int D>
struct BwdCfg {
  static constexpr int CTAS = D == 128 ? 1 : 2;       // that share an SM
  static constexpr int BN = D == 128 ? 128 : 64;      // rows of a streamed tile, and of every TMA copy
  static constexpr int CPT = BN / 2;                  // columns of a tile that a softmax thread has
  static constexpr int FIXED_BYTES = BT * D * 2;      // A0, A1
  static constexpr int STREAM_BYTES = BN * D * 2;
  static constexpr int FIXED_PANEL = BT * 128, STREAM_PANEL = BN * 128;   // 64 columns of every row
  static constexpr int DPANELS = D / 64;
  static constexpr int STAT_BYTES = 2 * BN * 4;       // -lse and -delta of the rows of a query tile
  // X is read by the first product of a tile and by the last: its next-but-one tile has to be on its way
  // before that last product is done
  static constexpr int NX = 3, NY = D == 128 ? 2 : 3;
  static constexpr int SMEM_DATA = 2 * FIXED_BYTES + (NX + NY) * STREAM_BYTES;
  static constexpr int SMEM_TOTAL = SMEM_DATA + 2 * STAT_BYTES + 256 /*ctrl*/;
  static constexpr int TMEM_COLS = 512 / CTAS;
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

// What a CTA works on: rows row0.. of head `head` of batch b; the tiles it streams are it0.. of the first..
// first + n_tiles - 1 of each of the heads from h0 on, n of them.
struct BwdItem {
  int head, b, row0, first, n_tiles, h0, it0, n, piece;
};

template <int D, bool KV>
__device__ __forceinline__ BwdItem item_at(const BwdParams& p, int idx) {
  constexpr int BN = BwdCfg<D>::BN;
  const int split = KV ? p.kv_split : p.q_split;
  const int shift = p.Skv - p.Sq;    // causal: query i sees keys j <= i + shift
  BwdItem w;
  w.piece = idx % split;
  idx /= split;
  int tile, n_heads;
  w.first = 0;
  if (KV) {
    item_of(idx, p.n_kt, p.kv_group, p.kv_small, w.head, tile);   // causal: key tile 0 is the longest
    w.b = w.head / p.Hkv;
    w.head -= w.b * p.Hkv;
    w.row0 = tile * BT;
    if (p.causal) {
      const int q_min = w.row0 - shift;                           // the first query that sees a key of the tile
      w.first = q_min > 0 ? q_min / BN : 0;
    }
    const int all = (p.Sq + BN - 1) / BN;
    w.n_tiles = all > w.first ? all - w.first : 0;
    w.h0 = w.head * p.group;
    n_heads = p.group;
  } else {
    item_of(idx, p.n_qt, p.q_group, p.q_small, w.head, tile);
    w.b = w.head / p.H;
    w.head -= w.b * p.H;
    if (p.causal) tile = p.n_qt - 1 - tile;
    w.row0 = tile * BT;
    int end = p.Skv;
    if (p.causal) {
      const int lim = w.row0 + BT + shift;
      end = lim < end ? lim : end;
      if (end < 0) end = 0;
    }
    w.n_tiles = (end + BN - 1) / BN;
    w.h0 = w.head / p.group;
    n_heads = 1;
  }
  const int all = w.n_tiles * n_heads, per = (all + split - 1) / split;
  w.it0 = w.piece * per;
  w.n = all - w.it0 < per ? all - w.it0 : per;
  if (w.n < 0) w.n = 0;
  return w;
}

// 2^x of pair k of a row: a share of the pairs (a fixed pattern, so that the two kinds of instruction
// interleave) takes the FMA-pipe polynomial, the rest the MUFU unit, which alone would need 1024 clocks
// for a 128 x 128 tile, as long as two of the tile's products.  (2/8 and 4/8 measure the same within 1 %.)
constexpr int POLY_EIGHTHS = 3;
__device__ __forceinline__ float2 exp2_share(int k, float2 x) {
  if (((k * 5) & 7) < POLY_EIGHTHS) {
    // the polynomial's lower end: such a P is 2^-125, nothing in any sum.  A NaN stays one, comes out as the
    // largest number and is infinite in bf16; O of such a row is NaN, so its delta is, and every dS.  (2^n as a
    // factor, which would keep the NaN in P itself, costs 1 to 4 %: 97.4 -> 101.8 us at 4 x 16 x 1024 x 64.)
    x.x = fmax_nan(x.x, -125.f);
    x.y = fmax_nan(x.y, -125.f);
    return ex2_quartic2(x);
  }
  x.x = ex2_approx(x.x);
  x.y = ex2_approx(x.y);
  return x;
}

// 32 columns of a row as bf16 in TMEM: the A operand's form, two elements per column.
__device__ __forceinline__ void store_a(uint32_t taddr, const float2* v) {
  uint32_t pk[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(v[i].x, v[i].y);
  tmem_st_32x16(taddr, pk);
}

// Where 16-byte chunk `chunk` of row r of a 128 x D bf16 tile is put for the output: rows in a row, the
// chunks exchanged so that both a column of chunks and a row meet all banks.
template <int D>
__device__ __forceinline__ uint32_t out_chunk(uint32_t tile, int r, int chunk) {
  return tile + r * (2 * D) + ((chunk ^ (r & 7)) << 4);
}

// Position in a ring of N stages.
template <int N>
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

// One arrival per warp, for what all of its lanes did in TMEM.
__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <int D, bool KV>
__device__ __forceinline__ void run_item(const CUtensorMap* tmA0, const CUtensorMap* tmA1, const CUtensorMap* tmX,
                                         const CUtensorMap* tmY, const BwdParams& p, int idx, uint8_t* smem) {
  using Cfg = BwdCfg<D>;
  constexpr int BN = Cfg::BN, CPT = Cfg::CPT, DPANELS = Cfg::DPANELS, NX = Cfg::NX, NY = Cfg::NY;
  constexpr int HALVES = CPT / 32;       // pieces of 32 columns in which a thread works, and P is handed over
  constexpr uint32_t TM_S = 0, TM_DP = BN, TM_ACC0 = 2 * BN, TM_ACC1 = KV ? TM_ACC0 + D : TM_ACC0;
  constexpr uint32_t TM_P = TM_S, TM_DS = KV ? TM_DP : TM_ACC1 + D;
  static_assert((KV ? TM_ACC1 + D : TM_DS + BN) <= Cfg::TMEM_COLS, "TMEM columns");
  constexpr uint32_t IDESC_S = make_idesc(UMMA_FMT_BF16, BT, BN, 0, 0);
  constexpr uint32_t IDESC_ACC = make_idesc(UMMA_FMT_BF16, BT, D, 0, 1);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int shift = p.Skv - p.Sq;
  const BwdItem w = item_at<D, KV>(p, idx);
  const int n_it = w.n;

  const uint32_t base = smem_u32(smem);
  const uint32_t s_a0 = base, s_a1 = base + Cfg::FIXED_BYTES, s_x = base + 2 * Cfg::FIXED_BYTES,
                 s_y = s_x + NX * Cfg::STREAM_BYTES, s_stat = base + Cfg::SMEM_DATA;
  const float* stat_gen = reinterpret_cast<const float*>(smem + Cfg::SMEM_DATA);
  uint8_t* ctrl = smem + Cfg::SMEM_DATA + 2 * Cfg::STAT_BYTES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(ctrl + 224);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 228);
  // barriers, with the arrivals that complete a phase; X, Y and the statistics have one per stage
  uint32_t bar_at = smem_u32(ctrl);
  auto bars = [&](int n, uint32_t count) {
    const uint32_t b = bar_at;
    bar_at += 8 * n;
    if (threadIdx.x == 0)
      for (int i = 0; i < n; ++i) mbar_init(b + 8 * i, count);
    return b;
  };
  const uint32_t b_fixed = bars(1, 1), b_xfull = bars(NX, 1), b_xempty = bars(NX, 1), b_yfull = bars(NY, 1);
  const uint32_t b_yempty = bars(NY, KV ? 2 : 1);                    // dP, and dV in a kv item
  const uint32_t b_tfull = bars(2, 1), b_tempty = bars(2, SW);
  const uint32_t b_sfull = bars(1, 1), b_sread = bars(1, SW), b_pfull = bars(2, SW), b_dpfull = bars(1, 1);
  const uint32_t b_dpread = bars(1, SW), b_dsfull = bars(2, SW), b_done = bars(1, 2);   // at most 26: 208 bytes

  auto load = [&](uint32_t dst, int panel, const CUtensorMap* map, uint32_t bar, int row, int hd) {
#pragma unroll
    for (int dp = 0; dp < DPANELS; ++dp) tma_load_4d(dst + dp * panel, map, bar, dp * 64, row, hd, w.b);
  };
  // the producer's place in the stream: X runs a tile ahead of Y, since S(i+1) may be issued as soon as S(i)
  // has been read
  struct Place {
    int t, h;
  };
  auto step_place = [&](Place& at) {
    if (++at.t == w.first + w.n_tiles) {
      at.t = w.first;
      ++at.h;
    }
  };
  Place px{0, 0}, py{0, 0};
  Ring<NX> xr;
  Ring<NY> yr;
  auto load_x = [&]() {
    mbar_expect_tx(b_xfull + 8 * xr.stage, Cfg::STREAM_BYTES);
    load(s_x + xr.stage * Cfg::STREAM_BYTES, Cfg::STREAM_PANEL, tmX, b_xfull + 8 * xr.stage, px.t * BN, px.h);
    xr.next();
    step_place(px);
  };
  auto load_y = [&]() {
    mbar_expect_tx(b_yfull + 8 * yr.stage, Cfg::STREAM_BYTES);
    load(s_y + yr.stage * Cfg::STREAM_BYTES, Cfg::STREAM_PANEL, tmY, b_yfull + 8 * yr.stage, py.t * BN, py.h);
    yr.next();
  };
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_fence_init();
    if (n_it > 0) {
      // the first tiles are in flight while TMEM is allocated and the CTA synchronises
      px.t = w.first + w.it0 % w.n_tiles;
      px.h = w.h0 + w.it0 / w.n_tiles;
      py = px;
      mbar_expect_tx(b_fixed, 2 * Cfg::FIXED_BYTES);
#pragma unroll
      for (int r0 = 0; r0 < BT; r0 += BN) load(s_a0 + r0 * 128, Cfg::FIXED_PANEL, tmA0, b_fixed, w.row0 + r0, w.head);
      load_x();
#pragma unroll
      for (int r0 = 0; r0 < BT; r0 += BN) load(s_a1 + r0 * 128, Cfg::FIXED_PANEL, tmA1, b_fixed, w.row0 + r0, w.head);
      load_y();
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  if (warp == 0) {
    if (lane == 0 && n_it > 0) {
      // ------------------------------- TMA producer -------------------------------------------
      auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        return mbar_wait(bar, parity, abort_flag, p.status, DEV_TIMEOUT_PRODUCER, p.spin);
      };
      bool ok = true;
      Ring<2> tr;
      for (int i = 0; i < n_it; ++i) {
        if (i > 0) {
          if (!(ok = wait(b_yempty + 8 * yr.stage, yr.phase ^ 1u))) break;
          load_y();
        }
        if (KV) {
          if (!(ok = wait(b_tempty + 8 * tr.stage, tr.phase ^ 1u))) break;
          // written by the launch before this one; the tiles are not
          if (i == 0) griddep_wait();
          const size_t at = (static_cast<size_t>(w.b) * p.H + py.h) * p.sq_pad + static_cast<size_t>(py.t) * BN;
          const uint32_t bar = b_tfull + 8 * tr.stage, to = s_stat + tr.stage * Cfg::STAT_BYTES;
          const bool inside = bounds_ok(at * 4, BN * 4, p.stat_extent, p.status, p.bounds_detail);
          mbar_expect_tx(bar, inside ? Cfg::STAT_BYTES : 0);
          if (inside) {
            bulk_load(to, p.nlse + at, BN * 4, bar);
            bulk_load(to + BN * 4, p.ndelta + at, BN * 4, bar);
          }
          tr.next();
        }
        step_place(py);
        if (i + 1 < n_it) {
          if (!(ok = wait(b_xempty + 8 * xr.stage, xr.phase ^ 1u))) break;
          load_x();
        }
      }
      if (!ok) {
        // Copies in flight land before shared memory is released: a wait, bounded, that long outlasts them
        // (which stages were armed last is of no use: their barriers may have moved on).
        for (int k = 0; k < 64; ++k) __nanosleep(2000);
      }
    }
  } else if (warp <= 2) {
    if (n_it > 0) {
      // ------------------------------- UMMA issuers -------------------------------------------
      // The whole warp walks the loop, one elected lane issues.  A wait that gives up leaves `ok` false and
      // the walk goes on (every later wait gives up soon): what is issued then is garbage that nothing
      // stores, and no lane leaves the others.
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        ok = mbar_wait(bar, parity, abort_flag, p.status, code, p.spin) && ok;
        __syncwarp();
        tc_fence_after();
      };
      constexpr uint32_t STAGE = Cfg::STREAM_BYTES >> 4;   // in units of a descriptor's address
      // 128 x BN = A . B^T over the head dimension, both K-major in shared memory (rows of 128 bytes along it)
      auto product = [&](uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          umma_bf16_ss_lo(d_tmem, a_lo + (((ks >> 2) * Cfg::FIXED_PANEL + (ks & 3) * 32) >> 4),
                          b_lo + (((ks >> 2) * Cfg::STREAM_PANEL + (ks & 3) * 32) >> 4), IDESC_S, ks ? 1u : 0u);
      };
      // step ks of acc += A . B over the tile's rows, 16 of them: A in TMEM, B MN-major (the same bytes, a
      // panel's 64 columns to the next)
      auto step = [&](uint32_t acc, uint32_t a_tmem, uint32_t b_lo, int ks, bool add) {
        umma_bf16_ts_lo(acc, a_tmem, b_lo + ((ks * 16 * 128) >> 4), IDESC_ACC, add ? 1u : 0u);
      };
      // where the A operand of step ks is: over S or dP each half of the columns is packed into its own
      // first half, a buffer of its own is packed all in a row
      auto over = [](int ks) { return static_cast<uint32_t>(CPT * (16 * ks / CPT) + (16 * ks % CPT) / 2); };
      wait(b_fixed, 0, DEV_TIMEOUT_Q);
      if (warp == 1) {
        const uint32_t a_lo = smem_desc_lo(s_a0, 16), x_lo = smem_desc_lo(s_x, 16), y_lo = smem_desc_lo(s_y, Cfg::STREAM_PANEL);
        Ring<NX> xk;
        Ring<NY> yt;
        auto wait_x = [&]() { wait(b_xfull + 8 * xk.stage, xk.phase, DEV_TIMEOUT_MMA_FULL); };
        auto issue_s = [&]() {
          if (elect_one()) {
            product(tmem_base + TM_S, a_lo, x_lo + xk.stage * STAGE);
            umma_commit(b_sfull);
          }
          __syncwarp();
          xk.next();
        };
        wait_x();
        issue_s();
        for (int i = 0; i < n_it; ++i) {
          const bool next = i + 1 < n_it;
          const uint32_t par = i & 1u;
          if (next) wait_x();
          if (!KV && next) {
            wait(b_sread, par, DEV_TIMEOUT_P);
            issue_s();
          }
          if (KV) {
            wait(b_yfull + 8 * yt.stage, yt.phase, DEV_TIMEOUT_MMA_FULL);
#pragma unroll
            for (int g = 0; g < HALVES; ++g) {
              wait(b_pfull + 8 * g, par, DEV_TIMEOUT_P);
              if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < BN / 16; ++ks)
                  if ((16 * ks % CPT) / 32 == g) step(tmem_base + TM_ACC0, tmem_base + TM_P + over(ks), y_lo + yt.stage * STAGE, ks, i | ks);
                if (g == HALVES - 1) umma_commit(b_yempty + 8 * yt.stage);
              }
              __syncwarp();
            }
            yt.next();
            if (next) issue_s();
          }
        }
      } else {
        const uint32_t a_lo = smem_desc_lo(s_a1, 16), y_lo = smem_desc_lo(s_y, 16), x_lo = smem_desc_lo(s_x, Cfg::STREAM_PANEL);
        Ring<NY> yk;
        Ring<NX> xt;
        auto wait_y = [&]() { wait(b_yfull + 8 * yk.stage, yk.phase, DEV_TIMEOUT_MMA_FULL); };
        auto issue_dp = [&]() {
          if (elect_one()) {
            product(tmem_base + TM_DP, a_lo, y_lo + yk.stage * STAGE);
            umma_commit(b_dpfull);
            umma_commit(b_yempty + 8 * yk.stage);
          }
          __syncwarp();
          yk.next();
        };
        wait_y();
        issue_dp();
        for (int i = 0; i < n_it; ++i) {
          const bool next = i + 1 < n_it;
          if (next) wait_y();
          if (!KV && next) {
            wait(b_dpread, i & 1u, DEV_TIMEOUT_P);
            issue_dp();
          }
          wait(b_xfull + 8 * xt.stage, xt.phase, DEV_TIMEOUT_MMA_FULL);
          if (KV) wait(b_dsfull, i & 1u, DEV_TIMEOUT_P);
          else wait(b_dsfull + 8 * (i & 1), (i >> 1) & 1u, DEV_TIMEOUT_P);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)
              step(tmem_base + TM_ACC1, tmem_base + TM_DS + (KV ? over(ks) : BN / 2 * (i & 1) + 8 * ks), x_lo + xt.stage * STAGE, ks, i | ks);
            umma_commit(b_xempty + 8 * xt.stage);     // (S of the tile is complete: dS came from it)
          }
          __syncwarp();
          xt.next();
          if (KV && next) issue_dp();
        }
      }
      if (elect_one()) umma_commit(b_done);
      __syncwarp();
      if (!ok) {
        // products in flight finish before TMEM is freed
        for (uint32_t it = 0; it < 65536u; ++it)
          if (mbar_try_wait(b_done, 0)) break;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------- P and dS, then the output ----------------------------------
    const int half = (warp >> 2) - 1;          // columns CPT * half .. of every tile
    const int q = warp & 3;                    // TMEM lane quarter this warp may access
    const int r = q * 32 + lane;               // row inside the item
    const int row = w.row0 + r;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t t_col = t_lane + CPT * half;
    // A wait that gives up leaves `ok` false and the walk goes on, as in the issuers: the accesses to TMEM
    // are collective, so no lane may leave the others.
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
      ok = mbar_wait(bar, parity, abort_flag, p.status, code, p.spin) && ok;
      __syncwarp();
    };
    const float c = p.scale_log2;
    float nl = 0.f, nd = 0.f;
    if (!KV && n_it > 0) {
      griddep_wait();
      const size_t at = (static_cast<size_t>(w.b) * p.H + w.head) * p.sq_pad + row;   // row < sq_pad
      if (bounds_ok(at * 4, 4, p.stat_extent, p.status, p.bounds_detail)) {
        nl = p.nlse[at];
        nd = p.ndelta[at];
      }
    }
    int t = n_it > 0 ? w.it0 % w.n_tiles : 0;
    for (int i = 0; i < n_it; ++i) {
      const uint32_t par = i & 1u;
      // visible columns of this thread's: [lo, hi)
      int lo = 0, hi = CPT;
      bool mask;
      const int at0 = (w.first + t) * BN;      // the tile's first query, or key
      if (++t == w.n_tiles) t = 0;
      if (KV) {
        mask = p.causal && w.row0 + BT - 1 > at0 + shift;
        lo = row - shift - at0 - CPT * half;   // query >= key - shift
      } else {
        int limit = p.Skv;
        if (p.causal) {
          const int l2 = row + shift + 1;
          limit = l2 < limit ? l2 : limit;
        }
        mask = at0 + BN > p.Skv || (p.causal && at0 + BN > w.row0 + shift + 1);
        hi = limit - at0 - CPT * half;
      }
      const float4* stat = reinterpret_cast<const float4*>(stat_gen + (i & 1) * 2 * BN + CPT * half);
      if (KV) wait(b_tfull + 8 * (i & 1), (i >> 1) & 1u, DEV_TIMEOUT_SOFTMAX);
      wait(b_sfull, par, DEV_TIMEOUT_SOFTMAX);
      tc_fence_after();
      float2 pv[CPT / 2];
      {
        uint32_t sr[HALVES][32];
#pragma unroll
        for (int g = 0; g < HALVES; ++g) tmem_ld_32x32(t_col + TM_S + 32 * g, sr[g]);
        tmem_ld_wait();
        if (!KV) warp_arrive(b_sread, lane);
#pragma unroll
        for (int g = 0; g < HALVES; ++g) {
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const float4 l4 = KV ? stat[8 * g + k / 2] : make_float4(nl, nl, nl, nl);
            const uint32_t* f = &sr[g][2 * k];
            pv[16 * g + k] = exp2_share(16 * g + k, fma2(make_float2(__uint_as_float(f[0]), __uint_as_float(f[1])), make_float2(c, c), make_float2(l4.x, l4.y)));
            pv[16 * g + k + 1] = exp2_share(16 * g + k + 1, fma2(make_float2(__uint_as_float(f[2]), __uint_as_float(f[3])), make_float2(c, c), make_float2(l4.z, l4.w)));
          }
          if (mask) {
#pragma unroll
            for (int k = 16 * g; k < 16 * g + 16; ++k) {
              if (2 * k < lo || 2 * k >= hi) pv[k].x = 0.f;
              if (2 * k + 1 < lo || 2 * k + 1 >= hi) pv[k].y = 0.f;
            }
          }
          if (KV) {
            store_a(t_col + TM_P + 16 * g, pv + 16 * g);
            tmem_st_wait();
            warp_arrive(b_pfull + 8 * g, lane);
          }
        }
      }
      // (in a q item dP(i) was issued after the product of dS(i-2), whose buffer dS(i) takes)
      wait(b_dpfull, par, DEV_TIMEOUT_PV);
      tc_fence_after();
      {
        uint32_t dr[HALVES][32];
#pragma unroll
        for (int g = 0; g < HALVES; ++g) tmem_ld_32x32(t_col + TM_DP + 32 * g, dr[g]);
        tmem_ld_wait();
        if (!KV) warp_arrive(b_dpread, lane);
#pragma unroll
        for (int g = 0; g < HALVES; ++g)
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const float4 d4 = KV ? stat[BN / 4 + 8 * g + k / 2] : make_float4(nd, nd, nd, nd);
            const uint32_t* f = &dr[g][2 * k];
            pv[16 * g + k] = mul2(pv[16 * g + k], add2(make_float2(__uint_as_float(f[0]), __uint_as_float(f[1])), make_float2(d4.x, d4.y)));
            pv[16 * g + k + 1] = mul2(pv[16 * g + k + 1], add2(make_float2(__uint_as_float(f[2]), __uint_as_float(f[3])), make_float2(d4.z, d4.w)));
          }
      }
      const uint32_t to = KV ? t_col + TM_DS : t_lane + TM_DS + BN / 2 * par + CPT / 2 * half;
#pragma unroll
      for (int g = 0; g < HALVES; ++g) store_a(to + 16 * g, pv + 16 * g);
      tmem_st_wait();
      warp_arrive(b_dsfull + (KV ? 0 : 8 * par), lane);
      if (KV && lane == 0) mbar_arrive(b_tempty + 8 * (i & 1));   // (the warp's reads are above its __syncwarp)
    }
    if (n_it > 0) {
      wait(b_done, 0, DEV_TIMEOUT_EPILOGUE);
      tc_fence_after();
    }
    // The accumulators, 32 columns at a time.  Nothing visible: zeros.
    const bool whole = (KV ? p.kv_split : p.q_split) == 1;
    constexpr int CHUNKS = (KV ? 2 : 1) * (D / 32);
#pragma unroll
    for (int j0 = 0; j0 < CHUNKS; j0 += 2) {
      const int j = j0 + half;
      const bool is_v = KV && j < D / 32;                      // dV, then dK; or dQ
      const int col = 32 * (KV && !is_v ? j - D / 32 : j);
      uint32_t v[32];
      if (n_it > 0) {
        tmem_ld_32x32(t_lane + (is_v ? TM_ACC0 : TM_ACC1) + col, v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = 0u;
      }
      if (whole) {
        // scaled, rounded, and through shared memory (the tiles have been consumed): a thread's row written
        // from here would be 32 rows to a store instruction
        const float f = is_v ? 1.f : p.scale;
        const uint32_t tile = base + (is_v ? BT * D * 2 : 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          auto f2 = [&](int e) { return pack_bf16x2(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f); };
          st_shared_v4(out_chunk<D>(tile, r, col / 8 + k), make_uint4(f2(8 * k), f2(8 * k + 2), f2(8 * k + 4), f2(8 * k + 6)));
        }
      } else if (ok) {
        // one piece of several goes to the workspace as it is, four columns of 128 rows together
        float* part = KV ? (is_v ? p.part_v : p.part_k) : p.part_q;
        const size_t items = static_cast<size_t>(KV ? p.bhkv : p.bh) * (KV ? p.n_kt : p.n_qt);
        const size_t item = (static_cast<size_t>(w.b) * (KV ? p.Hkv : p.H) + w.head) * (KV ? p.n_kt : p.n_qt) + w.row0 / BT;
        const size_t at = ((w.piece * items + item) * (D / 4) + col / 4) * BT + r;
        float4* dst = reinterpret_cast<float4*>(part) + at;
        if (bounds_ok(at * 16, (7 * BT + 1) * 16, KV ? p.part_kv_extent : p.part_q_extent, p.status, p.bounds_detail))
#pragma unroll
          for (int k = 0; k < 8; ++k)
            dst[k * BT] = make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3]));
      }
    }
    if (whole) {
      asm volatile("bar.sync 1, %0;" ::"n"(32 * SW) : "memory");   // the softmax warps
      constexpr int LPR = D / 8, RPW = 32 / LPR;                     // 16-byte chunks of a row, rows of a warp's store
      const int rows = KV ? p.Skv : p.Sq, chunk = lane % LPR;
#pragma unroll
      for (int m = 0; m < (KV ? 2 : 1); ++m) {                       // dK (dQ), then dV
        void* out = KV ? (m ? p.dV : p.dK) : p.dQ;
        const long long sb = KV ? (m ? p.v_sb : p.k_sb) : p.q_sb, sh = KV ? (m ? p.v_sh : p.k_sh) : p.q_sh,
                        sr = KV ? (m ? p.v_sr : p.k_sr) : p.q_sr;
        const unsigned long long extent = KV ? (m ? p.dv_extent : p.dk_extent) : p.dq_extent;
        const long long at0 = w.b * sb + w.head * sh + 8 * chunk;
#pragma unroll
        for (int k = 0; k < BT / (SW * RPW); ++k) {
          const int rr = (k * SW + warp - 4) * RPW + lane / LPR;
          const uint4 v = ld_shared_v4(out_chunk<D>(base + m * BT * D * 2, rr, chunk));
          const long long at = at0 + (w.row0 + rr) * sr;
          if (ok && w.row0 + rr < rows && bounds_ok(at * 2, 16, extent, p.status, p.bounds_detail))
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at) = v;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

template <int D>
__global__ void __launch_bounds__(BW_THREADS, BwdCfg<D>::CTAS)
fmha_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                const __grid_constant__ BwdParams p) {
  griddep_launch_dependents();   // (the launch that adds pieces up, where there is one)
  // The 128-byte swizzle is a function of address bits: the tiles start on a multiple of 1024, which is
  // where the shared memory of a kernel without static arrays starts (there is no room to round up).
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, static_cast<int>(DEV_BAD_SMEM));
    return;
  }
  const int idx = static_cast<int>(blockIdx.x), kv_ctas = p.kv_items * p.kv_split;
  if (idx < kv_ctas) run_item<D, true>(&tmK, &tmV, &tmQ, &tmDO, p, idx, smem);
  else run_item<D, false>(&tmQ, &tmDO, &tmK, &tmV, p, idx - kv_ctas, smem);
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
  int* status;            // bounds-checking build
  unsigned long long extent;
  unsigned long long* bounds_detail;
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
    if (sub == 0 && bounds_ok(at * 4, 4, p.extent, p.status, p.bounds_detail)) {
      p.nlse[at] = nl;
      p.ndelta[at] = -sum;
    }
  }
}

// Sum of an item's pieces, in order, scaled and rounded: 8 columns a thread.  blockIdx.y: dK, dV (each of
// kv_split pieces) or dQ; a tensor of one piece is complete already.
template <int D>
__global__ void __launch_bounds__(256) fmha_bwd_sum_kernel(const __grid_constant__ BwdParams p) {
  const int which = blockIdx.y;
  const int split = which == 2 ? p.q_split : p.kv_split;
  if (split == 1) return;
  griddep_wait();
  const float* part = which == 2 ? p.part_q : which ? p.part_v : p.part_k;
  void* out = which == 2 ? p.dQ : which ? p.dV : p.dK;
  const long long sb = which == 2 ? p.q_sb : which ? p.v_sb : p.k_sb, sh = which == 2 ? p.q_sh : which ? p.v_sh : p.k_sh,
                  sr = which == 2 ? p.q_sr : which ? p.v_sr : p.k_sr;
  const unsigned long long extent = which == 2 ? p.dq_extent : which ? p.dv_extent : p.dk_extent;
  const unsigned long long part_extent = which == 2 ? p.part_q_extent : p.part_kv_extent;
  const int heads = which == 2 ? p.H : p.Hkv, rows = which == 2 ? p.Sq : p.Skv, tiles = which == 2 ? p.n_qt : p.n_kt;
  const long long items = static_cast<long long>(which == 2 ? p.bh : p.bhkv) * tiles, piece = items * (D / 4) * BT;
  const float f = which == 1 ? 1.f : p.scale;
  const int r = threadIdx.x % BT, sub = threadIdx.x / BT;
  // (item, 8 columns) at a time for every 128 threads
  for (long long i = blockIdx.x * 2ll + sub; i < items * (D / 8); i += gridDim.x * 2ll) {
    const long long item = i / (D / 8);
    const int col = static_cast<int>(i % (D / 8)) * 8, row = static_cast<int>(item % tiles) * BT + r;
    const long long bh = item / tiles;
    const long long first = (item * (D / 4) + col / 4) * BT + r;
    const float4* src = reinterpret_cast<const float4*>(part) + first;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
    for (int s = 0; s < split; ++s) {
      if (!bounds_ok((first + s * piece) * 16, (BT + 1) * 16, part_extent, p.status, p.bounds_detail)) continue;
      const float4 x = src[s * piece], y = src[s * piece + BT];
      a = make_float4(a.x + x.x, a.y + x.y, a.z + x.z, a.w + x.w);
      b = make_float4(b.x + y.x, b.y + y.y, b.z + y.z, b.w + y.w);
    }
    const long long at = (bh / heads) * sb + (bh % heads) * sh + row * sr + col;
    if (row < rows && bounds_ok(at * 2, 16, extent, p.status, p.bounds_detail))
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at) =
          make_uint4(pack_bf16x2(a.x * f, a.y * f), pack_bf16x2(a.z * f, a.w * f), pack_bf16x2(b.x * f, b.y * f), pack_bf16x2(b.z * f, b.w * f));
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

// How the work of a descriptor is cut up, and what that takes of the workspace.
struct BwdPlan {
  long long n_qt, n_kt, kv_items, q_items, kv_split, q_split;
  size_t stat_floats, part_q, part_kv;   // of each of the two statistics; of dQ's pieces; of dK's, of dV's
  size_t bytes() const { return (2 * stat_floats + part_q + 2 * part_kv) * sizeof(float); }
};

// An item is cut where it alone would outlast an equal share of the whole launch on every CTA that the SMs
// hold (costs in products: 4 a tile in a kv item, 3 in a q item), into pieces of such a share, but of about 512
// rows of the longest item's stream (a CTA's start and end take as long as about two 128-row tiles); the count is
// rounded to the nearest, so that 768 rows make two pieces of 384.  All items of a kind are cut alike: under the mask
// the short ones have shorter pieces, down to none, whose CTAs write zeros.  The SM count is the B200's, so that the
// workspace query needs no device.
BwdPlan plan_bwd(const kcg_attn_desc* d) {
  BwdPlan n;
  const long long sq_pad = static_cast<long long>(stat_pad(d->Sq));
  n.n_qt = sq_pad / BT;
  n.n_kt = (static_cast<long long>(d->Skv) + BT - 1) / BT;
  const long long bh = static_cast<long long>(d->B) * d->H, bhkv = static_cast<long long>(d->B) * d->Hkv, group = d->H / d->Hkv;
  n.kv_items = bhkv * n.n_kt;
  n.q_items = bh * n.n_qt;
  const double slots = 148.0 * (d->D == 128 ? 1 : 2);
  const double total = 7.0 * bh * n.n_qt * n.n_kt * (d->causal ? 0.5 : 1.0);
  auto split = [&](double cost, double len) {       // products a tile, tiles of the longest item
    const double share = total / slots > 4 * cost ? total / slots : 4 * cost;
    const long long s = static_cast<long long>(cost * len / share + 0.5);
    return s < 1 ? 1ll : s > 32 ? 32ll : s;
  };
  n.kv_split = split(4, static_cast<double>(group) * n.n_qt);
  n.q_split = split(3, static_cast<double>(n.n_kt));
  n.stat_floats = static_cast<size_t>(bh * sq_pad);
  n.part_q = n.q_split > 1 ? static_cast<size_t>(n.q_split * n.q_items) * BT * d->D : 0;
  n.part_kv = n.kv_split > 1 ? static_cast<size_t>(n.kv_split * n.kv_items) * BT * d->D : 0;
  return n;
}

template <int D>
kcg_status_t launch_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                        const BwdParams& p, const StatParams& s, long long ctas, cudaStream_t stream) {
  using Cfg = BwdCfg<D>;
  static_assert(Cfg::CTAS * Cfg::SMEM_TOTAL <= 232448, "shared memory budget");
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
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(BW_THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM_TOTAL;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KCG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, tdo, p));
  g_launches.fetch_add(1);
  if (p.kv_split > 1 || p.q_split > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>(4 * device_sm_count()), 3);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    KCG_CUDA_TRY(cudaLaunchKernelEx(&cfg, fmha_bwd_sum_kernel<D>, p));
    g_launches.fetch_add(1);
  }
  return KCG_OK;
}

}  // namespace

size_t fmha_bwd_workspace_impl(const kcg_attn_desc* d) {
  return attn_check_desc(d) == KCG_OK ? plan_bwd(d).bytes() : 0;
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
  const BwdPlan n = plan_bwd(d);
  if (!ws || ws_bytes < n.bytes() || !aligned16(ws)) return KCG_BAD_WORKSPACE;
  // an output over an input or another output: it would be written while other CTAs still read it
  const HeadRegion regions[9] = {{vdq, 2}, {vdk, 2}, {vdv, 2}, {vdo, 2}, {vq, 2}, {vk, 2}, {vv, 2}, {vo, 2},
                                 {HeadView{lse, d->B, d->H, d->Sq, 1, static_cast<int64_t>(d->H) * d->Sq, d->Sq, 1}, 4}};
  for (int out = 0; out < 3; ++out)
    for (int i = out + 1; i < 9; ++i)
      if (views_overlap(regions[out], regions[i])) return KCG_BAD_ARGUMENT;
  const long long ctas = n.kv_items * n.kv_split + n.q_items * n.q_split;
  if (ctas > 0x7FFFFFFFll || static_cast<long long>(d->H / d->Hkv) * n.n_qt > 0x3FFFFFFFll) return KCG_BAD_SHAPE;
  CUtensorMap tq, tk, tv, tdo;
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const int box = d->D == 128 ? BwdCfg<128>::BN : BwdCfg<64>::BN;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  if ((st = encode_head_view(&tq, dt, 2, vq, sw, box)) != KCG_OK) return st;
  if ((st = encode_head_view(&tk, dt, 2, vk, sw, box)) != KCG_OK) return st;
  if ((st = encode_head_view(&tv, dt, 2, vv, sw, box)) != KCG_OK) return st;
  if ((st = encode_head_view(&tdo, dt, 2, vdo, sw, box)) != KCG_OK) return st;
  BwdParams p;
  // the stride of an extent of one is never multiplied by anything but zero
  p.dQ = dQ, p.q_sb = d->d_q[0], p.q_sh = d->d_q[1], p.q_sr = d->d_q[2];
  p.dK = dK, p.k_sb = d->d_k[0], p.k_sh = d->d_k[1], p.k_sr = d->d_k[2];
  p.dV = dV, p.v_sb = d->d_v[0], p.v_sh = d->d_v[1], p.v_sr = d->d_v[2];
  StatParams s;
  s.O = static_cast<const __nv_bfloat16*>(O);
  s.dO = static_cast<const __nv_bfloat16*>(dO);
  s.lse = lse;
  s.nlse = static_cast<float*>(ws);
  s.ndelta = s.nlse + n.stat_floats;
  s.o_sb = d->o[0], s.o_sh = d->o[1], s.o_sr = d->o[2];
  s.g_sb = d->d_o[0], s.g_sh = d->d_o[1], s.g_sr = d->d_o[2];
  s.H = d->H;
  s.Sq = d->Sq;
  s.sq_pad = static_cast<int>(stat_pad(d->Sq));
  s.rows = static_cast<long long>(n.stat_floats);
  p.nlse = s.nlse;
  p.ndelta = s.ndelta;
  p.part_q = s.ndelta + n.stat_floats;
  p.part_k = p.part_q + n.part_q;
  p.part_v = p.part_k + n.part_kv;
  p.H = d->H;
  p.Hkv = d->Hkv;
  p.group = d->H / d->Hkv;
  p.bh = d->B * d->H;
  p.bhkv = d->B * d->Hkv;
  p.Sq = d->Sq;
  p.Skv = d->Skv;
  p.sq_pad = s.sq_pad;
  p.causal = d->causal ? 1 : 0;
  p.scale = d->scale;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.n_qt = static_cast<int>(n.n_qt);
  p.n_kt = static_cast<int>(n.n_kt);
  p.kv_items = static_cast<int>(n.kv_items);
  p.kv_split = static_cast<int>(n.kv_split);
  p.q_split = static_cast<int>(n.q_split);
  item_groups(p.bhkv, p.n_kt, 4ll * p.group * d->Sq * d->D, p.kv_group, p.kv_small);
  item_groups(p.bh, p.n_qt, 4ll * d->Skv * d->D / p.group, p.q_group, p.q_small);
  p.dq_extent = head_view_extent(vdq, 2);
  p.dk_extent = head_view_extent(vdk, 2);
  p.dv_extent = head_view_extent(vdv, 2);
  p.stat_extent = n.stat_floats * 4;
  p.part_q_extent = n.part_q * 4;
  p.part_kv_extent = n.part_kv * 4;
  if (const unsigned long long cap = debug_extent_limit())
    for (unsigned long long* e : {&p.dq_extent, &p.dk_extent, &p.dv_extent, &p.stat_extent, &p.part_q_extent, &p.part_kv_extent})
      *e = *e < cap ? *e : cap;
  p.bounds_detail = nullptr;
  debug_bounds_detail_ptr(&p.bounds_detail);
  if ((st = device_status_ptr(&p.status)) != KCG_OK) return st;
  s.status = p.status;
  s.extent = p.stat_extent;
  s.bounds_detail = p.bounds_detail;
  const uint32_t spin = g_spin_limit.load();
  p.spin = spin ? spin : KCG_SPIN_LIMIT;
  if (d->D == 64) return launch_bwd<64>(tq, tk, tv, tdo, p, s, ctas, stream);
  return launch_bwd<128>(tq, tk, tv, tdo, p, s, ctas, stream);
}

}  // namespace kcg
