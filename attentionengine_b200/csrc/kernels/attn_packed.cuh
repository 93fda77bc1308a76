// Fused attention forward over packed sequences of different lengths (prompts), for sm_100a.
//
// The tiles, the roles' steps and the TMEM layout are attn_fwd.cuh's: two row warpgroups (thread = row = TMEM lane), one TMA warp, one MMA
// warp, S0 | S1 | O0 | O1 with P over S, K of the next step and V of this one on one barrier.  What differs:
//
// * A CTA's two q tiles are one 128-row tile of two heads where a kv head's query heads are even in number: both walk the same kv tiles, so a sequence with
//   an odd number of tiles leaves none alone and no tile idles in the last step of a causal pair.  Otherwise they are two neighbouring tiles of a head;
//   and where every tile finds an SM of its own, there is one (args.pair_mode).  Four prompts up to 8192 tokens, 32 heads of 128 dims: 848 us
//   with two tiles of a head, 706 with two heads (single calls in a burst, as first built: 680 now, 800 where calls follow each other under the power cap).
// * The grid is persistent: a CTA takes the next item (a block of query rows, its heads) near the end of one, longest first.  Barriers
//   and TMEM are set up once; a warp of its own finds the item from cu_seqlens, and its first copies and products run under this item's last row
//   work and epilogue.  One item a CTA spent 8000 clk around 4 to 5 steps of 3000 with twelve prompts up to 1500 tokens.
// * The rows behind a sequence's end are another sequence's: their scores do not count (AE_PACK_SCORES says how they are left out), and their values
//   are overwritten with zeros in shared memory before P V (a P of 0 times an infinity is NaN).
//
// Long prompts are bound by the tensor cores at 128 dims (2048 clk of products a step; what is left are the hand-overs), and by the exponentials, as many
// clk, at 64.  Short ones are not: twelve of up to 1500 tokens, 16 heads of 64 dims, take 39 us, of which the 14 steps of the longest CTA are 22; the rest
// lies around the ends of its three or four items, where both row groups write their outputs and the next scores are yet to come.
//
// Expects the forward prelude (AE_D, AE_DV, AE_BF16, AE_STAGES, AE_MASK_MODE 0, 1 or 3, AE_O_SCALE_ONE, AE_PACK_SCORES, AeRow and its functions).

#define AE_BM 128
#define AE_BN 128
#if AE_MASK_MODE == 2
#error "block lists are of one length"
#endif
#define AE_ROW_WARPS 8
#define AE_NTHREADS 384
#define AE_Q_BYTES (AE_BM * AE_D * 2)
#define AE_K_BYTES (AE_BN * AE_D * 2)
#define AE_V_BYTES (AE_BN * AE_DV * 2)
#define AE_SMEM_K (2 * AE_Q_BYTES)
#define AE_SMEM_V (AE_SMEM_K + AE_STAGES * AE_K_BYTES)
#define AE_SMEM_BAR (AE_SMEM_V + AE_STAGES * AE_V_BYTES)
#define AE_SMEM_SEQ (AE_SMEM_BAR + 512)  // blocks of each sequence behind the 32nd
#define AE_MAX_SEQ 4096

struct AePackItem {
  int b, block, start, len;  // b < 0: there are no more
  int hq;                    // of tile 0
};
struct AePackBars {
  u64 q_full[2];
  u64 q_free;               // the item's last S GEMM has read Q
  u64 near_end;             // the item is in its last but one step
  u64 s_full[2];
  u64 o_done[2];
  u64 kv_full[AE_STAGES];   // fill n of an item: V of its step n - 1 and K of step n
  u64 kv_empty[AE_STAGES];
  u64 item_full[2];
  u64 item_empty[2];        // the row warps, the TMA warp and the MMA warp have left it
  AePackItem item[2];
  AeCtaCtl ctl;
};
static_assert(sizeof(AePackBars) <= 512, "room in front of the blocks");
#define AE_PACK_READERS (AE_ROW_WARPS + 2)

// An item as the roles see it.
struct AePackWork {
  int b, hq, qt0, seq0, len, next_qt, next_h;  // tile t: q tile qt0 + t next_qt, head hq + t next_h
  int n0, n1, n_steps;                         // kv tiles of each q tile
  AE_DEVICE int tiles(int t) const { return t ? n1 : n0; }
  AE_DEVICE bool take(const AePackItem& it, const AeAttnFwdArgs& args) {
    b = it.b;
    hq = it.hq;
    seq0 = it.start;
    len = it.len;
    qt0 = args.pair_mode == 0 ? 2 * it.block : it.block;
    next_qt = args.pair_mode == 0 ? 1 : 0;
    next_h = args.pair_mode == 1 ? 1 : 0;
    const int tiles = (len + AE_BN - 1) / AE_BN;
    auto walk = [&](int qt) {
      if (qt >= tiles) return 0;
      return AE_MASK_MODE == 1 ? qt + 1 : tiles;
    };
    n0 = walk(qt0);
    n1 = args.pair_mode == 2 ? 0 : walk(qt0 + next_qt);
    n_steps = n0 > n1 ? n0 : n1;
    return b >= 0;
  }
  // whether some element of a kv tile is masked for q tile t
  AE_DEVICE bool partial(int kt, int t) const {
    return AE_MASK_MODE == 3 || (AE_MASK_MODE == 1 && kt * AE_BN + AE_BN - 1 > (qt0 + t * next_qt) * AE_BM);
  }
};

// The i-th block of `rows` query rows of the packed sequences, by the length of its walk: the last blocks of the longest sequences first.  The
// blocks behind block L of their sequence number S(L) = sum over the sequences of max(0, blocks - 1 - L), so the one that is i-th has the L
// with S(L) <= i < S(L - 1), by bisection.  One warp, a sequence in a lane (more than 32: `more` in shared memory, filled by the first call).
AE_DEVICE void ae_find_block(AePackItem& at, int* more, const AeAttnFwdArgs& args, int i, int rows, bool first) {
  const int lane = (int)lane_id(), n = args.B, T = args.Sq;
  // positions outside the tensors would be a caller's mistake: reported, and cut to them
  auto span = [&](int b, int& start) {
    const int s0 = args.cu_seqlens[b], s1 = args.cu_seqlens[b + 1];
    if ((s0 < 0 || s1 < s0 || s1 > T || (b == 0 && s0 != 0) || (b == n - 1 && s1 != T)) && args.status) atomicOr(args.status, 0x2000u);
    start = s0 < 0 ? 0 : s0 > T ? T : s0;
    const int end = s1 < start ? start : s1 > T ? T : s1;
    return end - start;
  };
  int start = 0, len = 0;
  if (lane < n) len = span(lane, start);
  const int mine = (len + rows - 1) / rows;
  int most = mine;
  for (int b = lane + 32; b < n; b += 32) {
    if (first) {
      int s;
      more[b] = (span(b, s) + rows - 1) / rows;
    }
    most = most > more[b] ? most : more[b];
  }
  most = __reduce_max_sync(0xffffffffu, most);
  __syncwarp();
  auto behind = [&](int L) {
    int s = mine - 1 > L ? mine - 1 - L : 0;
    for (int b = lane + 32; b < n; b += 32) s += more[b] - 1 > L ? more[b] - 1 - L : 0;
    return __reduce_add_sync(0xffffffffu, s);
  };
  if (behind(-1) <= i) {
    if (lane == 0) at.b = -1;
    return;
  }
  int lo = -1, hi = most, at_hi = 0;  // S(lo) > i >= S(hi) = at_hi
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, s = behind(mid);
    if (s > i) {
      lo = mid;
    } else {
      hi = mid;
      at_hi = s;
    }
  }
  int k = i - at_hi;  // the k-th of the sequences that have a block `hi`
  for (int b0 = 0; b0 < n; b0 += 32) {
    const bool has = (b0 == 0 ? mine : b0 + lane < n ? more[b0 + lane] : 0) > hi;
    const u32 m = __ballot_sync(0xffffffffu, has);
    if (has && __popc(m & ((1u << lane) - 1u)) == k) {
      if (b0 > 0) len = span(b0 + lane, start);
      at.b = b0 + lane;
      at.block = hi;
      at.start = start;
      at.len = len;
    }
    k -= __popc(m);
    if (k < 0) break;
  }
}

extern "C" __global__ void __launch_bounds__(AE_NTHREADS, 1)
ae_attn_packed(const __grid_constant__ AeAttnFwdArgs args) {
  extern __shared__ u8 smem_raw[];
  u8* smem = smem_align1024(smem_raw);
  AePackBars* bars = (AePackBars*)(smem + AE_SMEM_BAR);
  AeCtaCtl* ctl = &bars->ctl;
  const u32 warp = threadIdx.x >> 5;
  const u32 lane = threadIdx.x & 31;

  // barriers (60 to 80 clk each, so spread over the warps) and TMEM
  {
    u64* const bar = bars->q_full;  // and the others behind it, up to item_empty
    const int n_bar = 8 + 2 * AE_STAGES + 4;
    if (lane == 0)
      for (int i = (int)warp; i < n_bar; i += 12) mbar_init(bar + i, i >= n_bar - 2 ? AE_PACK_READERS : 1);
    if (threadIdx.x == 0) ctl->abort = 0;
    if (lane == 0) mbar_fence_init();
    if (warp == AE_ROW_WARPS && lane < 3) tma_prefetch_desc(lane == 0 ? &args.tm_q : lane == 1 ? &args.tm_k : &args.tm_v);
  }
  if (warp == AE_ROW_WARPS + 1) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const u32 tmem = ctl->tmem_base;
  ae_grid_wait();  // brought up under the kernel in front; nothing has been read or written outside this CTA so far
  ae_grid_trigger();
  const u32 TM_S0 = 0, TM_S1 = 128, TM_O0 = 256, TM_O1 = 256 + AE_DV;

  if (warp >= AE_ROW_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == AE_ROW_WARPS) {
      // =============================== TMA producer ===============================
      if (lane == 0) {
        u32 fill = 0;
        AePackWork w;
        for (u32 k = 0;; ++k) {
          if (!mbar_wait(&bars->item_full[k & 1], (k >> 1) & 1, ctl, args.status, 1)) break;
          if (!w.take(bars->item[k & 1], args)) break;
          const int hk = w.hq / (args.Hq / args.Hkv);
          if (!mbar_wait(&bars->q_free, (k & 1) ^ 1, ctl, args.status, 2)) break;
          for (int t = 0; t < 2; ++t) {
            if (w.tiles(t) == 0) continue;  // never waited for
            mbar_arrive_expect_tx(&bars->q_full[t], AE_Q_BYTES);
            for (int c = 0; c < AE_D / 64; ++c)
              tma_load_bshd(smem + t * AE_Q_BYTES + c * (AE_BM * 128), &args.tm_q, &bars->q_full[t], c * 64, w.hq + t * w.next_h,
                            w.seq0 + (w.qt0 + t * w.next_qt) * AE_BM, 0);
          }
          bool ok = true;
          for (int n = 0; n <= w.n_steps; ++n, ++fill) {
            const int stage = fill % AE_STAGES;
            const bool have = n < w.n_steps;
            ok = mbar_wait(&bars->kv_empty[stage], ((fill / AE_STAGES) & 1) ^ 1, ctl, args.status, 3);
            if (!ok) break;
            mbar_arrive_expect_tx(&bars->kv_full[stage], (have ? AE_K_BYTES : 0) + (n > 0 ? AE_V_BYTES : 0));
            if (n > 0)
              for (int c = 0; c < AE_DV / 64; ++c)
                tma_load_bshd(smem + AE_SMEM_V + stage * AE_V_BYTES + c * (AE_BN * 128), &args.tm_v, &bars->kv_full[stage], c * 64, hk,
                              w.seq0 + (n - 1) * AE_BN, 0);
            if (have)
              for (int c = 0; c < AE_D / 64; ++c)
                tma_load_bshd(smem + AE_SMEM_K + stage * AE_K_BYTES + c * (AE_BN * 128), &args.tm_k, &bars->kv_full[stage], c * 64, hk,
                              w.seq0 + n * AE_BN, 0);
          }
          if (!ok) break;
          mbar_arrive(&bars->item_empty[k & 1]);
        }
      }
    } else if (warp == AE_ROW_WARPS + 1) {
      // =============================== MMA issuer =================================
      const u32 idesc_s = umma_idesc_f16(AE_BM, AE_BN, AE_BF16, 0, 0);
      const u32 idesc_o = umma_idesc_f16(AE_BM, AE_DV, AE_BF16, 0, 1);
      const u32 q_addr = smem_u32(smem);
      const u64 dk0 = umma_base_k(smem_u32(smem + AE_SMEM_K));
      const u64 dv0 = umma_base_mn(smem_u32(smem + AE_SMEM_V), AE_BN);
      auto issue_s = [&](auto T, int stage) {
        constexpr int t = decltype(T)::value;
        const u64 da = umma_base_k(q_addr + t * AE_Q_BYTES);
        const u64 db = dk0 + (u64)((stage * AE_K_BYTES) >> 4);
        const u32 d = tmem + (t ? TM_S1 : TM_S0);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < AE_D / 16; ++kk) umma_ss(d, umma_step_k(da, kk, AE_BM), umma_step_k(db, kk, AE_BN), idesc_s, kk > 0);
          umma_commit(&bars->s_full[t]);
        }
      };
      auto issue_pv = [&](auto T, auto PC, int stage, u32 acc) {
        constexpr int t = decltype(T)::value;
        constexpr int k0 = decltype(PC)::value * (AE_BN / 32);
        const u64 db = dv0 + (u64)((stage * AE_V_BYTES) >> 4);
        const u32 d = tmem + (t ? TM_O1 : TM_O0);
        const u32 a = tmem + (t ? TM_S1 : TM_S0);
        if (elect_one()) {
#pragma unroll
          for (int kk = k0; kk < k0 + AE_BN / 32; ++kk) umma_ts(d, a + kk * 8, umma_step_mn(db, kk), idesc_o, acc | (kk > 0));
        }
      };
      u32 fill = 0, n_q0 = 0, n_q1 = 0, k = 0;
      bool ok = true;
      AePackWork w;
      for (;; ++k) {
        ok = mbar_wait_w(&bars->item_full[k & 1], (k >> 1) & 1, ctl, args.status, 4);
        if (!ok || !w.take(bars->item[k & 1], args)) break;
        ok = mbar_wait_w(&bars->kv_full[fill % AE_STAGES], (fill / AE_STAGES) & 1, ctl, args.status, 5);
        auto first_s = [&](auto T, u32& n_q) {
          constexpr int t = decltype(T)::value;
          if (!ok || w.tiles(t) == 0) return;
          ok = mbar_wait_w(&bars->q_full[t], n_q & 1, ctl, args.status, 6);
          ++n_q;
          if (ok) issue_s(T, fill % AE_STAGES);
        };
        // the S regions are free: the last item's P V (issued before) reads what was in them, and MMAs run in issue order
        first_s(AeInt<0>{}, n_q0);
        first_s(AeInt<1>{}, n_q1);
        if (!ok) break;
        umma_commit_w(&bars->kv_empty[fill % AE_STAGES]);
        for (int j = 0; j < w.n_steps; ++j) {
          ++fill;
          const int stage = fill % AE_STAGES;
          // A row group that gave up on a wait arrives for that step and leaves; the abort word then ends this loop before it
          // would wait for the group's next arrival.
          ok = mbar_wait_w(&bars->kv_full[stage], (fill / AE_STAGES) & 1, ctl, args.status, 7) && !ctl->abort;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (j == w.n_steps - 1) umma_commit_w(&bars->q_free);
          if (j == (w.n_steps > 1 ? w.n_steps - 2 : 0)) mbar_arrive_warp(&bars->near_end);
          // The sequence ends inside this tile: zeros in the place of the next one's values, as the copy fills them behind the end of a tensor.
          if (j * AE_BN + AE_BN > w.len) {
            for (int r = w.len - j * AE_BN + (int)(lane >> 3); r < AE_BN; r += 4)
#pragma unroll
              for (int c = 0; c < AE_DV / 64; ++c)
                *(uint4*)(smem + AE_SMEM_V + stage * AE_V_BYTES + c * (AE_BN * 128) + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
          auto tile_step = [&](auto T) {
            constexpr int t = decltype(T)::value;
            if (j >= w.tiles(t)) return;
            auto block = [&](auto PC) {
              constexpr int p = decltype(PC)::value;
              named_bar_sync(1 + t * 2 + p, 128 + 32);  // block p of P is in TMEM (and for j = 0 the last item's O has been read)
              tc_fence_after_sync();
              issue_pv(T, PC, stage, p > 0 ? 1u : (u32)(j > 0));
            };
            block(AeInt<0>{});
            block(AeInt<1>{});
            // S of the next step over P of this one (MMAs run in issue order); s_full also says that P V has completed
            if (j + 1 < w.tiles(t))
              issue_s(T, stage);
            else
              umma_commit_w(&bars->o_done[t]);  // the tile's last P V
          };
          tile_step(AeInt<0>{});
          tile_step(AeInt<1>{});
          umma_commit_w(&bars->kv_empty[stage]);
        }
        if (!ok) break;
        ++fill;
        mbar_arrive_warp(&bars->item_empty[k & 1]);
      }
      // every commit of this warp has arrived before the CTA may retire (the last ones have no other waiter)
      if (ok && k > 0) {
        ok = mbar_wait_w(&bars->kv_empty[(fill - 1) % AE_STAGES], ((fill - 1) / AE_STAGES) & 1, ctl, args.status, 8);
        ok = mbar_wait_w(&bars->q_free, (k - 1) & 1, ctl, args.status, 9);
      }
    } else if (warp == AE_ROW_WARPS + 2) {
      // =============================== finder of items ============================
      const int n_head = args.pair_mode == 1 ? args.Hq / 2 : args.Hq, grid = (int)gridDim.x;
      for (int k = 0;; ++k) {
        int i = (int)blockIdx.x;
        if (k > 0) {
          // Taken as late as hides the search, in the last but one step: who is done first has the next longest.  By turns that were settled beforehand
          // the longest CTA had 18 steps where the mean was 13.6 (twelve prompts up to 1500 tokens: 45.0 us, so 42.0).
          if (!mbar_wait_w(&bars->near_end, (k - 1) & 1, ctl, args.status, 14)) break;
          if (lane == 0 && args.n_items > grid) i = grid + atomicAdd(args.next_item, 1);
          i = args.n_items > grid ? __shfl_sync(0xffffffffu, i, 0) : args.n_items;
        }
        if (!mbar_wait_w(&bars->item_empty[k & 1], ((k >> 1) & 1) ^ 1, ctl, args.status, 10)) break;
        AePackItem& it = bars->item[k & 1];
        if (i < args.n_items)
          ae_find_block(it, (int*)(smem + AE_SMEM_SEQ), args, i / n_head, args.pair_mode == 0 ? 2 * AE_BM : AE_BM, k == 0);
        else if (lane == 0)
          it.b = -1;
        if (lane == 0) it.hq = i % n_head * (args.pair_mode == 1 ? 2 : 1);
        __syncwarp();
        const bool end = it.b < 0;
        mbar_arrive_warp(&bars->item_full[k & 1]);
        if (end) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // =============================== row warpgroups =============================
    const int t = warp / 4;                  // q tile of this group
    const u32 row = threadIdx.x & 127;       // row inside the tile == TMEM lane
    const u32 lane_base = ((warp & 3) * 32) << 16;
    const u32 tm_s = tmem + (t ? TM_S1 : TM_S0) + lane_base;
    const u32 tm_o = tmem + (t ? TM_O1 : TM_O0) + lane_base;
    AeCustom cu;
#pragma unroll
    for (int i = 0; i < AE_MAX_CUSTOM; ++i) {
      cu.p[i] = args.custom[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) cu.st[i][k] = args.custom_st[i][k];
    }
    auto p_ready = [&](auto K) { named_bar_arrive(1 + t * 2 + decltype(K)::value, 128 + 32); };
    u32 n_s = 0, n_o = 0;  // score tiles and outputs of this group so far
    bool ok = true;
    AePackWork w;
    for (u32 k = 0; ok; ++k) {
      ok = mbar_wait_row(ok, &bars->item_full[k & 1], (k >> 1) & 1, ctl, args.status, 11);
      if (!ok) {  // the MMA warp may have entered the item: see its loop
        p_ready(AeInt<0>{});
        p_ready(AeInt<1>{});
        break;
      }
      if (!w.take(bars->item[k & 1], args)) break;
      const int n_tiles = w.tiles(t), h_row = w.hq + t * w.next_h;
      const int q_idx = (w.qt0 + t * w.next_qt) * AE_BM + (int)row;
      const bool row_valid = q_idx < w.len;
      AeRow st;
      st.init();
      for (int j = 0; j < n_tiles; ++j) {
        ok = mbar_wait_row(ok, &bars->s_full[t], n_s & 1, ctl, args.status, 12);
        tc_fence_after_sync();
        float s[AE_BN];
        tmem_ld_f32x128(tm_s, s);
        const int kv0 = j * AE_BN;
        // Keys behind the sequence's end do not count, whatever score_mod makes of them.  Compile-time columns and selects, as in attn_fwd.cuh.
#if AE_PACK_SCORES == 1  // score_mod may not keep -inf (a tanh, a slope of the caller's): behind it the mask and the end
#pragma unroll
        for (int c = 0; c < AE_BN; ++c) s[c] = ae_score_mod(s[c], w.b, h_row, q_idx, kv0 + c, cu);
#endif
#if AE_PACK_SCORES == 2  // not a softmax: left out of the row reductions, and P 0
        st.lim = w.len - kv0;
        if (st.lim < AE_BN) {
#pragma unroll
          for (int c = 0; c < AE_BN; ++c) s[c] = c < st.lim ? s[c] : 0.f;
        }
#elif AE_MASK_MODE != 1  // (under a causal mask a row inside the sequence keeps no key behind itself)
        if (kv0 + AE_BN > w.len) {
          const int lim = w.len - kv0;
#pragma unroll
          for (int c = 0; c < AE_BN; ++c) s[c] = c < lim ? s[c] : -__int_as_float(0x7f800000);
        }
#endif
#if AE_MASK_MODE != 0  // (the mask value is -inf: the engine takes no other)
        if (w.partial(j, t)) {
#pragma unroll
          for (int c = 0; c < AE_BN; ++c) s[c] = ae_mask(w.b, h_row, q_idx, kv0 + c) ? s[c] : -__int_as_float(0x7f800000);
        }
#endif
        ae_online_tile<2>(s, st, w.b, h_row, q_idx, kv0, cu, [&](auto K, float o_scale, float (&p)[AE_BN]) {
          constexpr int kb = decltype(K)::value;
          if constexpr (kb == -1) {
#if !AE_O_SCALE_ONE
            // O is rescaled only when some row of the warp needs it.  The previous step's P V has completed: it was issued before these
            // scores' S GEMM.
            if (j > 0 && __any_sync(0xffffffffu, o_scale != 1.0f)) {
#pragma unroll
              for (int c = 0; c < AE_DV / 32; ++c) {
                float f[32];
                u32 r[32];
                tmem_ld_f32x32(tm_o + c * 32, f);
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(f[i] * o_scale);
                tmem_st32(tm_o + c * 32, r);
              }
            }
#endif
          } else {
            // P -> TMEM (16-bit pairs, column c / 2 holds kv columns c, c + 1), a block of 64 columns at a time
#if AE_PACK_SCORES == 2
            if (st.lim < AE_BN) {
#pragma unroll
              for (int c = kb * 64; c < kb * 64 + 64; ++c) p[c] = c < st.lim ? p[c] : 0.f;
            }
#endif
            u32 pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) pk[i] = pack2<AE_BF16>(p[kb * 64 + 2 * i], p[kb * 64 + 2 * i + 1]);
            tmem_st32(tm_s + kb * 32, pk);
            tc_wait_st();
            tc_fence_before_sync();
            p_ready(K);
          }
        });
        ++n_s;
        if (!ok) break;
      }

      // ---- epilogue ----------------------------------------------------------------
      if (n_tiles > 0 && ok) {
        ok = mbar_wait_row(ok, &bars->o_done[t], n_o & 1, ctl, args.status, 13);
        ++n_o;
        tc_fence_after_sync();
        // tcgen05.ld is warp-collective: every lane of the warp runs it; only the stores are per-row.
        const bool store = row_valid && ok;
        u16* orow = (u16*)args.o + (i64)(w.seq0 + (store ? q_idx : 0)) * args.o_ss + (i64)h_row * args.o_sh;
#pragma unroll
        for (int c = 0; c < AE_DV / 32; ++c) {
          float r[32];
          tmem_ld_f32x32(tm_o + c * 32, r);
          if (store) {
            uint4* dst = (uint4*)(orow + c * 32);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint4 x;
              x.x = pack2<AE_BF16>(ae_epilogue_o(r[v * 8 + 0], st), ae_epilogue_o(r[v * 8 + 1], st));
              x.y = pack2<AE_BF16>(ae_epilogue_o(r[v * 8 + 2], st), ae_epilogue_o(r[v * 8 + 3], st));
              x.z = pack2<AE_BF16>(ae_epilogue_o(r[v * 8 + 4], st), ae_epilogue_o(r[v * 8 + 5], st));
              x.w = pack2<AE_BF16>(ae_epilogue_o(r[v * 8 + 6], st), ae_epilogue_o(r[v * 8 + 7], st));
              dst[v] = x;
            }
          }
        }
        tc_fence_before_sync();  // before this group's next hand-over of P, behind which the next item's P V overwrites O
      }
      mbar_arrive_warp(&bars->item_empty[k & 1]);
    }
  }

  // ---- teardown --------------------------------------------------------------------
  tc_fence_before_sync();
  __syncthreads();
  if (warp == AE_ROW_WARPS + 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
  // the last CTA leaves the counters at 0 for the next call
  if (threadIdx.x == 0 && args.n_items > (int)gridDim.x && atomicAdd(args.next_item + 1, 1) == (int)gridDim.x - 1) {
    args.next_item[0] = 0;
    args.next_item[1] = 0;
  }
}
