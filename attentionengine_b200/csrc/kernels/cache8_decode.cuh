// Softmax attention of a few query rows per request over a paged cache of 8-bit floating point (e4m3 codes, a scale for each page and
// kv head), the decode step of a serving loop.
//
//   s = score_mod(ks (q . k_code)),  p = exp(s - max),  o = sum p vs v_code / sum p
//
// Bound by HBM: a key and its value are D + DV bytes for at most 16 query rows (4 flops a byte and row), far below the tensor cores' rate, so
// what counts is that the bytes come without a pause and that the work per byte is small.  Hence mma.sync on 16 x 8 x 16 tiles with the
// keys (and the value dims) as the 16 rows and the query rows as the 8 columns: a warp works for itself, codes go from shared memory through a
// conversion straight into operand registers, and no accumulator takes a trip through TMEM for 8 used rows in 128.
//
// Precision: e4m3 is exact in fp16, so K and V enter the products as they are.  Each query row enters as fp16 times a power of two that
// brings its largest value to [1, 2): exact down to 2^-14 of that power for fp16 input and 2^-17 for bf16, below it within 2^-25 of it.  P is fp16 in [0, 1].  Sums, maxima and the
// scales are fp32.  The value scale goes into the exponent, p' = 2^(x + log2(vs) - m) with m the maximum of x + log2(vs): no page's values are
// scaled after the product, and the row sum takes p' / vs.
//
// Layout of a warp's tile of AE_T keys, lane = 4 g + t: row g + 8 h of score tile i is key 16 i + 8 h + g, so a lane has AE_T / 8 scores
// each of query rows 2 t and 2 t + 1.  The contraction over dims may take them in any order, so lane t takes dims D/4 t ... of a key, whole
// 16-byte chunks.  P goes from the accumulators' layout to the operand's by a transpose of 8 x 8 blocks in registers.  Row g + 8 h of output
// tile m is value dim DV/8 g + 2 m + h: a lane ends with DV/8 dims in order of two query rows.
//
// Copies: warps of their own fetch a tile's keys and values as TMA boxes: the rows of one page (all of them, or AE_T) of a team's heads (below), with the
// swizzle that the reads want.  Page numbers, addresses and barriers are then those warps' instructions (200 of 572 a tile when each warp fetched for
// itself, 300 with 16-byte cp.async), and a box is large: 16 rows of one head at a time, pages of 16 keys took 125 us where pages of 64 took 95.  There
// are four of them, which costs no registers (an SM's quarter has three warps either way): a copy takes one some 600 clk, and with one kv head, eight
// teams, one fetching warp took 43 us where two take 29 and four 22; with one team it makes no difference.  What they do not need of their registers the
// others get (16 query rows of one kv head: 38 us, 30 so).  A warp of a single unit (below) fetches its
// few tiles itself, their pages read together: 9.4 us for 700 keys, 10.0 by the fetching warps (8.3 since the pieces' reads go together too).
//
// Work split: a team of 1, 2, 4 or 8 warps takes the same tiles of as many neighbouring heads, whose keys lie side by side in a token's row of the
// pool: read at one time they come out of DRAM as whole rows (722 MB of eight heads' pages took 172 us head by head, without any arithmetic,
// and 128 us where the heads' pages were apart).  The tiles of all (request, heads, row tile) units stand in one line, which is cut into equal
// intervals, one for each team of a persistent grid; a warp's next tiles are always under way, across the ends of requests too.  A unit that
// lies in one interval is written at once.  What is cut is merged from fp32 partials: inside a CTA through shared memory, between CTAs by
// ae_cache8_merge behind this kernel; the teams are as large as leaves it no more than 16 partials of a unit.  (Merged by the last CTA to arrive
// instead, the partials of eight heads came to that one CTA in 30 us.)  Every CTA finds its interval from the lengths by itself, so the host needs
// to know none of them.  Where the table says that few units cannot be long (args.single), each is a CTA's, without a search and a merge.
//
// Expects the forward prelude (AE_D, AE_DV, AE_BF16, AE_MASK_MODE 0 or 3, ae_score_mod, ae_mask), AE_RT (8 or 16: query rows of a
// tile), AE_T, AE_WARPS, AE_C8_SLOTS, AE_FETCH, AE_MIN_TILES (of a team).

#define AE_KPT (AE_T / 8)
#define AE_NB (AE_RT / 8)      // column blocks: query rows 8 n ... 8 n + 7
#define AE_KB (AE_T * AE_D)    // bytes of a tile's keys
#define AE_VB (AE_T * AE_DV)
#define AE_NEG_INF (-__int_as_float(0x7f800000))

// Byte of 16-byte chunk c of row r in a tile of rows of W bytes, as TMA's swizzle of that width places it.  Read by a quarter warp as
// chunks 2 t (+ 1) or t of rows 8 x + g (keys), and as chunks g (or 8-byte halves g) of rows 2 t + e (values): all in different banks.
template <int W>
AE_DEVICE u32 ae_c8_at(u32 r, u32 c) {
  if constexpr (W == 128) return r * 128 + ((c ^ (r & 7u)) << 4);
  return r * 64 + ((c ^ (r >> 1 & 3u)) << 4);
}
AE_DEVICE u32 ae_e4m3_f16(u32 w, int half) {  // bytes 0, 1 or 2, 3 as a pair of fp16
  u32 x;
  if (half)
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h; }" : "=r"(x) : "r"(w));
  else
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l; }" : "=r"(x) : "r"(w));
  return x;
}
AE_DEVICE void ae_mma16816(float (&c)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
AE_DEVICE u32 ae_transpose8(u32 x) {  // an 8 x 8 block of 16-bit values, row g's columns 2 t, 2 t + 1 in lane 4 g + t
  u32 y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Where the blocks of 16 keys of a head lie in a team's tile: boxes of min(page, AE_T) keys behind each other, in each the heads one after the
// other.  In rows.
struct AeC8Blocks {
  int log2, heads;  // blocks of a box
  AE_DEVICE int at(int i) const { return ((i >> log2) * heads << log2 | (i & ((1 << log2) - 1))) * 16; }
  AE_DEVICE int head(int j) const { return j * (16 << log2); }
};

// One unit's query rows: operands, running maxima (log2, with the value scale in), sums and output of rows 8 n + 2 t + e.
struct AeC8Rows {
  u32 q[AE_NB][AE_D / 16][2];  // of row 8 n + g
  float qs[AE_NB][2];          // what a product is to be multiplied with
  float m[AE_NB][2], l[AE_NB][2];
  float o[AE_NB][AE_DV / 16][4];  // [tile][2 h + e]
};

AE_DEVICE void ae_c8_begin(AeC8Rows& R, const AeCache8DecodeArgs& a, int b, int head, int row0) {
  const u32 g = lane_id() >> 2, t = lane_id() & 3u;
#pragma unroll
  for (int n = 0; n < AE_NB; ++n) {
    const int r = row0 + (int)g + 8 * n;
    u32 w[AE_D / 8];
#pragma unroll
    for (int i = 0; i < AE_D / 8; ++i) w[i] = 0;
    if (r < a.rows) {
      const i64 at = (i64)b * a.q_sb + (a.gq > 1 ? (i64)(head * a.gq + r) * a.q_sh : (i64)r * a.q_ss + (i64)head * a.q_sh);
      const uint4* src = (const uint4*)((const u16*)a.q + at + t * (AE_D / 4));
#pragma unroll
      for (int i = 0; i < AE_D / 32; ++i) {
        const uint4 x = src[i];
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < AE_D / 8; ++i) top = fmaxf(top, fmaxf(fabsf(unpack_lo<AE_BF16>(w[i])), fabsf(unpack_hi<AE_BF16>(w[i]))));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    u32 e = __float_as_uint(top) >> 23;      // 0: zero or below 2^-126; 255: an infinity, which stays one
    e = e < 1u ? 1u : e > 253u ? 127u : e;
    const float f = __uint_as_float((254u - e) << 23), qs = __uint_as_float(e << 23);
#pragma unroll
    for (int i = 0; i < AE_D / 8; ++i) R.q[n][i >> 1][i & 1] = pack2<0>(unpack_lo<AE_BF16>(w[i]) * f, unpack_hi<AE_BF16>(w[i]) * f);
#pragma unroll
    for (int e2 = 0; e2 < 2; ++e2) {
      R.qs[n][e2] = __shfl_sync(0xffffffffu, qs, 4 * (2 * t + e2));
      R.m[n][e2] = AE_NEG_INF;
      R.l[n][e2] = 0.f;
    }
#pragma unroll
    for (int m = 0; m < AE_DV / 16; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) R.o[n][m][i] = 0.f;
  }
}

// The tile's scores, softmax step and P V.  `ks`, `vs`: the scales of the page that this lane's keys lie in; `kv0`: the tile's first key; keys
// from `len` on are zeros in the tile and do not count.
// Keys first (`keys`: the raw products), then the rest, each behind its own copy.
AE_DEVICE void ae_c8_keys(const AeC8Rows& R, const u8* kt, const AeC8Blocks& blk, float (&s)[AE_NB][2][AE_KPT]) {
  const u32 g = lane_id() >> 2, t = lane_id() & 3u;
  u32 w[AE_T / 16][2][AE_D / 16];
#pragma unroll
  for (int i = 0; i < AE_T / 16; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < AE_D / 64; ++j) {
        const uint4 x = *(const uint4*)(kt + blk.at(i) * AE_D + ae_c8_at<AE_D>(8 * h + g, t * (AE_D / 64) + j));
        w[i][h][4 * j] = x.x; w[i][h][4 * j + 1] = x.y; w[i][h][4 * j + 2] = x.z; w[i][h][4 * j + 3] = x.w;
      }
  float c[AE_T / 16][AE_NB][4];
#pragma unroll
  for (int i = 0; i < AE_T / 16; ++i)
#pragma unroll
    for (int n = 0; n < AE_NB; ++n) c[i][n][0] = c[i][n][1] = c[i][n][2] = c[i][n][3] = 0.f;
#pragma unroll
  for (int k = 0; k < AE_D / 16; ++k)  // the score tiles side by side: products into one of them wait for each other
#pragma unroll
    for (int i = 0; i < AE_T / 16; ++i) {
      u32 x[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[h] = ae_e4m3_f16(w[i][h][k], 0);
        x[2 + h] = ae_e4m3_f16(w[i][h][k], 1);
      }
#pragma unroll
      for (int n = 0; n < AE_NB; ++n) ae_mma16816(c[i][n], x[0], x[1], x[2], x[3], R.q[n][k][0], R.q[n][k][1]);
    }
#pragma unroll
  for (int i = 0; i < AE_T / 16; ++i)
#pragma unroll
    for (int n = 0; n < AE_NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e][2 * i] = c[i][n][e];
        s[n][e][2 * i + 1] = c[i][n][2 + e];
      }
}
AE_DEVICE void ae_c8_weights(AeC8Rows& R, float (&s)[AE_NB][2][AE_KPT], u32 (&p)[AE_NB][AE_KPT], int kv0, int len, const float* scales, int heads, int b,
                             int head, int row0, const AeCache8DecodeArgs& a, const AeCustom& cu) {
  const u32 g = lane_id() >> 2, t = lane_id() & 3u;
  const int k0 = kv0 + (int)g;
  float ks[AE_T / 16], lv[AE_T / 16], iv[AE_T / 16];
#pragma unroll
  for (int i = 0; i < AE_T / 16; ++i) {
    const float vs = scales[(AE_T / 16 + i) * heads];
    ks[i] = scales[i * heads];
    lv[i] = ae_log2(vs);
    iv[i] = ae_rcp(vs);
  }
  const bool tail = kv0 + AE_T > len;
  float osc[AE_NB][2];
#pragma unroll
  for (int n = 0; n < AE_NB; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row0 + 8 * n + 2 * (int)t + e;
      const bool valid = r < a.rows;
      const int h = a.gq > 1 ? head * a.gq + (valid ? r : 0) : head, q_idx = a.gq > 1 || !valid ? 0 : r;
      float (&x)[AE_KPT] = s[n][e];
#pragma unroll
      for (int c = 0; c < AE_KPT; ++c) {
        x[c] = fmaf(ae_score_mod(x[c] * (R.qs[n][e] * ks[c / 2]), b, h, q_idx, k0 + 8 * c, cu), AE_LOG2E, lv[c / 2]);
#if AE_MASK_MODE == 3
        x[c] = ae_mask(b, h, q_idx, k0 + 8 * c) ? x[c] : AE_NEG_INF;
#endif
      }
      if (tail) {
#pragma unroll
        for (int c = 0; c < AE_KPT; ++c) x[c] = k0 + 8 * c < len ? x[c] : AE_NEG_INF;
      }
      float top = x[0];
#pragma unroll
      for (int c = 1; c < AE_KPT; ++c) top = fmaxf(top, x[c]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float m = fmaxf(R.m[n][e], top), mu = m == AE_NEG_INF ? 0.f : m;  // nothing kept so far: p = 0
      osc[n][e] = ae_exp2(R.m[n][e] - mu);
      R.m[n][e] = m;
      float l = R.l[n][e] * osc[n][e];  // this lane's keys; the lanes are added at the end
#pragma unroll
      for (int c = 0; c < AE_KPT; ++c) {
        x[c] = ae_exp2(x[c] - mu);
        l = fmaf(x[c], iv[c / 2], l);
      }
      R.l[n][e] = l;
    }
#pragma unroll
    for (int c = 0; c < AE_KPT; ++c) p[n][c] = ae_transpose8(pack2<0>(s[n][0][c], s[n][1][c]));
  }
  bool grown = false;
#pragma unroll
  for (int n = 0; n < AE_NB; ++n) grown |= osc[n][0] != 1.f || osc[n][1] != 1.f;
  if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
    for (int n = 0; n < AE_NB; ++n)
#pragma unroll
      for (int m = 0; m < AE_DV / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) R.o[n][m][i] *= osc[n][i & 1];
  }
}
AE_DEVICE void ae_c8_values(AeC8Rows& R, const u8* vt, const AeC8Blocks& blk, const u32 (&p)[AE_NB][AE_KPT]) {
  const u32 g = lane_id() >> 2, t = lane_id() & 3u;
#pragma unroll
  for (int k = 0; k < AE_T / 16; ++k) {
    constexpr int NW = AE_DV / 32;  // words of a key's values that this lane takes
    u32 w[4][NW];                   // keys 16 k + 2 t, the next, and 8 further on
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (AE_DV == 128) {
        const uint4 x = *(const uint4*)(vt + blk.at(k) * AE_DV + ae_c8_at<AE_DV>(8 * (i >> 1) + 2 * t + (i & 1), g));
        w[i][0] = x.x; w[i][1] = x.y; w[i][NW - 2] = x.z; w[i][NW - 1] = x.w;
      } else {  // odd t the other way round: two rows of 64 bytes share the banks
        const uint2 x = *(const uint2*)(vt + blk.at(k) * AE_DV + ae_c8_at<AE_DV>(8 * (i >> 1) + 2 * t + ((i ^ t) & 1u), g >> 1) + (g & 1u) * 8);
        w[i][0] = x.x; w[i][1] = x.y;
      }
    }
    const bool turned = AE_DV == 64 && (t & 1u);
#pragma unroll
    for (int m = 0; m < AE_DV / 16; ++m) {  // two value dims of two keys in a word
      const u32 sel = (m & 1) ? (turned ? 0x3726 : 0x7362) : (turned ? 0x1504 : 0x5140);
      const u32 lo = __byte_perm(w[0][m / 2], w[1][m / 2], sel), hi = __byte_perm(w[2][m / 2], w[3][m / 2], sel);
      const u32 x0 = ae_e4m3_f16(lo, 0), x1 = ae_e4m3_f16(lo, 1), x2 = ae_e4m3_f16(hi, 0), x3 = ae_e4m3_f16(hi, 1);
#pragma unroll
      for (int n = 0; n < AE_NB; ++n) ae_mma16816(R.o[n][m], x0, x1, x2, x3, p[n][2 * k], p[n][2 * k + 1]);
    }
  }
}

#define AE_SLB (AE_KB + AE_VB)  // a slot of the ring: a tile's keys and its values
#define AE_SCF (AE_T / 8)        // and their scales
#define AE_REC (AE_RT * (AE_DV + 2))  // floats of a partial: output, maxima, sums
#define AE_C8_THREADS ((AE_WARPS + AE_FETCH) * 32)
#define AE_SMEM_HEAD (AE_WARPS * AE_C8_SLOTS * AE_SLB)
#define AE_SMEM_SCALE (AE_SMEM_HEAD + AE_WARPS * AE_REC * 4)
#define AE_SMEM_INFO (AE_SMEM_SCALE + AE_WARPS * AE_C8_SLOTS * AE_SCF * 4)
static_assert(AE_WARPS == 8 && AE_FETCH == 4, "three warpgroups, and their registers");
static_assert(AE_C8_SLOTS * AE_SLB >= AE_REC * 4, "a warp's last partial lies in its own slots");

// A place in the line of tiles: request, heads, row tile, tile; the request's tiles and keys.
struct AeC8Pos {
  int b, h, rt, t, nt, len;  // h: heads of the team's size
};
struct AeC8Record {  // a cut piece
  int b, h, rt;      // b = -1: none
  int begin;         // the unit's first tile in the line
  int from, to, nt;  // tiles of the unit in this piece, and of the whole
  int pad;
};
#define AE_FEW 47
struct AeC8Info {
  u64 full[AE_WARPS][AE_C8_SLOTS], empty[AE_WARPS][AE_C8_SLOTS];  // of each team
  AeC8Record rec[2 * AE_WARPS];  // of each team: the piece it began with (if it was begun before), the piece it ended in (if it goes on)
  int longest, pad;
  int before[AE_FEW + 1];  // tiles of one head's row tile in front of each of a few rows (of more: where the tiles will be)
  AeCtaCtl ctl;
};

AE_DEVICE int ae_c8_len(const AeCache8DecodeArgs& a, int b) {
  const i64 want = a.lens[b], most = (i64)a.max_pages << a.page_log2;
  return (int)(want < 0 ? 0 : want > most ? most : want);
}
AE_DEVICE int ae_c8_tiles(int len) { return len > AE_T ? (len + AE_T - 1) / AE_T : 1; }  // a row without keys has its zeros to write

AE_DEVICE void ae_c8_next(AeC8Pos& p, const AeCache8DecodeArgs& a, int team_log2) {
  if (++p.t < p.nt) return;
  p.t = 0;
  if (++p.rt < a.row_tiles) return;
  p.rt = 0;
  if (++p.h < a.Hkv >> team_log2) return;
  p.h = 0;
  if (++p.b >= a.B) return;  // behind the last tile: not used
  p.len = ae_c8_len(a, p.b);
  p.nt = ae_c8_tiles(p.len);
}

AE_DEVICE bool ae_c8_test(u64* bar, u32 parity) {
  u32 ok;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}
AE_DEVICE void ae_cp4(u32 dst, const float* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
AE_DEVICE void ae_cp16(u32 dst, const float* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

// Copies of a tile of keys kv0 ... and of its scales into a slot, by a whole warp.  `page`: the page of keys 16 i ... of the tile, the same in every lane.
// The boxes are one lane's, the scales AE_C8_HANDS lanes': 64 ragged rows of up to 16384 keys take 122 us, 150 when one lane copies them all.
#define AE_C8_HANDS 8
AE_DEVICE void ae_c8_copy(const AeCache8DecodeArgs& a, u8* kt, float* sc, u64* full, int kv0, int head0, int len, const int (&page)[AE_T / 16], int tl,
                          const AeC8Blocks& blk) {
  const int lane = (int)lane_id(), heads = 1 << tl, box = 16 << blk.log2;  // box: keys of a copy
  u8* const vt = kt + heads * AE_KB;
  u32 want = 0, there = 0;  // blocks of 16 keys
#pragma unroll
  for (int i = 0; i < AE_T / 16; ++i) {
    if (kv0 + 16 * i >= len) continue;
    want |= 1u << i;
    if ((u32)page[i] < (u32)a.num_pages) there |= 1u << i;
  }
  auto page_of = [&](int i) {
    int x = page[0];
#pragma unroll
    for (int k = 1; k < AE_T / 16; ++k) x = i == k ? page[k] : x;
    return x;
  };
  if (there != (1u << AE_T / 16) - 1u) {
    for (int x = lane; x < AE_T / 8 << tl; x += 32)
      if (!(there >> ((x >> tl) & (AE_T / 16 - 1)) & 1u)) sc[x] = 1.f;
    if (want != there) {  // a page that is not there: zeros
      if (lane == 0 && a.status) atomicOr(a.status, 0x1000u);
      for (int i = 0; i < AE_T / 16; ++i) {
        if (!((want & ~there) >> i & 1u)) continue;
        for (int j = 0; j < heads; ++j) {
          const int row = blk.at(i) + blk.head(j);
          for (int x = lane; x < AE_D; x += 32) *(uint4*)(kt + row * AE_D + x * 16) = make_uint4(0, 0, 0, 0);
          for (int x = lane; x < AE_DV; x += 32) *(uint4*)(vt + row * AE_DV + x * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
    }
    __syncwarp();  // what was written comes before the arrival below
  }
  u32 boxes = there;  // the blocks that begin one
  if (blk.log2 > 0) boxes &= blk.log2 > 1 ? 0x11111111u : 0x55555555u;
  if (elect_one()) {
    mbar_arrive_expect_tx(full, (u32)(__popc(boxes) * box * heads) * (AE_D + AE_DV));
#pragma unroll
    for (int i = 0; i < AE_T / 16; ++i) {
      if (!(boxes >> i & 1u)) continue;
      const int row = (kv0 + 16 * i) & ((1 << a.page_log2) - 1);
      if (tl == 0 || tl == a.team_log2) {  // the heads are one box
        tma_load_4d(kt + blk.at(i) * AE_D, &a.tm_k[tl != 0], full, 0, row, head0, page[i]);
        tma_load_4d(vt + blk.at(i) * AE_DV, &a.tm_v[tl != 0], full, 0, row, head0, page[i]);
      } else {
        for (int j = 0; j < heads; ++j) {
          tma_load_4d(kt + (blk.at(i) + blk.head(j)) * AE_D, &a.tm_k[0], full, 0, row, head0 + j, page[i]);
          tma_load_4d(vt + (blk.at(i) + blk.head(j)) * AE_DV, &a.tm_v[0], full, 0, row, head0 + j, page[i]);
        }
      }
    }
  }
  __syncwarp();
  if (lane < AE_C8_HANDS) {
    const int log2 = tl >= 2 && a.scales16 ? tl - 2 : tl;  // copies of a block's scales
    for (int x = lane; x < AE_T / 8 << log2; x += AE_C8_HANDS) {
      const int i = (x >> log2) & (AE_T / 16 - 1), j = x & ((1 << log2) - 1), v = x >> log2 >= AE_T / 16;
      if (!(there >> i & 1u)) continue;
      const float* const src = v ? a.vs + (i64)page_of(i) * a.vs_sp + head0 : a.ks + (i64)page_of(i) * a.ks_sp + head0;
      if (log2 < tl)
        ae_cp16(smem_u32(sc + 4 * x), src + 4 * j);
      else
        ae_cp4(smem_u32(sc + x), src + j);
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
  }
  __syncwarp();
}
// Pages of a tile's blocks of 16 keys.
AE_DEVICE void ae_c8_pages(int (&page)[AE_T / 16], const AeCache8DecodeArgs& a, const AeC8Pos& p, bool is) {
  const int* const row = a.table + (i64)p.b * a.table_stride;
#pragma unroll
  for (int i = 0; i < AE_T / 16; ++i) {
    const i64 first = (i64)p.t * AE_T + 16 * i;
    page[i] = is && first < p.len ? row[first >> a.page_log2] : -1;
  }
}
// After a wait that gave up: nothing may land in the shared memory of a CTA that has left.
AE_DEVICE void ae_c8_drain(u64* full, int fetched) {
  const i64 t0 = clock64();
  for (int i = fetched > AE_C8_SLOTS ? fetched - AE_C8_SLOTS : 0; i < fetched; ++i)
    while (!ae_c8_test(&full[i % AE_C8_SLOTS], (u32)(i / AE_C8_SLOTS) & 1u) && clock64() - t0 < AE_WAIT_CYCLES) {
    }
}

// A fetching warp, for teams `first`, first + AE_FETCH ...: a lane finds a team's tiles, whose interval is [n, n1) and begins at `p`; the copies are
// the whole warp's.
AE_DEVICE void ae_c8_fetch(const AeCache8DecodeArgs& a, u8* smem_raw, AeC8Info* info, int first, AeC8Pos p, int n, int n1, int tl,
                           const AeC8Blocks blk) {
  const int lane = (int)lane_id(), team = lane * AE_FETCH + first < AE_WARPS >> tl ? lane * AE_FETCH + first : 0;
  int page[AE_T / 16];  // of the next tile
  ae_c8_pages(page, a, p, n < n1);
  int slot = 0, fetched = 0;
  u32 parity = 1;  // a slot is free at first
  i64 t0 = clock64();
  while (__any_sync(0xffffffffu, n < n1)) {
    const bool go = n < n1 && ae_c8_test(&info->empty[team][slot], parity);
    const u32 due = __ballot_sync(0xffffffffu, go);
    if (due == 0) {
      // no team is done with a tile: again, within a limit
      const bool late = info->ctl.abort || clock64() - t0 > AE_WAIT_CYCLES;
      if (__any_sync(0xffffffffu, late)) {
        if (info->ctl.abort == 0 && a.status) atomicCAS(a.status, 0u, AE_ST_TIMEOUT_BASE + 2u);
        info->ctl.abort = 1;
        break;
      }
      __nanosleep(300);
      continue;
    }
    for (u32 left = due; left; left &= left - 1) {
      const int w = __ffs(left) - 1, mine = w * AE_FETCH + first, at = __shfl_sync(0xffffffffu, slot, w), s = (mine << tl) * AE_C8_SLOTS + (at << tl);
      int pg[AE_T / 16];
#pragma unroll
      for (int i = 0; i < AE_T / 16; ++i) pg[i] = __shfl_sync(0xffffffffu, page[i], w);
      ae_c8_copy(a, smem_raw + s * AE_SLB, (float*)(smem_raw + AE_SMEM_SCALE) + s * AE_SCF, &info->full[mine][at],
                 __shfl_sync(0xffffffffu, p.t, w) * AE_T, __shfl_sync(0xffffffffu, p.h, w) << tl, __shfl_sync(0xffffffffu, p.len, w), pg, tl, blk);
    }
    if (go) {
      ++n;
      ++fetched;
      ae_c8_next(p, a, tl);
      ae_c8_pages(page, a, p, n < n1);
      if (slot == AE_C8_SLOTS - 1) {
        slot = 0;
        parity ^= 1u;
      } else {
        ++slot;
      }
      t0 = clock64();
    }
    __syncwarp();
  }
  if (info->ctl.abort) ae_c8_drain(info->full[team], fetched);
}

AE_DEVICE void ae_c8_store(const AeCache8DecodeArgs& a, int b, int h, int row, int d, float4 x, float l) {
  if (row >= a.rows) return;
  const i64 at = a.gq > 1 ? (i64)b * a.Hq + h * a.gq + row : ((i64)b * a.rows + row) * a.Hq + h;
  const float f = l == 0.f ? 0.f : 1.f / l;  // l = 0: no kept key
  if (l == 0.f) x = make_float4(0.f, 0.f, 0.f, 0.f);
  *(uint2*)((u16*)a.o + at * AE_DV + d) = make_uint2(pack2<AE_BF16>(x.x * f, x.y * f), pack2<AE_BF16>(x.z * f, x.w * f));
}

// `put(row of the tile, dim, four values)` for the lane's output, then `end(row, m, l)`.
template <class Put, class End>
AE_DEVICE void ae_c8_out(AeC8Rows& R, Put&& put, End&& end) {
  const int g = (int)(lane_id() >> 2), t = (int)(lane_id() & 3u);
#pragma unroll
  for (int n = 0; n < AE_NB; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) R.l[n][e] += __shfl_xor_sync(0xffffffffu, R.l[n][e], o);
#pragma unroll
      for (int m = 0; m < AE_DV / 16; m += 2) {
        const float4 x = make_float4(R.o[n][m][e], R.o[n][m][2 + e], R.o[n][m + 1][e], R.o[n][m + 1][2 + e]);
        put(8 * n + 2 * t + e, (AE_DV / 8) * g + 2 * m, x, R.l[n][e]);
      }
      if (g == 0) end(8 * n + 2 * t + e, R.m[n][e], R.l[n][e]);
    }
}
struct AeC8Sum {
  float m, l;
  float4 o;
};
extern "C" __global__ void __launch_bounds__(AE_C8_THREADS, 1) ae_cache8_decode(const __grid_constant__ AeCache8DecodeArgs a) {
  extern __shared__ u8 smem_dyn[];
  u8* const smem_raw = smem_align1024(smem_dyn);
  const int warp = (int)threadIdx.x >> 5, lane = (int)lane_id();
  AeC8Info* const info = (AeC8Info*)(smem_raw + AE_SMEM_INFO);

  // ---- the line of tiles, and this warp's interval [n0, n1) ----
  int* const before = a.B <= AE_FEW ? info->before : (int*)smem_raw;
  // (a barrier's initialisation takes 60 to 80 clk, one lane after the other: spread over the warps)
  if (warp >= AE_WARPS) {
    if (warp == AE_WARPS && lane < 4) tma_prefetch_desc(lane < 2 ? &a.tm_k[lane] : &a.tm_v[lane - 2]);
    if (warp == AE_WARPS && lane == 0) info->ctl.abort = 0;
  } else if (lane == 0) {
    for (int i = 0; i < AE_C8_SLOTS; ++i) mbar_init(&info->full[warp][i], 1 + AE_C8_HANDS);  // the boxes, and the scales
    mbar_fence_init();
    info->rec[2 * warp].b = info->rec[2 * warp + 1].b = -1;
  }
  ae_grid_wait();     // brought up under the kernel in front; nothing has been read or written outside this CTA so far
  ae_grid_trigger();  // the merge may come up beside
  if (!a.single && threadIdx.x == AE_WARPS * 32) a.cuts[blockIdx.x].parts = 0;
  const int cta = (int)blockIdx.x;
  int tl = 0, teams = AE_WARPS, per = 1, more = 0;  // warps of a team, log2; teams of a CTA; tiles of a team, teams with one more
  int team = warp, n0, n1, cta0 = 0;
  AeC8Pos at;
  auto cut = [&](int w) { return w * per + (w < more ? w : more); };  // first tile of team w of the grid
  auto team_of = [&](int x) { return x < more * (per + 1) ? x / (per + 1) : more + (x - more * (per + 1)) / per; };
  if (a.single) {  // a unit that cannot be long, by its row's place in the grid
    at.b = blockIdx.y;
    at.len = ae_c8_len(a, at.b);
    at.nt = ae_c8_tiles(at.len);
    at.h = a.row_tiles == 1 ? cta : cta / a.row_tiles;
    at.rt = cta - at.h * a.row_tiles;
    if (warp == 0 && lane == 0 && (a.lens[at.b] < 0 || (i64)a.lens[at.b] > (i64)a.max_pages << a.page_log2) && a.status) atomicOr(a.status, 0x800u);
    n0 = at.nt * team / AE_WARPS;
    n1 = at.nt * (team + 1) / AE_WARPS;
    at.t = n0;
  } else {
    if (warp == 0) {
      int sum = 0, longest = 0;
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + lane;
        int x = 0;
        if (b < a.B) {
          x = ae_c8_tiles(ae_c8_len(a, b));
          if ((a.lens[b] < 0 || (i64)a.lens[b] > (i64)a.max_pages << a.page_log2) && a.status) atomicOr(a.status, 0x800u);
        }
        longest = longest > x ? longest : x;
        int s = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += y;
        }
        if (b < a.B) before[b] = sum + s - x;
        sum += __shfl_sync(0xffffffffu, s, 31);
      }
      longest = __reduce_max_sync(0xffffffffu, longest);
      if (lane == 0) {
        before[a.B] = sum;
        info->longest = longest;
      }
    }
    __syncthreads();
    // equal intervals of at least AE_MIN_TILES for each team, the first `more` one longer
    for (int i = 1; i <= a.team_log2; ++i)
      if ((i64)info->longest * gridDim.x <= (i64)16 * before[a.B] * (a.Hkv >> i) * a.row_tiles) tl = i;
    const int units = (a.Hkv >> tl) * a.row_tiles, total = before[a.B] * units;
    teams = AE_WARPS >> tl;
    int n_team = (int)gridDim.x * teams;
    if (n_team * AE_MIN_TILES > total) n_team = total < teams * AE_MIN_TILES ? teams : (total / AE_MIN_TILES) & ~(teams - 1);
    per = total / n_team;
    more = total - per * n_team;
    if (cta * teams >= n_team) return;
    // a warp for its team, a lane of the fetching warps for each of theirs
    const int theirs = lane * AE_FETCH + warp - AE_WARPS;
    team = warp < AE_WARPS ? warp >> tl : theirs < teams ? theirs : 0;
    cta0 = cut(cta * teams);
    n0 = cut(cta * teams + team);
    n1 = cut(cta * teams + team + 1);
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] * units <= n0)
        lo = mid;
      else
        hi = mid;
    }
    at.b = lo;
    at.len = ae_c8_len(a, lo);
    at.nt = before[lo + 1] - before[lo];
    const int in = n0 - before[lo] * units, u = in / at.nt;
    at.t = in - u * at.nt;
    at.h = a.row_tiles == 1 ? u : u / a.row_tiles;
    at.rt = u - at.h * a.row_tiles;
  }
  const int mate = warp & ((1 << tl) - 1);
  if (!a.single && warp < AE_WARPS && lane == 0) {
    for (int i = warp; i < teams * AE_C8_SLOTS; i += AE_WARPS) mbar_init(&info->empty[0][0] + i, 1u << tl);
    mbar_fence_init();
  }
  if (!a.single && a.B > AE_FEW) fence_proxy_async_smem();
  __syncthreads();  // `before` has been read: the copies may come

  AeCustom cu;
#pragma unroll
  for (int i = 0; i < AE_MAX_CUSTOM; ++i) {
    cu.p[i] = a.custom[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) cu.st[i][k] = a.custom_st[i][k];
  }
  const AeC8Blocks blk = {(a.page_log2 < AE_T_LOG2 ? a.page_log2 : AE_T_LOG2) - 4, 1 << tl};
  u8* const ring = smem_raw + (team << tl) * (AE_C8_SLOTS * AE_SLB);  // the team's
  float* const scales = (float*)(smem_raw + AE_SMEM_SCALE) + (team << tl) * (AE_C8_SLOTS * AE_SCF);
  auto slot_of = [&](int c, int later, int j) { return a.part + (((i64)c * 2 + later) * AE_WARPS + j) * AE_REC; };
  auto part_of = [&](int i, int j) {  // record i's partial of the team's j-th head
    const int w = ((i >> 1) << tl) + j;
    return (i & 1) ? (float*)(smem_raw + w * (AE_C8_SLOTS * AE_SLB)) : (float*)(smem_raw + AE_SMEM_HEAD) + w * AE_REC;
  };
  if (warp >= AE_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int first = warp - AE_WARPS;
    if (!a.single) ae_c8_fetch(a, smem_raw, info, first, at, n0, lane * AE_FETCH + first < teams ? n1 : n0, tl, blk);
    return;
  }
  asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");  // 8 x 208 + 4 x 88 = 12 x 168
  AeC8Rows R;
  int pages = 0, fetched = n0;  // of a single unit: lane i's page of keys 16 i ... of the warp's tiles
  if (a.single) {
    const i64 first = (i64)n0 * AE_T + 16 * lane;
    pages = first < at.len && first < (i64)n1 * AE_T ? a.table[(i64)at.b * a.table_stride + (first >> a.page_log2)] : -1;
  }
  int from = 0, slot = 0;
  u32 parity = 0;
#pragma unroll 1
  for (int n = n0; n < n1; ++n) {
    const int row0 = at.rt * AE_RT, kv0 = at.t * AE_T, head = (at.h << tl) + mate;
    if (n == n0 || at.t == 0) {
      ae_c8_begin(R, a, at.b, head, row0);
      from = at.t;
    }
    if (a.single) {
      __syncwarp();  // the tile in front has been used
      for (; fetched < n1 && fetched < n + AE_C8_SLOTS; ++fetched) {
        int pg[AE_T / 16];
#pragma unroll
        for (int i = 0; i < AE_T / 16; ++i) pg[i] = __shfl_sync(0xffffffffu, pages, (fetched - n0) * (AE_T / 16) + i);
        const int x = (fetched - n0) % AE_C8_SLOTS;
        ae_c8_copy(a, ring + x * AE_SLB, scales + x * AE_SCF, &info->full[team][x], fetched * AE_T, at.h, at.len, pg, 0, blk);
      }
    }
    // a wait that gives up is reported; the CTA goes on to its end
    mbar_wait_w(&info->full[team][slot], parity, &info->ctl, a.status, 1);
    u8* const kt = ring + (slot << tl) * AE_SLB + blk.head(mate) * AE_D;
    u8* const vt = ring + (slot << tl) * AE_SLB + (AE_KB << tl) + blk.head(mate) * AE_DV;
    if (kv0 + AE_T > at.len) {  // what lies behind the row's keys may be anything, and a P of 0 makes a NaN of a NaN
      for (int x = (at.len - kv0) * (AE_DV / 16) + lane; x < AE_T * (AE_DV / 16); x += 32)
        *(uint4*)(vt + blk.at(x / AE_DV) * AE_DV + x % AE_DV * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();  // before the next copy into the slot
      __syncwarp();
    }
    float s[AE_NB][2][AE_KPT];
    u32 p[AE_NB][AE_KPT];
    ae_c8_keys(R, kt, blk, s);
    ae_c8_weights(R, s, p, kv0, at.len, scales + (slot << tl) * AE_SCF + mate, 1 << tl, at.b, head, row0, a, cu);
    ae_c8_values(R, vt, blk, p);
    if (!a.single) mbar_arrive_warp(&info->empty[team][slot]);
    if (slot == AE_C8_SLOTS - 1) {
      slot = 0;
      parity ^= 1u;
    } else {
      ++slot;
    }
    const bool ends = at.t == at.nt - 1;
    if (ends && from == 0) {
      ae_c8_out(R, [&](int r, int d, float4 x, float l) { ae_c8_store(a, at.b, head, row0 + r, d, x, l); }, [](int, float, float) {});
    } else if (ends || n == n1 - 1) {
      // what was begun before is the team's first piece; what goes on is its last, and its copies have all been used.  A team that is the
      // whole CTA has nothing to add to it.
      const bool later = n - at.t >= cta0;
      float* const part = teams == 1 ? slot_of(cta, later ? 1 : 0, mate) : part_of(2 * team + (ends ? 0 : 1), mate);
      if (teams > 1 && tl > 0 && n == n1 - 1) named_bar_sync(1 + team, 32 << tl);  // the slots are the team's
      ae_c8_out(R, [&](int r, int d, float4 x, float) { *(float4*)(part + r * AE_DV + d) = x; },
                [&](int r, float m, float l) {
                  part[AE_RT * AE_DV + r] = m;
                  part[AE_RT * AE_DV + AE_RT + r] = l;
                });
      if (lane == 0 && mate == 0) {
        if (teams > 1)
          info->rec[2 * team + (ends ? 0 : 1)] = {at.b, at.h, at.rt, n - at.t, from, at.t + 1, at.nt, 0};
        else if (later)
          a.cuts[cta] = {team_of(n - at.t + at.nt - 1) - cta + 1, at.b, at.h << tl, at.rt, 1 << tl};
      }
    }
    if (n < n1 - 1) ae_c8_next(at, a, tl);
  }
  if (a.single && info->ctl.abort) ae_c8_drain(info->full[team], fetched - n0);
  if (teams == 1) return;
  named_bar_sync(15, AE_WARPS * 32);

  // ---- cut units: the pieces of this CTA, then of all CTAs ----
  constexpr int ITEMS = AE_RT * (AE_DV / 4);
  // records in a lane each; the pieces of a unit are those with the same first tile
  AeC8Record rec = info->rec[lane < 2 * teams ? lane : 0];
  u32 left = __ballot_sync(0xffffffffu, lane < 2 * teams && rec.b >= 0);
  while (left) {
    const int i = __ffs(left) - 1;
    const AeC8Record first = info->rec[i];
    const u32 has = __ballot_sync(0xffffffffu, rec.begin == first.begin) & left;
    const int to = __shfl_sync(0xffffffffu, rec.to, 31 - __clz(has));
    left &= ~has;
    const bool whole = first.from == 0 && to == first.nt, later = first.begin >= cta0;
    for (int x = (int)threadIdx.x; x < ITEMS << tl; x += AE_WARPS * 32) {
      const int m0 = x / ITEMS, r = x % ITEMS / (AE_DV / 4), d = x % (AE_DV / 4) * 4;
      if (first.rt * AE_RT + r >= a.rows) continue;
      AeC8Sum s = {AE_NEG_INF, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
      float m[2 * AE_WARPS], l[2 * AE_WARPS];  // all pieces' reads on their way together
#pragma unroll
      for (int k = 0; k < 2 * AE_WARPS; ++k) {
        const float* const p = part_of(k, m0) + AE_RT * AE_DV + r;
        m[k] = has >> k & 1u ? p[0] : AE_NEG_INF;
        l[k] = has >> k & 1u ? p[AE_RT] : 0.f;
        s.m = fmaxf(s.m, m[k]);
      }
#pragma unroll
      for (int k = 0; k < 2 * AE_WARPS; ++k) {
        const bool none = m[k] == AE_NEG_INF && l[k] == 0.f;  // no kept key, or not of this unit
        const float f = none ? 0.f : ae_exp2(m[k] - s.m);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!none) o = *(const float4*)(part_of(k, m0) + r * AE_DV + d);
        s.l += f * l[k];
        s.o.x += f * o.x; s.o.y += f * o.y; s.o.z += f * o.z; s.o.w += f * o.w;
      }
      if (whole) {
        ae_c8_store(a, first.b, (first.h << tl) + m0, first.rt * AE_RT + r, d, s.o, s.l);
      } else {
        float* const slot = slot_of(cta, later ? 1 : 0, m0);
        *(float4*)(slot + r * AE_DV + d) = s.o;
        if (d == 0) {
          slot[AE_RT * AE_DV + r] = s.m;
          slot[AE_RT * AE_DV + AE_RT + r] = s.l;
        }
      }
    }
    if (!whole && later && threadIdx.x == 0)  // it goes on: what the merge has to know
      a.cuts[cta] = {team_of(first.begin + first.nt - 1) / teams - cta + 1, first.b, first.h << tl, first.rt, 1 << tl};
  }
}
