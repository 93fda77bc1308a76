// Softmax attention of a few query rows per request over a paged cache of 8-bit floating point (e4m3 codes, a scale for each page and
// kv head), the decode step of a serving loop.
//
//   s = score_mod(ks (q . k_code)),  p = exp(s - max),  o = sum p vs v_code / sum p
//
// Bound by HBM: a key and its value are D + DV bytes for at most 16 query rows (4 flops a byte and row), far below the tensor cores' rate, so
// what counts is that the bytes come without a pause and that the work per byte is small.  Hence mma.sync on 16 x 8 x 16 tiles (query rows
// x keys x dims): a warp works for itself, keys stay in the registers that the conversion wrote, scores leave the products in the layout in which
// P enters the next, and no accumulator takes a trip through TMEM for 8 rows of use in 128.
//
// Precision: e4m3 is exact in fp16, so K and V enter the products as they are.  Each query row enters as fp16 times a power of two that
// brings its largest value to [1, 2): exact for fp16 input, and for bf16 down to 2^-24 of that value.  P is fp16 in [0, 1].  Sums, maxima and the
// scales are fp32.  The value scale goes into the exponent, p' = 2^(x + log2(vs) - m) with m the maximum of x + log2(vs): no page's values are
// scaled after the product, and the row sum takes p' / vs.
//
// Layout of a warp's tile (AE_T keys, AE_T / 4 = KPT for each of the four lanes t of a quad): column n of score tile j is key
// KPT (n / 2) + 2 j + n % 2, so lane t's scores of a row are keys KPT t ... KPT t + KPT - 1 in order, all in one page (a page has 16 slots or more):
// one key scale, one value scale a lane.  The contraction over dims may take them in any order, so lane t takes dims
// D/4 t ... of a key, whole 16-byte chunks.  Value dims likewise: column n of output tile m is dim DV/8 n + m.
//
// Expects the forward prelude (AE_D, AE_DV, AE_BF16, AE_MASK_MODE 0 or 3, ae_score_mod, ae_mask), AE_RT (8 or 16: query rows of a
// tile), AE_T, AE_WARPS.

#define AE_KPT (AE_T / 4)
#define AE_KB (AE_T * AE_D)    // bytes of a tile's keys
#define AE_VB (AE_T * AE_DV)
#define AE_NEG_INF (-__int_as_float(0x7f800000))

// Byte of 16-byte chunk c of row r in a tile of rows of W bytes.  Written a row's chunks at a time; read by a quarter warp as chunks 2 t (+ 1)
// or t of two rows (keys), and as neighbouring chunks of the four rows KPT t + i (values): all eight in different banks.
template <int W>
AE_DEVICE u32 ae_c8_at(u32 r, u32 c) {
  const u32 t = r / AE_KPT & 3u;
  if constexpr (W == 128) return r * 128 + ((c ^ (t << 1) ^ (r & 1u)) << 4);
  return (r ^ (t >> 1)) * 64 + ((c ^ ((t & 1u) << 1)) << 4);  // two rows of 64 bytes share the banks
}
AE_DEVICE void ae_cp16(u32 dst, const void* src, bool fetch) {  // zeros where `fetch` is false
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fetch ? 16 : 0) : "memory");
}
AE_DEVICE u32 ae_e4m3_f16(u32 w, int half) {  // bytes 0, 1 or 2, 3 as a pair of fp16
  u32 h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((u16)(half ? w >> 16 : w)));
  return h;
}
AE_DEVICE void ae_mma16816(float (&c)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One request's query rows of a unit: fragments, running maxima (log2, with the value scale in) and sums, output.
struct AeC8Rows {
  u32 q[AE_D / 16][AE_RT / 4];  // [k step][low dims, high dims (of row g), the same of row g + 8]
  float qs[AE_RT / 8];          // what a product is to be multiplied with
  float m[AE_RT / 8], l[AE_RT / 8];
  float o[AE_DV / 8][AE_RT / 4];  // [tile][2 (row / 8) + column]
};

AE_DEVICE void ae_c8_begin(AeC8Rows& R, const AeCache8DecodeArgs& a, int b, int unit, int row0) {
  const u32 g = lane_id() >> 2, t = lane_id() & 3u;
#pragma unroll
  for (int hf = 0; hf < AE_RT / 8; ++hf) {
    const int r = row0 + (int)g + 8 * hf;
    u32 w[AE_D / 8];
#pragma unroll
    for (int i = 0; i < AE_D / 8; ++i) w[i] = 0;
    if (r < a.rows) {
      const i64 at = a.gq > 1 ? (i64)b * a.q_sb + (i64)(unit * a.gq + r) * a.q_sh : (i64)b * a.q_sb + (i64)r * a.q_ss + (i64)unit * a.q_sh;
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
    const float f = __uint_as_float((254u - e) << 23);
    R.qs[hf] = __uint_as_float(e << 23);
#pragma unroll
    for (int i = 0; i < AE_D / 8; ++i) R.q[i >> 1][2 * hf + (i & 1)] = pack2<0>(unpack_lo<AE_BF16>(w[i]) * f, unpack_hi<AE_BF16>(w[i]) * f);
    R.m[hf] = AE_NEG_INF;
    R.l[hf] = 0.f;
  }
#pragma unroll
  for (int m = 0; m < AE_DV / 8; ++m)
#pragma unroll
    for (int i = 0; i < AE_RT / 4; ++i) R.o[m][i] = 0.f;
}

// The tile's scores, softmax step and P V.  `ks`, `vs`: the scales of the page that this lane's keys lie in; `kv0`: the tile's first key; keys
// from `len` on are zeros in the tile and do not count.
AE_DEVICE void ae_c8_tile(AeC8Rows& R, const u8* kt, const u8* vt, int kv0, int len, float ks, float vs, int b, int unit, int row0,
                          const AeCache8DecodeArgs& a, const AeCustom& cu) {
  const u32 g = lane_id() >> 2, t = lane_id() & 3u;
  float s[AE_RT / 8][AE_KPT];
#pragma unroll
  for (int j = 0; j < AE_T / 8; ++j) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    const u32 r = AE_KPT * (g >> 1) + 2 * j + (g & 1u);
    u32 w[AE_D / 16];
#pragma unroll
    for (int i = 0; i < AE_D / 64; ++i) {
      const uint4 x = *(const uint4*)(kt + ae_c8_at<AE_D>(r, t * (AE_D / 64) + i));
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
#pragma unroll
    for (int k = 0; k < AE_D / 16; ++k) {
      if constexpr (AE_RT == 16)
        ae_mma16816(c, R.q[k][0], R.q[k][AE_RT / 4 - 2], R.q[k][1], R.q[k][AE_RT / 4 - 1], ae_e4m3_f16(w[k], 0), ae_e4m3_f16(w[k], 1));
      else
        ae_mma16816(c, R.q[k][0], 0u, R.q[k][1], 0u, ae_e4m3_f16(w[k], 0), ae_e4m3_f16(w[k], 1));
    }
#pragma unroll
    for (int hf = 0; hf < AE_RT / 8; ++hf) {
      s[hf][2 * j] = c[2 * hf];
      s[hf][2 * j + 1] = c[2 * hf + 1];
    }
  }
  const int k0 = kv0 + (int)t * AE_KPT;
  const float lv = ae_log2(vs), iv = 1.f / vs;
  float osc[AE_RT / 8];
  u32 p[AE_RT / 8][AE_KPT / 2];
#pragma unroll
  for (int hf = 0; hf < AE_RT / 8; ++hf) {
    const int r = row0 + (int)g + 8 * hf;
    const bool valid = r < a.rows;
    const int h = a.gq > 1 ? unit * a.gq + (valid ? r : 0) : unit, q_idx = a.gq > 1 || !valid ? 0 : r;
    const float f = R.qs[hf] * ks;
    float top = AE_NEG_INF;
#pragma unroll
    for (int c = 0; c < AE_KPT; ++c) {
      float x = ae_score_mod(s[hf][c] * f, b, h, q_idx, k0 + c, cu) * AE_LOG2E + lv;
#if AE_MASK_MODE == 3
      x = ae_mask(b, h, q_idx, k0 + c) ? x : AE_NEG_INF;
#endif
      x = k0 + c < len ? x : AE_NEG_INF;
      s[hf][c] = x;
      top = fmaxf(top, x);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float m = fmaxf(R.m[hf], top), mu = m == AE_NEG_INF ? 0.f : m;  // nothing kept so far: p = 0
    osc[hf] = ae_exp2(R.m[hf] - mu);
    R.m[hf] = m;
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < AE_KPT; c += 2) {
      const float x = ae_exp2(s[hf][c] - mu), y = ae_exp2(s[hf][c + 1] - mu);
      sum += x + y;
      p[hf][c / 2] = pack2<0>(x, y);
    }
    R.l[hf] = R.l[hf] * osc[hf] + sum * iv;  // this lane's keys; the quad's lanes are added at the end
  }
  if (__any_sync(0xffffffffu, osc[0] != 1.f || osc[AE_RT / 8 - 1] != 1.f)) {
#pragma unroll
    for (int m = 0; m < AE_DV / 8; ++m)
#pragma unroll
      for (int i = 0; i < AE_RT / 4; ++i) R.o[m][i] *= osc[i >> 1];
  }
#pragma unroll
  for (int k = 0; k < AE_T / 16; ++k) {
    constexpr int NW = AE_DV / 32;  // words of a key's values that this lane takes
    u32 w[4][NW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32 r = AE_KPT * t + 4 * k + i;
      if constexpr (AE_DV == 128) {
        const uint4 x = *(const uint4*)(vt + ae_c8_at<AE_DV>(r, g));
        w[i][0] = x.x; w[i][1] = x.y; w[i][NW - 2] = x.z; w[i][NW - 1] = x.w;
      } else {
        const uint2 x = *(const uint2*)(vt + ae_c8_at<AE_DV>(r, g >> 1) + (g & 1u) * 8);
        w[i][0] = x.x; w[i][1] = x.y;
      }
    }
#pragma unroll
    for (int n = 0; n < NW; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // two value dims of two keys in a word
        const u32 b0 = __byte_perm(w[0][n], w[1][n], e ? 0x7362 : 0x5140), b1 = __byte_perm(w[2][n], w[3][n], e ? 0x7362 : 0x5140);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          float (&o)[AE_RT / 4] = R.o[4 * n + 2 * e + d];
          float c[4] = {o[0], o[1], AE_RT == 16 ? o[AE_RT / 4 - 2] : 0.f, AE_RT == 16 ? o[AE_RT / 4 - 1] : 0.f};
          ae_mma16816(c, p[0][2 * k], AE_RT == 16 ? p[AE_RT / 8 - 1][2 * k] : 0u, p[0][2 * k + 1], AE_RT == 16 ? p[AE_RT / 8 - 1][2 * k + 1] : 0u,
                      ae_e4m3_f16(b0, d), ae_e4m3_f16(b1, d));
#pragma unroll
          for (int i = 0; i < AE_RT / 4; ++i) o[i] = c[i];
        }
      }
    }
  }
}

// A tile into shared memory: keys kv0 ... of the row, zeros from `len` on.  `page`: lane l holds the page of keys kv0 + 16 l ...
template <int W>
AE_DEVICE void ae_c8_fetch(u8* dst, const u8* pool, i64 sp, i64 st, int page_log2, int kv0, int len, int page) {
  constexpr int CPR = W / 16, RPI = 32 / CPR;  // chunks of a row, rows of an instruction
  const int c = (int)lane_id() % CPR, rr = (int)lane_id() / CPR;
#pragma unroll
  for (int i = 0; i < AE_T / RPI; ++i) {
    const int r = i * RPI + rr;
    const int pg = __shfl_sync(0xffffffffu, page, i * RPI / 16);
    const i64 at = (i64)pg * sp + (i64)((kv0 + r) & ((1 << page_log2) - 1)) * st + c * 16;
    const bool in = kv0 + r < len && pg >= 0;
    ae_cp16(smem_u32(dst) + ae_c8_at<W>(r, c), pool + (in ? at : 0), in);
  }
}

// One CTA per (request, unit, row tile): the warps take its tiles in turn and merge at the end.
extern "C" __global__ void __launch_bounds__(AE_WARPS * 32) ae_cache8_decode(const __grid_constant__ AeCache8DecodeArgs a) {
  extern __shared__ __align__(128) u8 smem_raw[];
  const u32 warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  u8* const kt = smem_raw + warp * (AE_KB + AE_VB);
  u8* const vt = kt + AE_KB;
  float* const part = (float*)(smem_raw + AE_WARPS * (AE_KB + AE_VB));  // [warp][row][DV], then [warp][row] maxima and sums
  float* const part_m = part + AE_WARPS * AE_RT * AE_DV;
  float* const part_l = part_m + AE_WARPS * AE_RT;
  const int b = blockIdx.z, unit = blockIdx.y, row0 = blockIdx.x * AE_RT;
  AeCustom cu;
#pragma unroll
  for (int i = 0; i < AE_MAX_CUSTOM; ++i) {
    cu.p[i] = a.custom[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) cu.st[i][k] = a.custom_st[i][k];
  }
  i64 want = a.lens[b];
  const i64 most = (i64)a.max_pages << a.page_log2;
  if ((want > most || want < 0) && threadIdx.x == 0 && a.status) atomicOr(a.status, 0x800u);
  const int len = (int)(want < 0 ? 0 : want > most ? most : want);
  AeC8Rows R;
  ae_c8_begin(R, a, b, unit, row0);
  for (int kv0 = (int)warp * AE_T; kv0 < len; kv0 += AE_WARPS * AE_T) {
    int page = -1;
    const i64 first = (i64)kv0 + 16 * (i64)lane;
    if ((int)lane < AE_T / 16 && first < len) {
      page = a.table[(i64)b * a.table_stride + (first >> a.page_log2)];
      if ((u32)page >= (u32)a.num_pages) {
        if (a.status) atomicOr(a.status, 0x1000u);
        page = -1;
      }
    }
    ae_c8_fetch<AE_D>(kt, a.k + (i64)unit * a.k_sh, a.k_sp, a.k_st, a.page_log2, kv0, len, page);
    ae_c8_fetch<AE_DV>(vt, a.v + (i64)unit * a.v_sh, a.v_sp, a.v_st, a.page_log2, kv0, len, page);
    asm volatile("cp.async.commit_group;" ::: "memory");
    float ks = page >= 0 ? a.ks[(i64)page * a.ks_sp + unit] : 1.f, vs = page >= 0 ? a.vs[(i64)page * a.vs_sp + unit] : 1.f;
    ks = __shfl_sync(0xffffffffu, ks, t * AE_KPT / 16);
    vs = __shfl_sync(0xffffffffu, vs, t * AE_KPT / 16);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    ae_c8_tile(R, kt, vt, kv0, len, ks, vs, b, unit, row0, a, cu);
    __syncwarp();
  }
#pragma unroll
  for (int hf = 0; hf < AE_RT / 8; ++hf) {
    R.l[hf] += __shfl_xor_sync(0xffffffffu, R.l[hf], 1);
    R.l[hf] += __shfl_xor_sync(0xffffffffu, R.l[hf], 2);
    const u32 r = g + 8 * hf;
    if (t == 0) {
      part_m[warp * AE_RT + r] = R.m[hf];
      part_l[warp * AE_RT + r] = R.l[hf];
    }
#pragma unroll
    for (int m = 0; m < AE_DV / 8; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) part[(warp * AE_RT + r) * AE_DV + (AE_DV / 8) * (2 * t + e) + m] = R.o[m][2 * hf + e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < AE_RT * AE_DV / 2; i += AE_WARPS * 32) {
    const int r = i / (AE_DV / 2), d = i % (AE_DV / 2) * 2;
    if (row0 + r >= a.rows) continue;
    float m = AE_NEG_INF;
    for (int w = 0; w < AE_WARPS; ++w) m = fmaxf(m, part_m[w * AE_RT + r]);
    float l = 0.f, x = 0.f, y = 0.f;
    for (int w = 0; w < AE_WARPS; ++w) {
      if (part_m[w * AE_RT + r] == AE_NEG_INF && part_l[w * AE_RT + r] == 0.f) continue;  // no kept key
      const float f = ae_exp2(part_m[w * AE_RT + r] - m);
      l += f * part_l[w * AE_RT + r];
      x += f * part[(w * AE_RT + r) * AE_DV + d];
      y += f * part[(w * AE_RT + r) * AE_DV + d + 1];
    }
    if (l == 0.f) x = y = 0.f, l = 1.f;  // a row without a kept key
    const i64 row = a.gq > 1 ? (i64)b * a.Hq + unit * a.gq + row0 + r : ((i64)b * a.rows + row0 + r) * a.Hq + unit;
    *(u32*)((u16*)a.o + row * AE_DV + d) = pack2<AE_BF16>(x / l, y / l);
  }
}
