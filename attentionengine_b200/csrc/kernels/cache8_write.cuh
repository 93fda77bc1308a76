// Write of new keys and values into a paged cache of 8-bit floating point (e4m3), a scale for each page and head.
//
// The scale is the smallest power of two s with amax / s <= 448 (the largest e4m3 value), at least 2^-64; codes are x / s rounded to
// nearest even.  A power of two, because e4m3 is a floating-point format: any scale gives the same relative precision, and with this
// one x / s is exact, so the only rounding is the one to e4m3; and when a page that goes on needs a coarser scale, the codes that are there are
// multiplied by a power of two, which changes none of them but at the bottom of the range.  (Where a page came with another scale, both are
// rounded once all the same: ae_sticky.)  amax takes the finite values: an infinity or a NaN becomes NaN and does not take the others'
// precision.
//
// One CTA per (segment, head, K or V) owns the page's part for that head, so there is nothing to lock; a segment's heads run side by side, since their
// values are neighbours in memory.  A page is at most 128 x 128 values: the CTA holds its 16-bit values in registers between the maximum and the
// rounding, one pass over the data.  Bound by HBM (2 bytes in and 1 out a value) once the instructions are few: the maximum is taken of the
// 16-bit patterns without their sign, two at a time, and infinities are looked for again only where that maximum is one (or a NaN).
// A thread has 64 of a full page's values, eight loads on their way: 16029 tokens of 8 heads of 128 dims (98.5 MB) take 18.5 us in pages of 64
// (5.3 TB/s; 26.2 value by value in fp32), 19.1 in pages of 32 and 19.3 in pages of 16; with half the values a thread, 20.5 (pages of 32) and
// 20.7 (of 16), with twice as many 23.5 (of 64 and of 32).  For a step of single tokens, latency.
#define AE_W_MAXD (AE_D > AE_DV ? AE_D : AE_DV)
#define AE_W_CHUNKS (AE_PAGE * (AE_W_MAXD / 8))                                 // 16-byte chunks of a full page's values
#define AE_W_PER ((AE_W_CHUNKS + AE_W_THREADS - 1) / AE_W_THREADS)
#define AE_E4M3_MAX 448.f
#define AE_SCALE_MIN 5.421010862427522e-20f                                       // 2^-64

// The power-of-two scale of amax, from its bits: amax = 1.m 2^e; 448 = 1.75 2^8.
AE_DEVICE float ae_pow2_scale(float amax) {
  const u32 u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased
  return e >= 1 ? fmaxf(__uint_as_float((u32)e << 23), AE_SCALE_MIN) : AE_SCALE_MIN;
}
// Two values to e4m3, `lo` in the low byte; beyond +-448 it saturates.
AE_DEVICE u32 ae_e4m3x2(float lo, float hi) {
  u16 r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
AE_DEVICE u32 ae_e4m3x2_half(u32 x, u32 factor) {  // of a pair of fp16 times a pair
  u16 r;
  asm("{ .reg .b32 y; mul.rn.f16x2 y, %1, %2; cvt.rn.satfinite.e4m3x2.f16x2 %0, y; }" : "=h"(r) : "r"(x), "r"(factor));
  return r;
}
AE_DEVICE void ae_from_e4m3x2(u32 w, float& lo, float& hi) {
  u32 h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((u16)w));
  lo = unpack_lo<0>(h);
  hi = unpack_hi<0>(h);
}

// A quotient or product rounded towards 0, its last bit set where something was left (`rest`): rounded again to fewer bits it gives what the exact
// value gives.
AE_DEVICE float ae_sticky(float x, float rest) { return rest != 0.f ? __uint_as_float(__float_as_uint(x) | 1u) : x; }
AE_DEVICE float ae_div_odd(float x, float y) {
  const float q = __fdiv_rz(x, y);
  return ae_sticky(q, fmaf(-q, y, x));
}
AE_DEVICE float ae_mul_odd(float x, float y) {
  const float p = __fmul_rz(x, y);
  return ae_sticky(p, fmaf(x, y, -p));
}

AE_DEVICE u32 ae_max2(u32 a, u32 b) {  // of two unsigned halves each
  u32 r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The largest of all threads' x.
AE_DEVICE u32 ae_block_max(u32 x, u32* red) {
  x = __reduce_max_sync(0xffffffffu, x);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < AE_W_THREADS / 32; ++i) x = x > red[i] ? x : red[i];
  return x;
}

// The values of a segment by a scale that is not a power of two: a page that goes on may have come with one, which it keeps while it is the coarser
// one.  Rare, so in a loop of its own over values read once more; unrolled into the loop below the divisions made the writes of a step 2 us slower.
template <int BF16, int D>
__device__ __noinline__ void ae_write_divided(const AeCache8WriteArgs& a, const AePageSegment seg, int h, int which, float s) {
  const u16* const x = (const u16*)a.x[which] + (i64)h * a.x_sh[which];
  u8* const codes = a.codes[which] + (i64)seg.page * a.c_sp[which] + (i64)h * a.c_sh[which];
#pragma unroll 1
  for (int c = (int)threadIdx.x; c < seg.tokens * (D / 2); c += AE_W_THREADS) {
    const int row = c / (D / 2), col = c % (D / 2) * 2;
    const u32 u = *(const u32*)(x + (i64)(seg.token + row) * a.x_st[which] + col);
    const float v[2] = {unpack_lo<BF16>(u), unpack_hi<BF16>(u)};
    u32 r = ae_e4m3x2(ae_div_odd(v[0], s), ae_div_odd(v[1], s));
    if (fabsf(v[0]) == __int_as_float(0x7f800000)) r |= 0x7fu;  // the conversion saturates; an infinity is to be NaN
    if (fabsf(v[1]) == __int_as_float(0x7f800000)) r |= 0x7f00u;
    *(u16*)(codes + (i64)(seg.slot + row) * a.c_st[which] + col) = (u16)r;
  }
}

template <int BF16, int D>
AE_DEVICE void ae_write_part(const AeCache8WriteArgs& a, const AePageSegment seg, int h, int which, u32* red) {
  constexpr int CPR = D / 8;  // chunks of a row
  constexpr u32 INF = BF16 ? 0x7f80u : 0x7c00u;
  const u16* const x = (const u16*)a.x[which] + (i64)h * a.x_sh[which];
  u8* const codes = a.codes[which] + (i64)seg.page * a.c_sp[which] + (i64)h * a.c_sh[which];
  float* const scale = a.scales[which] + (i64)seg.page * a.s_sp[which] + h;
  // a thread's chunks lie RPI rows apart, in the same column
  constexpr int RPI = AE_W_THREADS / CPR;
  static_assert(AE_W_THREADS % CPR == 0, "whole rows");
  const int row = (int)threadIdx.x / CPR, col = (int)threadIdx.x % CPR * 8, n = seg.tokens - row;  // chunk i is there if i RPI < n
  const u16* src = x + (i64)(seg.token + row) * a.x_st[which] + col;
  const i64 src_step = (i64)RPI * a.x_st[which];
  uint4 w[AE_W_PER];
#pragma unroll
  for (int i = 0; i < AE_W_PER; ++i) {
    w[i] = make_uint4(0, 0, 0, 0);
    if (i * RPI < n) w[i] = *(const uint4*)src;
    src += src_step;
  }
  const float before = *scale;
  u32 top = 0;
#pragma unroll
  for (int i = 0; i < AE_W_PER; ++i)
    top = ae_max2(ae_max2(top, ae_max2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu)), ae_max2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
  top = ae_block_max(top >> 16 > (top & 0xffffu) ? top >> 16 : top & 0xffffu, red);  // also: every thread has read `before`
  const bool special = top >= INF;
  if (special) {  // an infinity or a NaN: the largest of the others
    auto finite = [](u32 u) { return u < INF ? u : 0u; };
    top = 0;
#pragma unroll
    for (int i = 0; i < AE_W_PER; ++i) {
      const u32 u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32 lo = finite(u[k] & 0x7fffu), hi = finite(u[k] >> 16 & 0x7fffu);
        top = top > lo ? top : lo;
        top = top > hi ? top : hi;
      }
    }
    __syncthreads();  // `red` has been read
    top = ae_block_max(top, red);
  }
  float s = ae_pow2_scale(unpack_lo<BF16>(top));
  if (seg.slot > 0) {
    s = fmaxf(s, before);
    if (s != before) {  // the page goes on at a coarser scale
      const float f = before / s;
      for (int c = (int)threadIdx.x; c < seg.slot * CPR; c += AE_W_THREADS) {
        uint2* const at = (uint2*)(codes + (i64)(c / CPR) * a.c_st[which] + (c % CPR) * 8);
        const uint2 u = *at;
        u32 r[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const u32 v = k ? u.y : u.x;
          float e0, e1, e2, e3;
          ae_from_e4m3x2(v & 0xffffu, e0, e1);
          ae_from_e4m3x2(v >> 16, e2, e3);
          r[k] = ae_e4m3x2(ae_mul_odd(e0, f), ae_mul_odd(e1, f)) | ae_e4m3x2(ae_mul_odd(e2, f), ae_mul_odd(e3, f)) << 16;
        }
        *at = make_uint2(r[0], r[1]);
      }
    } else if (__float_as_uint(s) & 0x7fffffu) {
      ae_write_divided<BF16, D>(a, seg, h, which, s);
      return;  // *scale stays
    }
  }
  const float inv = 1.f / s;  // a power of two
  u8* dst = codes + (i64)(seg.slot + row) * a.c_st[which] + col;
  const i64 dst_step = (i64)RPI * a.c_st[which];
  // fp16 is scaled as it is where the factor is one of fp16's normal numbers: exact down to 2^-14, and what is smaller is the code 0
  const bool halves = !BF16 && !special && inv <= 32768.f && inv >= 6.103515625e-5f;
  if (halves) {
    const u32 inv2 = pack2<0>(inv, inv);
#pragma unroll
    for (int i = 0; i < AE_W_PER; ++i) {
      if (i * RPI < n)
        *(uint2*)dst = make_uint2(ae_e4m3x2_half(w[i].x, inv2) | ae_e4m3x2_half(w[i].y, inv2) << 16,
                                  ae_e4m3x2_half(w[i].z, inv2) | ae_e4m3x2_half(w[i].w, inv2) << 16);
      dst += dst_step;
    }
  } else {
#pragma unroll
    for (int i = 0; i < AE_W_PER; ++i) {
      const u32 u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      u32 r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        r[k] = ae_e4m3x2(unpack_lo<BF16>(u[k]) * inv, unpack_hi<BF16>(u[k]) * inv);
        if (special) {  // the conversion saturates; an infinity is to be NaN
          if ((u[k] & 0x7fffu) == INF) r[k] |= 0x7fu;
          if ((u[k] >> 16 & 0x7fffu) == INF) r[k] |= 0x7f00u;
        }
      }
      if (i * RPI < n) *(uint2*)dst = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
      dst += dst_step;
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

#define AE_W_CTAS (8 * 128 / AE_W_THREADS)  // 64 registers a thread (pages of 128: 18.9 us, 20.0 with 85)
extern "C" __global__ void __launch_bounds__(AE_W_THREADS, AE_W_CTAS) ae_cache8_write(const __grid_constant__ AeCache8WriteArgs a) {
  __shared__ u32 red[AE_W_THREADS / 32];
  ae_grid_wait();  // brought up under the kernel in front
  ae_grid_trigger();
  const AePageSegment seg = a.segments[blockIdx.x / a.H];
  // a segment without tokens, or one that a caller made up outside the pool or the tokens: nothing is written
  if (seg.tokens <= 0 || seg.page < 0 || seg.page >= a.num_pages || seg.slot < 0 || seg.slot >= AE_PAGE || seg.tokens > AE_PAGE - seg.slot || seg.token < 0 ||
      seg.token > a.n_tokens - seg.tokens)
    return;
  const int h = blockIdx.x % a.H;
  if (blockIdx.y == 0) {
    if (a.bf16)
      ae_write_part<1, AE_D>(a, seg, h, 0, red);
    else
      ae_write_part<0, AE_D>(a, seg, h, 0, red);
  } else {
    if (a.bf16)
      ae_write_part<1, AE_DV>(a, seg, h, 1, red);
    else
      ae_write_part<0, AE_DV>(a, seg, h, 1, red);
  }
}
