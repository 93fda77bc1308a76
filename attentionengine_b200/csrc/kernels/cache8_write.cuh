// Write of new keys and values into a paged cache of 8-bit floating point (e4m3), a scale for each page and head.
//
// The scale is the smallest power of two s with amax / s <= 448 (the largest e4m3 value), at least 2^-64; codes are x / s rounded to
// nearest even.  A power of two, because e4m3 is a floating-point format: any scale gives the same relative precision, and with this
// one x / s is exact, so the only rounding is the one to e4m3; and when a page that goes on needs a coarser scale, the codes that are there are
// multiplied by a power of two, which changes none of them but at the bottom of the range.  amax takes the finite values: an infinity or a
// NaN becomes NaN and does not take the others' precision.
//
// One CTA per (segment, head, K or V) owns the page's part for that head, so there is nothing to lock.  A page is at most 128 x 128 values: the
// CTA holds its 16-bit values in registers between the maximum and the rounding, one pass over the data.  Bound by HBM (2 bytes in and 1 out
// a value), for a step of single tokens by latency.
// Expects AE_PAGE, AE_D, AE_DV, AE_W_THREADS.

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
// Two values to e4m3, `lo` in the low byte.  The conversion saturates; only an infinity can, and it is made NaN.
AE_DEVICE u32 ae_e4m3x2(float lo, float hi) {
  u16 r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  u32 w = r;
  if (fabsf(lo) == __int_as_float(0x7f800000)) w |= 0x7fu;
  if (fabsf(hi) == __int_as_float(0x7f800000)) w |= 0x7f00u;
  return w;
}
AE_DEVICE void ae_from_e4m3x2(u32 w, float& lo, float& hi) {
  u32 h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((u16)w));
  lo = unpack_lo<0>(h);
  hi = unpack_hi<0>(h);
}

template <int BF16, int D>
AE_DEVICE void ae_write_part(const AeCache8WriteArgs& a, const AePageSegment seg, int h, int which, float* red) {
  constexpr int CPR = D / 8;  // chunks of a row
  const u16* const x = (const u16*)a.x[which] + (i64)h * a.x_sh[which];
  u8* const codes = a.codes[which] + (i64)seg.page * a.c_sp[which] + (i64)h * a.c_sh[which];
  float* const scale = a.scales[which] + (i64)seg.page * a.s_sp[which] + h;
  const int n = seg.tokens * CPR;
  uint4 w[AE_W_PER];
  float amax = 0.f;
  auto finite = [](float f) { return fabsf(f) < __int_as_float(0x7f800000) ? fabsf(f) : 0.f; };
#pragma unroll
  for (int i = 0; i < AE_W_PER; ++i) {
    const int c = i * AE_W_THREADS + (int)threadIdx.x;
    w[i] = make_uint4(0, 0, 0, 0);
    if (c < n) w[i] = *(const uint4*)(x + (i64)(seg.token + c / CPR) * a.x_st[which] + (c % CPR) * 8);
  }
  const float before = *scale;
#pragma unroll
  for (int i = 0; i < AE_W_PER; ++i) {
    const u32 u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(finite(unpack_lo<BF16>(u[k])), finite(unpack_hi<BF16>(u[k]))));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();  // also: every thread has read `before`
#pragma unroll
  for (int i = 0; i < AE_W_THREADS / 32; ++i) amax = fmaxf(amax, red[i]);
  float s = ae_pow2_scale(amax);
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
          r[k] = ae_e4m3x2(e0 * f, e1 * f) | ae_e4m3x2(e2 * f, e3 * f) << 16;
        }
        *at = make_uint2(r[0], r[1]);
      }
    }
  }
  const float inv = 1.f / s;  // a power of two
#pragma unroll
  for (int i = 0; i < AE_W_PER; ++i) {
    const int c = i * AE_W_THREADS + (int)threadIdx.x;
    if (c >= n) continue;
    const u32 u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
    u32 r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = ae_e4m3x2(unpack_lo<BF16>(u[k]) * inv, unpack_hi<BF16>(u[k]) * inv);
    *(uint2*)(codes + (i64)(seg.slot + c / CPR) * a.c_st[which] + (c % CPR) * 8) = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
  }
  if (threadIdx.x == 0) *scale = s;
}

extern "C" __global__ void __launch_bounds__(AE_W_THREADS) ae_cache8_write(const __grid_constant__ AeCache8WriteArgs a) {
  __shared__ float red[AE_W_THREADS / 32];
  const AePageSegment seg = a.segments[blockIdx.x];
  // a segment without tokens, or one that a caller made up outside the pool or the tokens: nothing is written
  if (seg.tokens <= 0 || seg.page < 0 || seg.page >= a.num_pages || seg.slot < 0 || seg.slot >= AE_PAGE || seg.tokens > AE_PAGE - seg.slot || seg.token < 0 ||
      seg.token > a.n_tokens - seg.tokens)
    return;
  const int h = blockIdx.y;
  if (blockIdx.z == 0) {
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
