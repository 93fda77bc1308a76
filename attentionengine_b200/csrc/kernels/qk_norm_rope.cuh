// Norm of each query and key head and its rotation by the token's position, forward and backward, one pass over the data.
//
// With x one head's D values, w a weight, f_i the frequency of pair i and p the position:
//   n = x (mean(x^2) + eps)^-1/2,  z = n w,  y_a = m (z_a cos(p f_i) - z_b sin(p f_i)),  y_b = m (z_b cos(p f_i) + z_a sin(p f_i))
// for the pairs (a, b) = (i, i + R / 2), or (2i, 2i + 1); the D - R values behind are z.  Backward, from the gradient g of y:
//   dz_a = m (g_a cos + g_b sin),  dz_b = m (g_b cos - g_a sin),  dw = sum over tokens and heads of dz n,
//   dx = (mean(x^2) + eps)^-1/2 (dz w - n mean(dz w n)).
// Angles: p f / 2 pi is wanted modulo 1, so a frequency is held as its 64-bit fraction of a turn and the product wraps around by itself: exact for any
// position, where an fp32 angle is off by 0.03 at position 500000.
//
// A team of D / 16 threads has a head, each thread 16 values that hold both halves of its 8 pairs, so that the rotation needs no exchange and the norm
// log2(D / 16) shuffles.  A warp has a token and a share of its heads: cosines and sines are made once for them (two pairs a lane, through shared
// memory) and folded with the weights into four factors a pair.  Bound by HBM for long calls: everything is read and written once.
// Expects AE_D (32, 64, 128 or 256), AE_R (rotary dims, a multiple of 16), AE_NORM, AE_NEXT (pairs of neighbours), AE_ROPE_WARPS, AE_ROPE_U (heads
// of a team on their way together), AE_ROPE_KERNEL (0 forward, 1 backward, 2 the weights' sums).
#define AE_TPR (AE_D / 16)      // threads of a team
#define AE_TEAMS (32 / AE_TPR)  // teams of a warp
#define AE_ROPE_THREADS (32 * AE_ROPE_WARPS)
#define AE_PAIRS (AE_R / 2)
#define AE_PAIRS1 (AE_PAIRS > 0 ? AE_PAIRS : 1)

// cos and sin of the turns that position p makes.
AE_DEVICE float2 ae_turn(u64 per_position, i64 p) {
  const float half_turns = (float)(int)((u64)p * per_position >> 32) * 4.656612873077393e-10f;  // 2^-31
  float2 r;
  sincospif(half_turns, &r.y, &r.x);
  return r;
}

// First value of the two chunks of 8 that thread t of a team has.
AE_DEVICE int ae_chunk(int t, int second) {
#if AE_NEXT
  return 16 * t + 8 * second;
#else
  return t < AE_R / 16 ? 8 * t + second * (AE_R / 2) : AE_R + 16 * (t - AE_R / 16) + 8 * second;
#endif
}
// Where of a thread's 16 values pair e has its first and second.
AE_DEVICE constexpr int ae_first(int e) { return AE_NEXT ? 2 * e : e; }
AE_DEVICE constexpr int ae_second(int e) { return AE_NEXT ? 2 * e + 1 : e + 8; }

template <int BF16>
AE_DEVICE void ae_unpack16(const uint4 (&v)[2], float (&x)[16]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const u32 u[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[8 * c + 2 * k] = unpack_lo<BF16>(u[k]);
      x[8 * c + 2 * k + 1] = unpack_hi<BF16>(u[k]);
    }
  }
}
template <int BF16>
AE_DEVICE uint4 ae_pack8(const float* x) {
  return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
}

AE_DEVICE float ae_team_sum(float x) {
#pragma unroll
  for (int o = 1; o < AE_TPR; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// The weights of a thread's 16 values.
AE_DEVICE void ae_load_weights(const AeQkRopeArgs& a, int kind, int t, float (&w)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = 1.f;
  if (!a.w[kind]) return;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int at = ae_chunk(t, c);
    if (a.w32) {
      const float4* const p = (const float4*)((const float*)a.w[kind] + at);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 u = p[j];
        w[8 * c + 4 * j] = u.x;
        w[8 * c + 4 * j + 1] = u.y;
        w[8 * c + 4 * j + 2] = u.z;
        w[8 * c + 4 * j + 3] = u.w;
      }
    } else {
      const uint4 v = *(const uint4*)((const u16*)a.w[kind] + at);
      const u32 u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[8 * c + 2 * j] = a.bf16 ? unpack_lo<1>(u[j]) : unpack_lo<0>(u[j]);
        w[8 * c + 2 * j + 1] = a.bf16 ? unpack_hi<1>(u[j]) : unpack_hi<0>(u[j]);
      }
    }
  }
}

struct AeRopeSmem {
  u64 turns[AE_PAIRS1];
  float2 cs[AE_ROPE_WARPS][AE_PAIRS1];
#if AE_ROPE_KERNEL == 1 && AE_NORM
  float dw[AE_ROPE_WARPS][AE_D];
#endif
};

AE_DEVICE i64 ae_position(const AeQkRopeArgs& a, int b, int s) {
  const i64 at = b * a.pos_st[0] + s * a.pos_st[1];
  return a.pos64 ? ((const i64*)a.pos)[at] : (i64)((const int*)a.pos)[at];
}

// cos and sin times m of a thread's pairs, made by the warp together.
AE_DEVICE void ae_cos_sin(const AeQkRopeArgs& a, AeRopeSmem& sm, i64 p, int t, float (&c)[8], float (&s)[8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncwarp();  // the pairs of the item in front have been read
#pragma unroll
  for (int i = 0; i < (AE_PAIRS + 31) / 32; ++i)
    if (i * 32 + lane < AE_PAIRS) {
      const float2 r = ae_turn(sm.turns[i * 32 + lane], p);
      sm.cs[warp][i * 32 + lane] = make_float2(r.x * a.scale, r.y * a.scale);
    }
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float2 r = make_float2(1.f, 0.f);
    if (t < AE_R / 16) r = sm.cs[warp][8 * t + e];
    c[e] = r.x;
    s[e] = r.y;
  }
}

AE_DEVICE void ae_load_turns(const AeQkRopeArgs& a, AeRopeSmem& sm) {
  for (int i = threadIdx.x; i < AE_PAIRS; i += AE_ROPE_THREADS) sm.turns[i] = a.turns[i];
  __syncthreads();
}

#if AE_ROPE_KERNEL == 0

// Heads h0 ... h1 - 1 of a token, by a warp.
template <int BF16>
AE_DEVICE void ae_rope_heads(const AeQkRopeArgs& a, AeRopeSmem& sm, int kind, int token, int h0, int h1) {
  const int lane = threadIdx.x & 31, t = lane % AE_TPR, team = lane / AE_TPR;
  const int b = token / a.S, s = token - b * a.S;
  const u16* const x = (const u16*)a.x[kind] + b * a.x_st[kind][0] + s * a.x_st[kind][1];
  u16* const y = (u16*)a.y[kind] + (i64)token * a.H[kind] * AE_D;
  const int at[2] = {ae_chunk(t, 0), ae_chunk(t, 1)};
  const i64 p = ae_position(a, b, s);
  if (p < 0) {  // no token
    for (int h = h0 + team; h < h1; h += AE_TEAMS)
#pragma unroll
      for (int c = 0; c < 2; ++c) *(uint4*)(y + h * AE_D + at[c]) = make_uint4(0, 0, 0, 0);
    return;
  }
  uint4 v[AE_ROPE_U][2];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < AE_ROPE_U; ++u) {
      const int h = base + u * AE_TEAMS + team;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        v[u][c] = make_uint4(0, 0, 0, 0);
        if (h < h1) v[u][c] = *(const uint4*)(x + h * a.x_st[kind][2] + at[c]);
      }
    }
  };
  load(h0);
  // y_a = rstd (x_a fa[0] - x_b fb[0]), y_b = rstd (x_b fb[1] + x_a fa[1])
  float fa[2][8], fb[2][8];
  {
    float c[8], sn[8], w[16];
    ae_cos_sin(a, sm, p, t, c, sn);
    ae_load_weights(a, kind, t, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      fa[0][e] = c[e] * w[ae_first(e)];
      fa[1][e] = sn[e] * w[ae_first(e)];
      fb[0][e] = sn[e] * w[ae_second(e)];
      fb[1][e] = c[e] * w[ae_second(e)];
    }
  }
  for (int base = h0;;) {
#pragma unroll
    for (int u = 0; u < AE_ROPE_U; ++u) {
      float f[16], o[16];
      ae_unpack16<BF16>(v[u], f);
      float r = 1.f;
#if AE_NORM
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) sum = fmaf(f[j], f[j], sum);
      r = rsqrtf(fmaf(ae_team_sum(sum), 1.f / AE_D, a.eps));
#endif
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xa = f[ae_first(e)], xb = f[ae_second(e)];
        o[ae_first(e)] = r * fmaf(xa, fa[0][e], -(xb * fb[0][e]));
        o[ae_second(e)] = r * fmaf(xb, fb[1][e], xa * fa[1][e]);
      }
      const int h = base + u * AE_TEAMS + team;
      if (h < h1)
#pragma unroll
        for (int c = 0; c < 2; ++c) *(uint4*)(y + h * AE_D + at[c]) = ae_pack8<BF16>(o + 8 * c);
    }
    base += AE_ROPE_U * AE_TEAMS;
    if (base >= h1) break;
    load(base);
  }
}

extern "C" __global__ void __launch_bounds__(AE_ROPE_THREADS) ae_qk_rope_fwd(const __grid_constant__ AeQkRopeArgs a) {
  __shared__ AeRopeSmem sm;
  ae_load_turns(a, sm);
  ae_grid_wait();  // brought up under the kernel in front
  ae_grid_trigger();
  const int slices = a.slices[0] + a.slices[1];
  const int item = blockIdx.x * AE_ROPE_WARPS + (threadIdx.x >> 5);
  const int token = item / slices;
  if (token >= a.T) return;
  int slice = item - token * slices;
  const int kind = slice >= a.slices[0];
  if (kind) slice -= a.slices[0];
  const int h0 = slice * a.per, h1 = min(h0 + a.per, a.H[kind]);
  if (a.bf16)
    ae_rope_heads<1>(a, sm, kind, token, h0, h1);
  else
    ae_rope_heads<0>(a, sm, kind, token, h0, h1);
}

#elif AE_ROPE_KERNEL == 1

// A CTA works on queries alone or keys alone, so that its threads keep one set of weight sums.  They are joined in a fixed order: teams, warps,
// and by ae_qk_rope_dw CTAs; results do not vary.
template <int BF16>
AE_DEVICE void ae_rope_bwd_heads(const AeQkRopeArgs& a, AeRopeSmem& sm, int kind, const float (&w)[16], float (&dw)[16], int token, int h0, int h1) {
  const int lane = threadIdx.x & 31, t = lane % AE_TPR, team = lane / AE_TPR;
  const int b = token / a.S, s = token - b * a.S;
  const u16* const x = (const u16*)a.x[kind] + b * a.x_st[kind][0] + s * a.x_st[kind][1];
  const u16* const g = (const u16*)a.g[kind] + b * a.g_st[kind][0] + s * a.g_st[kind][1];
  u16* const y = (u16*)a.y[kind] + (i64)token * a.H[kind] * AE_D;
  const int at[2] = {ae_chunk(t, 0), ae_chunk(t, 1)};
  const i64 p = ae_position(a, b, s);
  if (p < 0) {
    for (int h = h0 + team; h < h1; h += AE_TEAMS)
#pragma unroll
      for (int c = 0; c < 2; ++c) *(uint4*)(y + h * AE_D + at[c]) = make_uint4(0, 0, 0, 0);
    return;
  }
  uint4 v[AE_ROPE_U][2], gv[AE_ROPE_U][2];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < AE_ROPE_U; ++u) {
      const int h = base + u * AE_TEAMS + team;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        v[u][c] = gv[u][c] = make_uint4(0, 0, 0, 0);
        if (h < h1) {
#if AE_NORM
          v[u][c] = *(const uint4*)(x + h * a.x_st[kind][2] + at[c]);
#endif
          gv[u][c] = *(const uint4*)(g + h * a.g_st[kind][2] + at[c]);
        }
      }
    }
  };
  load(h0);
  float c[8], sn[8];
  ae_cos_sin(a, sm, p, t, c, sn);
  for (int base = h0;;) {
#pragma unroll
    for (int u = 0; u < AE_ROPE_U; ++u) {
      float gf[16], dz[16];
      ae_unpack16<BF16>(gv[u], gf);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ga = gf[ae_first(e)], gb = gf[ae_second(e)];
        dz[ae_first(e)] = fmaf(ga, c[e], gb * sn[e]);
        dz[ae_second(e)] = fmaf(gb, c[e], -(ga * sn[e]));
      }
#if AE_NORM
      float f[16], sum = 0.f, dot = 0.f;  // of x^2, of x dz w
      ae_unpack16<BF16>(v[u], f);
#pragma unroll
      for (int j = 0; j < 16; ++j) sum = fmaf(f[j], f[j], sum);
      float r = rsqrtf(fmaf(ae_team_sum(sum), 1.f / AE_D, a.eps));
      if (base + u * AE_TEAMS + team >= h1) r = 0.f;  // no head: with eps = 0 its zeros would make the sums NaN
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        f[j] *= r;  // n
        dw[j] = fmaf(dz[j], f[j], dw[j]);
        dz[j] *= w[j];
        dot = fmaf(dz[j], f[j], dot);
      }
      const float mean = ae_team_sum(dot) * (1.f / AE_D);
#pragma unroll
      for (int j = 0; j < 16; ++j) dz[j] = r * fmaf(-f[j], mean, dz[j]);
#endif
      const int h = base + u * AE_TEAMS + team;
      if (h < h1)
#pragma unroll
        for (int k = 0; k < 2; ++k) *(uint4*)(y + h * AE_D + at[k]) = ae_pack8<BF16>(dz + 8 * k);
    }
    base += AE_ROPE_U * AE_TEAMS;
    if (base >= h1) break;
    load(base);
  }
}

template <int BF16>
AE_DEVICE void ae_rope_bwd(const AeQkRopeArgs& a, AeRopeSmem& sm) {
  const int kind = (int)blockIdx.x >= a.ctas[0], cta = (int)blockIdx.x - kind * a.ctas[0];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane % AE_TPR;
  float w[16], dw[16];
  ae_load_weights(a, kind, t, w);
#pragma unroll
  for (int j = 0; j < 16; ++j) dw[j] = 0.f;
  const i64 items = (i64)a.T * a.slices[kind];
  for (i64 item = (i64)cta * AE_ROPE_WARPS + warp; item < items; item += (i64)a.ctas[kind] * AE_ROPE_WARPS) {
    const int token = (int)(item / a.slices[kind]), h0 = (int)(item - (i64)token * a.slices[kind]) * a.per;
    ae_rope_bwd_heads<BF16>(a, sm, kind, w, dw, token, h0, min(h0 + a.per, a.H[kind]));
  }
#if AE_NORM
  if (!a.dw_part) return;
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int o = AE_TPR; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
  if (lane < AE_TPR)
#pragma unroll
    for (int j = 0; j < 16; ++j) sm.dw[warp][ae_chunk(t, j >> 3) + (j & 7)] = dw[j];
  __syncthreads();
  for (int d = threadIdx.x; d < AE_D; d += AE_ROPE_THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < AE_ROPE_WARPS; ++i) sum += sm.dw[i][d];
    a.dw_part[(i64)blockIdx.x * AE_D + d] = sum;
  }
#endif
}

extern "C" __global__ void __launch_bounds__(AE_ROPE_THREADS, AE_ROPE_CTAS) ae_qk_rope_bwd(const __grid_constant__ AeQkRopeArgs a) {
  __shared__ AeRopeSmem sm;
  ae_load_turns(a, sm);
  ae_grid_wait();
  ae_grid_trigger();
  if (a.bf16)
    ae_rope_bwd<1>(a, sm);
  else
    ae_rope_bwd<0>(a, sm);
}

#else

// The weights' gradients: a CTA sums 32 dims of the CTAs' rows, for queries or keys.
extern "C" __global__ void __launch_bounds__(AE_ROPE_THREADS) ae_qk_rope_dw(const __grid_constant__ AeQkRopeArgs a) {
  __shared__ float sm[AE_ROPE_WARPS][32];
  ae_grid_wait();
  ae_grid_trigger();
  const int kind = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane;
  const float* const part = a.dw_part + (i64)(kind ? a.ctas[0] : 0) * AE_D + d;
  float sum = 0.f;
#pragma unroll 8
  for (int i = warp; i < a.ctas[kind]; i += AE_ROPE_WARPS) sum += part[(i64)i * AE_D];
  sm[warp][lane] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < AE_ROPE_WARPS; ++i) sum += sm[i][lane];
    if (a.w32)
      ((float*)a.dw[kind])[d] = sum;
    else
      ((u16*)a.dw[kind])[d] = (u16)(a.bf16 ? pack2<1>(sum, sum) : pack2<0>(sum, sum));
  }
}
#endif
