// Norm of each query and key head and its rotation by the token's position, forward and backward, one pass over the data.
//
// With x one head's D values, w a weight, f_i the frequency of pair i and p the position:
//   n = x (mean(x^2) + eps)^-1/2,  z = n w,  y_a = m (z_a cos(p f_i) - z_b sin(p f_i)),  y_b = m (z_b cos(p f_i) + z_a sin(p f_i))
// for the pairs (a, b) = (i, i + R / 2), or (2i, 2i + 1); the D - R values behind are z.  Backward, from the gradient g of y:
//   dz_a = m (g_a cos + g_b sin),  dz_b = m (g_b cos - g_a sin),  dw = sum over tokens and heads of dz n,
//   dx = (mean(x^2) + eps)^-1/2 (dz w - n mean(dz w n)).
// Angles: p f / 2 pi is wanted modulo 1, so a frequency is held as its 64-bit fraction of a turn and the product wraps around by itself.  That is off by
// p 2^-65 of a turn (the frequency's rounding), and by 2^-26 of one for the angle's fp32, which is the larger part up to p = 2^39; beyond, 64-bit positions lose
// their angle bit by bit (an eighth of a turn at 2^62).  An fp32 product is off by 0.03 radians at position 500000.
//
// A team of D / 16 threads has a head, each thread 16 values that hold both halves of its 8 pairs, so that the rotation needs no exchange and the norm
// log2(D / 16) shuffles.  A warp has a token, or where tokens are few a share of its heads: its lanes make the token's cosines and sines once and fold
// them (forward: with the weights) into two factors a value, which pass through shared memory.  Arithmetic on two fp32 values an instruction.
//
// Bound by HBM for long calls: everything is read and written once.  What that takes is bytes on their way, and a warp has four chains of reads in a row
// (position, two batches of queries, keys): the forward asks L2 for a token's heads before anything else.  In a graph, 40 heads of 128 dims, bf16: 11542 tokens (236 MB) 39.3 us,
// 6.0 TB/s (42.9 without that request; 44 to 45 with the factors made by every team for itself; 79 with factors at 64-byte steps, four-fold bank conflicts;
// 84 with whole CTAs a token, whose barriers leave nothing on its way); forward and backward of 16384 tokens (839 MB) 145 us.  64 tokens, one a request: 2.6.
// The backward is joined work of 24 warps an SM with one head a team on its way (80 registers): 88 us, 5.7 TB/s; a ring of copies through shared memory, two heads on their
// way, or requests to L2 ahead took 1 to 30 % more.
// Expects AE_D (32, 64, 128 or 256), AE_R (rotary dims, a multiple of 16), AE_NORM, AE_NEXT (pairs of neighbours), AE_ROPE_WARPS, AE_ROPE_U (backward: heads
// of a team on their way together), AE_ROPE_CTAS (of an SM), AE_ROPE_KERNEL (0 forward, 1 backward, 2 the weights' sums).
#define AE_ROPE_THREADS (32 * AE_ROPE_WARPS)
#define AE_TPR (AE_D / 16)      // threads of a team
#define AE_TEAMS (32 / AE_TPR)  // teams of a warp
#define AE_PAIRS (AE_R / 2)
// The forward's products come before the norm's factor.  That is 0 for values whose squares' sum is infinite, and must find them finite: so a power of two
// goes from the factors of the values to the norm's, room for weights times rotary_scale up to 180.
#define AE_ROOM (AE_NORM ? 256.f : 1.f)

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
// Two fp32 values in a register pair.
AE_DEVICE u64 ae_mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
AE_DEVICE u64 ae_fma22(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
AE_DEVICE float ae_sum2(u64 a) {
  float lo, hi;
  ae_unpack2f(a, lo, hi);
  return lo + hi;
}

// A thread's 16 values as 8 pairs of neighbours.
template <int BF16>
AE_DEVICE void ae_unpack16(const uint4& lo, const uint4& hi, u64 (&x)[8]) {
  const u32 u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = ae_pack2f(unpack_lo<BF16>(u[k]), unpack_hi<BF16>(u[k]));
}
template <int BF16>
AE_DEVICE uint4 ae_pack8(const u64* x) {
  u32 r[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float lo, hi;
    ae_unpack2f(x[k], lo, hi);
    r[k] = pack2<BF16>(lo, hi);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// What the rotation mixes with pair k: the values of the other half, or the same two the other way round.
AE_DEVICE u64 ae_partner(const u64 (&x)[8], int k) {
#if AE_NEXT
  float lo, hi;
  ae_unpack2f(x[k], lo, hi);
  return ae_pack2f(hi, lo);
#else
  return x[k ^ 4];
#endif
}
// Whether thread t's values are rotated ones; the others must not meet their partners, not even times 0 (an infinity would make them NaN).
AE_DEVICE bool ae_rotates(int t) { return AE_R == AE_D || t < AE_R / 16; }

AE_DEVICE float ae_team_sum(float x) {
#pragma unroll
  for (int o = 1; o < AE_TPR; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

#if AE_ROPE_KERNEL < 2

#define AE_KINDS (AE_ROPE_KERNEL == 0 ? 2 : 1)
// Factors of each value and of its partner, as the threads read them (ae_place).
struct AeRopeSmem {
  float f[AE_ROPE_WARPS][AE_KINDS][2][AE_D];  // forward: with the weights; backward: cos and sin
  float w[AE_KINDS][AE_D];  // weights, in that order too
  u64 turns[AE_PAIRS];
#if AE_ROPE_KERNEL == 1 && AE_NORM
  float dw[AE_ROPE_WARPS][AE_D];
#endif
};

// Place of dim d among the threads' values (ae_chunk the other way round): four values of every thread behind each other, so that a warp's wide loads
// meet every bank once.
AE_DEVICE int ae_place(int d) {
#if AE_NEXT
  const int t = d >> 4, j = d & 15;
#else
  const int second = d >= AE_R / 2, i = d - second * (AE_R / 2);
  const int t = d < AE_R ? i >> 3 : d >> 4, j = d < AE_R ? 8 * second + (i & 7) : d & 15;
#endif
  return ((j >> 2) * AE_TPR + t) * 4 + (j & 3);
}

AE_DEVICE float ae_weight(const AeQkRopeArgs& a, int kind, int d) {
  if (!a.w[kind]) return 1.f;
  if (a.w32) return ((const float*)a.w[kind])[d];
  const u32 u = ((const u16*)a.w[kind])[d];
  return a.bf16 ? unpack_lo<1>(u) : unpack_lo<0>(u);
}

struct AeRopeToken {
  int b, s;
  AE_DEVICE AeRopeToken(const AeQkRopeArgs& a, int token) : b(0), s(token) {
    if (a.S < a.T) b = token / a.S, s = token - b * a.S;
  }
  AE_DEVICE i64 position(const AeQkRopeArgs& a) const {
    const i64 at = b * a.pos_st[0] + s * a.pos_st[1];
    return a.pos64 ? ((const i64*)a.pos)[at] : (i64)((const int*)a.pos)[at];
  }
  AE_DEVICE const u16* heads(const void* x, const i64 (&st)[3]) const { return (const u16*)x + b * st[0] + s * st[1]; }
};

// Thread t's 16 values, or the first 8.
template <int N>
AE_DEVICE void ae_read(const float* f, int t, u64 (&x)[N]) {
  const u32 at = smem_u32(f) + 16 * t;
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(x[2 * i]), "=l"(x[2 * i + 1]) : "r"(at + 16 * AE_TPR * i) : "memory");
}

#endif
#if AE_ROPE_KERNEL == 0

// n heads on their way into L2, by a warp: what registers have no room for yet.
AE_DEVICE void ae_prefetch_heads(const u16* x, i64 st, int n) {
  const bool run = st == AE_D;  // heads behind each other go in pieces of 8 KB
  const int each = run ? 8192 / (2 * AE_D) : 1;
  for (int h = (threadIdx.x & 31) * each; h < n; h += 32 * each)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(x + h * st), "r"(min(each, n - h) * AE_D * 2) : "memory");
}

// U heads of each team from h on: y = x f0 + partner(x) f1 times the norm's factor; f1 holds the partner's weight.
template <int BF16, int U>
AE_DEVICE void ae_rope_batch(const AeQkRopeArgs& a, const u64 (&f)[2][8], bool rotates, const u16* x, u16* y, i64 st, const int (&at)[2], int h, int end) {
  uint4 v[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {  // a team without a head reads the last one's values, which nothing takes
    const i64 hh = min(h + u * AE_TEAMS, end - 1);
#pragma unroll
    for (int c = 0; c < 2; ++c) v[u][c] = *(const uint4*)(x + hh * st + at[c]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    u64 z[8], o[8];
    ae_unpack16<BF16>(v[u][0], v[u][1], z);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const u64 other = rotates ? ae_partner(z, k) : 0;
      o[k] = ae_fma22(z[k], f[0][k], ae_mul2(other, f[1][k]));
    }
#if AE_NORM
    u64 sum = ae_mul2(z[0], z[0]);
#pragma unroll
    for (int k = 1; k < 8; ++k) sum = ae_fma22(z[k], z[k], sum);
    const float r = rsqrtf(fmaf(ae_team_sum(ae_sum2(sum)), 1.f / AE_D, a.eps)) * AE_ROOM;
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = ae_mul2(o[k], ae_pack2f(r, r));
#endif
    if (h + u * AE_TEAMS < end)
#pragma unroll
      for (int c = 0; c < 2; ++c) __stcs((uint4*)(y + (h + u * AE_TEAMS) * AE_D + at[c]), ae_pack8<BF16>(o + 4 * c));
  }
}

// Heads h0 ... h1 - 1 of a token, queries or keys, by a warp.
template <int BF16>
AE_DEVICE void ae_rope_heads(const AeQkRopeArgs& a, const AeRopeSmem& sm, bool none, int kind, int token, const AeRopeToken& at_token, int h0, int h1) {
  const int lane = threadIdx.x & 31, t = lane % AE_TPR, team = lane / AE_TPR;
  u16* const y = (u16*)a.y[kind] + (i64)token * a.H[kind] * AE_D;
  if (none) {
    for (int i = h0 * (AE_D / 8) + lane; i < h1 * (AE_D / 8); i += 32) ((uint4*)y)[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const u16* const x = at_token.heads(a.x[kind], a.x_st[kind]);
  const i64 st = a.x_st[kind][2];
  const int at[2] = {ae_chunk(t, 0), ae_chunk(t, 1)};
  u64 f[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) ae_read(sm.f[threadIdx.x >> 5][kind][i], t, f[i]);
#pragma unroll 1
  for (; h0 + 2 * AE_TEAMS < h1; h0 += 4 * AE_TEAMS) ae_rope_batch<BF16, 4>(a, f, ae_rotates(t), x, y, st, at, h0 + team, h1);
  if (h0 + AE_TEAMS < h1)
    ae_rope_batch<BF16, 2>(a, f, ae_rotates(t), x, y, st, at, h0 + team, h1);
  else if (h0 < h1)
    ae_rope_batch<BF16, 1>(a, f, ae_rotates(t), x, y, st, at, h0 + team, h1);
}

template <int BF16>
AE_DEVICE void ae_rope_fwd(const AeQkRopeArgs& a, AeRopeSmem& sm) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x * AE_ROPE_WARPS + warp, token = a.slices[0] == 1 ? item : item / a.slices[0];
  // heads of queries, then keys, as one line
  const int c0 = (item - token * a.slices[0]) * a.per, c1 = min(c0 + a.per, a.H[0] + a.H[1]);
  const int q1 = min(c1, a.H[0]), k0 = max(c0 - a.H[0], 0), k1 = c1 - a.H[0];
  const AeRopeToken at(a, token);
  i64 p = -1;
  if (token < a.T) {
    p = at.position(a);
    if (a.prefetch) {
      ae_prefetch_heads(at.heads(a.x[0], a.x_st[0]) + c0 * a.x_st[0][2], a.x_st[0][2], q1 - c0);
      if (k1 > 0) ae_prefetch_heads(at.heads(a.x[1], a.x_st[1]) + k0 * a.x_st[1][2], a.x_st[1][2], k1 - k0);
    }
  }
  for (int i = threadIdx.x; i < 2 * AE_D; i += AE_ROPE_THREADS) {
    const int kind = i / AE_D, d = i % AE_D, place = ae_place(d);
    const float w = ae_weight(a, kind, d) * (1.f / AE_ROOM);
    sm.w[kind][place] = w;
    if (d >= AE_R)
#pragma unroll
      for (int k = 0; k < AE_ROPE_WARPS; ++k) sm.f[k][kind][0][place] = w, sm.f[k][kind][1][place] = 0.f;
  }
  __syncthreads();
  if (token >= a.T) return;
#pragma unroll
  for (int e = lane; e < AE_PAIRS; e += 32) {
    const float2 r = ae_turn(sm.turns[e], p);
    const float c = r.x * a.scale, s = r.y * a.scale;
    const int pa = ae_place(AE_NEXT ? 2 * e : e), pb = ae_place(AE_NEXT ? 2 * e + 1 : e + AE_R / 2);
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const float wa = sm.w[kind][pa], wb = sm.w[kind][pb];
      float(&f)[2][AE_D] = sm.f[warp][kind];
      f[0][pa] = c * wa;
      f[1][pa] = -s * wb;
      f[0][pb] = c * wb;
      f[1][pb] = s * wa;
    }
  }
  __syncwarp();
  if (c0 < q1) ae_rope_heads<BF16>(a, sm, p < 0, 0, token, at, c0, q1);
  if (k0 < k1) ae_rope_heads<BF16>(a, sm, p < 0, 1, token, at, k0, k1);
}

extern "C" __global__ void __launch_bounds__(AE_ROPE_THREADS, AE_ROPE_CTAS) ae_qk_rope_fwd(const __grid_constant__ AeQkRopeArgs a) {
  __shared__ __align__(16) AeRopeSmem sm;
  for (int i = threadIdx.x; i < AE_PAIRS; i += AE_ROPE_THREADS) sm.turns[i] = a.turns[i];
  ae_grid_wait();  // brought up under the kernel in front
  ae_grid_trigger();
  if (a.bf16)
    ae_rope_fwd<1>(a, sm);
  else
    ae_rope_fwd<0>(a, sm);
}

#elif AE_ROPE_KERNEL == 1

// A CTA works on queries alone or keys alone, so that its threads keep one set of weight sums.  They are joined in a fixed order: teams, warps,
// and by ae_qk_rope_dw CTAs; results do not vary.
template <int BF16>
AE_DEVICE void ae_rope_bwd(const AeQkRopeArgs& a, AeRopeSmem& sm) {
  const int kind = (int)blockIdx.x >= a.ctas[0], cta = (int)blockIdx.x - kind * a.ctas[0], H = a.H[kind], slices = a.slices[kind], per = a.per;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane % AE_TPR, team = lane / AE_TPR;
  const int at[2] = {ae_chunk(t, 0), ae_chunk(t, 1)};
  const i64 x_st = a.x_st[kind][2], g_st = a.g_st[kind][2];
  for (int d = threadIdx.x; d < AE_D; d += AE_ROPE_THREADS) sm.w[0][ae_place(d)] = ae_weight(a, kind, d);
  __syncthreads();
  u64 dw2[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) dw2[j] = 0;
  float(&f)[2][AE_D] = sm.f[warp][0];
  const int items = a.T * slices, step = a.ctas[kind] * AE_ROPE_WARPS;
#pragma unroll 1
  for (int item = cta * AE_ROPE_WARPS + warp; item < items; item += step) {
    const int token = slices == 1 ? item : item / slices, h0 = (item - token * slices) * per, h1 = min(h0 + per, H);
    const AeRopeToken here(a, token);
    const i64 p = here.position(a);
    const u16* const g = here.heads(a.g[kind], a.g_st[kind]);
    const u16* const x = AE_NORM ? here.heads(a.x[kind], a.x_st[kind]) : g;
    u16* const y = (u16*)a.y[kind] + (i64)token * H * AE_D;
    uint4 v[AE_ROPE_U][2], gv[AE_ROPE_U][2];
    auto load = [&](int h) {  // a team without a head reads the last one's values, which nothing takes
#pragma unroll
      for (int u = 0; u < AE_ROPE_U; ++u) {
        const int hh = min(h + u * AE_TEAMS, h1 - 1);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          gv[u][c] = *(const uint4*)(g + hh * g_st + at[c]);
          if (AE_NORM) v[u][c] = *(const uint4*)(x + hh * x_st + at[c]);
        }
      }
    };
    load(h0 + team);
    if (p < 0) {  // no token
      for (int i = h0 * (AE_D / 8) + lane; i < h1 * (AE_D / 8); i += 32) ((uint4*)y)[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    __syncwarp();  // the factors of the token in front have been read
#pragma unroll
    for (int i = lane; i < AE_PAIRS; i += 32) {  // dz_a = g_a c + g_b s, dz_b = g_b c - g_a s
      const float2 r = ae_turn(sm.turns[i], p);
      const float c = r.x * a.scale, s = r.y * a.scale;
#if AE_NEXT
      f[0][ae_place(2 * i)] = f[0][ae_place(2 * i + 1)] = c;
      f[1][ae_place(2 * i)] = s;
      f[1][ae_place(2 * i + 1)] = -s;
#else
      f[0][ae_place(i)] = c;  // of both halves
      f[1][ae_place(i)] = s;
#endif
    }
    __syncwarp();
#pragma unroll 1
    for (int base = h0;;) {
#pragma unroll
      for (int u = 0; u < AE_ROPE_U; ++u) {
        const int h = base + u * AE_TEAMS + team;
        u64 g2[8], dz[8], k2[8];
        ae_unpack16<BF16>(gv[u][0], gv[u][1], g2);
        if (ae_rotates(t)) {
#if AE_NEXT
          ae_read(f[1], t, k2);
#pragma unroll
          for (int k = 0; k < 8; ++k) dz[k] = ae_mul2(ae_partner(g2, k), k2[k]);
          ae_read(f[0], t, k2);
#pragma unroll
          for (int k = 0; k < 8; ++k) dz[k] = ae_fma22(g2[k], k2[k], dz[k]);
#else
          u64 c2[4], s2[4];
          ae_read(f[0], t, c2);
          ae_read(f[1], t, s2);
          const u64 minus = ae_pack2f(-1.f, -1.f);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            dz[k] = ae_fma22(g2[k + 4], s2[k], ae_mul2(g2[k], c2[k]));
            dz[k + 4] = ae_fma22(ae_mul2(g2[k], s2[k]), minus, ae_mul2(g2[k + 4], c2[k]));
          }
#endif
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) dz[k] = g2[k];
        }
#if AE_NORM
        u64 z[8];
        ae_unpack16<BF16>(v[u][0], v[u][1], z);
        u64 sum = ae_mul2(z[0], z[0]);
#pragma unroll
        for (int k = 1; k < 8; ++k) sum = ae_fma22(z[k], z[k], sum);
        const float r = rsqrtf(fmaf(ae_team_sum(ae_sum2(sum)), 1.f / AE_D, a.eps));
        u64 dot = 0;  // of (dz r w) x: sum of dn n
        ae_read(sm.w[0], t, k2);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          dz[k] = ae_mul2(dz[k], ae_pack2f(r, r));
          if (h < h1) dw2[k] = ae_fma22(dz[k], z[k], dw2[k]);
          dz[k] = ae_mul2(dz[k], k2[k]);
          dot = ae_fma22(dz[k], z[k], dot);
        }
        const float mean = -r * r * ae_team_sum(ae_sum2(dot)) * (1.f / AE_D);
#pragma unroll
        for (int k = 0; k < 8; ++k) dz[k] = ae_fma22(z[k], ae_pack2f(mean, mean), dz[k]);
#endif
        if (h < h1)
#pragma unroll
          for (int c = 0; c < 2; ++c) __stcs((uint4*)(y + h * AE_D + at[c]), ae_pack8<BF16>(dz + 4 * c));
      }
      base += AE_ROPE_U * AE_TEAMS;
      if (base >= h1) break;
      load(base + team);
    }
  }
#if AE_NORM
  if (!a.dw_part) return;
  float dw[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) ae_unpack2f(dw2[j], dw[2 * j], dw[2 * j + 1]);
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
  __shared__ __align__(16) AeRopeSmem sm;
  for (int i = threadIdx.x; i < AE_PAIRS; i += AE_ROPE_THREADS) sm.turns[i] = a.turns[i];
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
  __shared__ float sm[AE_ROPE_THREADS / 32][32];
  ae_grid_wait();
  ae_grid_trigger();
  const int kind = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = blockIdx.x * 32 + lane;
  const float* const part = a.dw_part + (i64)(kind ? a.ctas[0] : 0) * AE_D + d;
  float sum = 0.f;
#pragma unroll 8
  for (int i = warp; i < a.ctas[kind]; i += AE_ROPE_THREADS / 32) sum += part[(i64)i * AE_D];
  sm[warp][lane] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < AE_ROPE_THREADS / 32; ++i) sum += sm[i][lane];
    if (a.w32)
      ((float*)a.dw[kind])[d] = sum;
    else
      ((u16*)a.dw[kind])[d] = (u16)(a.bf16 ? pack2<1>(sum, sum) : pack2<0>(sum, sum));
  }
}
#endif
