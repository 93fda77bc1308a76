// Merge of the units that the decode over a paged 8-bit cache cut between CTAs: block (c, j) takes the unit that begins in CTA c and goes on behind it,
// if there is one, for the j-th of its heads.  CTA c's partial is slot (c, 1), those of the CTAs behind it are slots (c + i, 0).
// Latency-bound: a thread's partials of four value dims are on their way while the weights are made (once for each partial and row, in shared
// memory); up to 16 partials are one round.  Expects AE_BF16, AE_DV, AE_RT, AE_WARPS.

#define AE_REC (AE_RT * (AE_DV + 2))
#define AE_NEG_INF (-__int_as_float(0x7f800000))
#define AE_FLY (AE_RT * AE_DV >= 2048 ? 8 : 16)  // partials in flight

extern "C" __global__ void __launch_bounds__(128) ae_cache8_merge(const __grid_constant__ AeCache8MergeArgs a) {
  __shared__ float wt[AE_FLY][AE_RT];
  ae_grid_wait();  // brought up under the decode kernel
  ae_grid_trigger();
  const int c = blockIdx.x, j = blockIdx.y, tid = threadIdx.x;
  const AeC8Cut u = a.cuts[c];
  if (u.parts == 0 || j >= u.heads) return;
  const int rows = a.rows - u.rt * AE_RT < AE_RT ? a.rows - u.rt * AE_RT : AE_RT, head = u.h + j;
  auto part = [&](int i) { return a.part + (((i64)(c + i) * 2 + (i == 0)) * AE_WARPS + j) * AE_REC; };
  constexpr int PER = AE_RT * (AE_DV / 4) / 128;  // places of a thread: row, four value dims
  static_assert(PER >= 1, "128 threads");
  float4 acc[PER];
  float m_all = AE_NEG_INF, l_all[PER];  // of thread tid < AE_RT: its row's maximum; of each place: its row's sum
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    l_all[k] = 0.f;
  }
  __shared__ float scale[AE_RT], sum[AE_RT];
  for (int i0 = 0; i0 < u.parts; i0 += AE_FLY) {
    const int n = u.parts - i0 < AE_FLY ? u.parts - i0 : AE_FLY;
    float4 o[PER][AE_FLY];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int x = tid + 128 * k, r = x / (AE_DV / 4), d = x % (AE_DV / 4) * 4;
#pragma unroll
      for (int i = 0; i < AE_FLY; ++i)
        if (i < n && r < rows) o[k][i] = *(const float4*)(part(i0 + i) + r * AE_DV + d);
    }
    if (tid < AE_RT) {  // this round's maximum joins the row's
      float m[AE_FLY], l[AE_FLY], top = m_all;
#pragma unroll
      for (int i = 0; i < AE_FLY; ++i) {
        m[i] = AE_NEG_INF;
        l[i] = 0.f;
        if (i < n && tid < rows) {
          m[i] = part(i0 + i)[AE_RT * AE_DV + tid];
          l[i] = part(i0 + i)[AE_RT * AE_DV + AE_RT + tid];
        }
      }
#pragma unroll
      for (int i = 0; i < AE_FLY; ++i) top = fmaxf(top, m[i]);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < AE_FLY; ++i) {
        const bool none = m[i] == AE_NEG_INF && l[i] == 0.f;  // no kept key
        const float f = none ? 0.f : ae_exp2(m[i] - top);
        wt[i][tid] = none ? AE_NEG_INF : f;  // left out below: 0 times what such a partial holds need not be 0
        if (!none) s += f * l[i];
      }
      scale[tid] = m_all == AE_NEG_INF ? 0.f : ae_exp2(m_all - top);
      sum[tid] = s;
      m_all = top;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = (tid + 128 * k) / (AE_DV / 4);
      if (r >= rows) continue;
      if (i0 > 0) {
        const float f = scale[r];
        l_all[k] *= f;
        acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f;
      }
      l_all[k] += sum[r];
#pragma unroll
      for (int i = 0; i < AE_FLY; ++i) {
        const float f = i < n ? wt[i][r] : AE_NEG_INF;
        if (f == AE_NEG_INF) continue;
        acc[k].x += f * o[k][i].x; acc[k].y += f * o[k][i].y; acc[k].z += f * o[k][i].z; acc[k].w += f * o[k][i].w;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int x = tid + 128 * k, r = x / (AE_DV / 4), d = x % (AE_DV / 4) * 4, row = u.rt * AE_RT + r;
    if (r >= rows) continue;
    const i64 at = a.gq > 1 ? (i64)u.b * a.Hq + head * a.gq + row : ((i64)u.b * a.rows + row) * a.Hq + head;
    const float f = l_all[k] == 0.f ? 0.f : 1.f / l_all[k];  // 0: no kept key
    float4 v = acc[k];
    if (l_all[k] == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
    *(uint2*)((u16*)a.o + at * AE_DV + d) = make_uint2(pack2<AE_BF16>(v.x * f, v.y * f), pack2<AE_BF16>(v.z * f, v.w * f));
  }
}
