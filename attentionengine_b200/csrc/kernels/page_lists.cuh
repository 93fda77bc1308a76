// What the planners of a pool's pages share: a cluster of CTAs works through phases over the rows and over a word of state for each page, and
// everything that a phase needs of the one before it lies behind a barrier of the cluster (the hardware's: no CTA spins on memory).  One launch;
// tables of hundreds of rows are small, and what such a plan takes is latency, not bandwidth.
// Expects AE_LIST_THREADS, AE_LIST_CTAS.

// Exclusive sum over the CTA's threads; `total` is the whole.  `warp_sum` may be used again behind the next barrier.
AE_DEVICE int ae_cta_scan(int x, int* warp_sum, int& total) {
  const u32 lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if ((int)lane >= o) s += y;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < AE_LIST_THREADS / 32; ++w) {
    if (w < (int)warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  return before + s - x;
}

// Pages of a CTA's and a thread's share: [first, last), whole groups of four.
AE_DEVICE void ae_page_share(int num_pages, int cta, int& first, int& last) {
  const int groups = (num_pages + 3) / 4, per = (groups + AE_LIST_CTAS - 1) / AE_LIST_CTAS;
  first = min(cta * per, groups) * 4;
  last = min((cta + 1) * per, groups) * 4;
}

AE_DEVICE void ae_phase_end() {
  __syncwarp();
  cluster_sync_all();
}
