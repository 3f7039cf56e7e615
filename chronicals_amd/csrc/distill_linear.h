// Distillation fused with the head's product: the logits H . W^T + b are never
// stored.  The forward's GEMM gives each row's log-sum-exp (at the temperature
// and, where the labels' loss needs it, at 1) and the logits at the row's K + 1
// columns are dot products of their own.  The backward is the cross-entropy's,
// band by band, with the dense part of the gradient in the recompute's epilogue
// and the K + 1 columns written over it before the band's products read it.

// rows[n]: -1 where row n does not count, else its label, or V without a target.
// One wave per row.  Only the order of the rows needs this ahead of the loss:
// without one (a single row tile) kd_linear_loss_kernel does it, a launch less (64
// rows, d 896, V 32000, forward and backward 119 -> 117 us).
__global__ __launch_bounds__(256) void kd_rows_kernel(Teacher a, int N, int V, int* __restrict__ rows) {
  const int l = threadIdx.x & 63;
  const long n = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (n >= N) return;
  int r = V;
  if (a.labels) {
    const long lab = load_label(a.labels, a.labels64, n);
    r = lab == a.ignore_index ? -1 : (lab >= 0 && lab < V ? (int)lab : V);
  } else {
    bool any = false;
    for (int k = l; k < a.K; k += 64) {
      float t;
      any = any || load_entry(a, n, k, V, t) >= 0;
    }
    if (__ballot(any) == 0) r = -1;
  }
  if (l == 0) rows[n] = r;
}

// One workgroup per row: joins the vocabulary splits, takes the logits at the
// row's columns (xk[n][j], j = K: the label; 0 where there is none) and forms its loss.  Bound by the
// weight's rows that the columns name: K = 64, 2048 x 896 43 us (5.4 TB/s, most of
// it from the memory-side cache), 8192 x 4096 689 us (6.2 TB/s).
// stats[n] = {log2-sum-exp2 at the temperature, at 1}.
template <bool DU>
__global__ __launch_bounds__(256) void kd_linear_loss_kernel(
    const float* __restrict__ pm, const float* __restrict__ ps, const float* __restrict__ ps1, int splits, long ldp,
    const bf16_t* __restrict__ H, const bf16_t* __restrict__ W, const float* __restrict__ bias, int d, int V, Teacher a,
    int* __restrict__ rows, int rows_known, const int* __restrict__ idx, const int* __restrict__ live,
    float2* __restrict__ stats, float* __restrict__ xk, float* __restrict__ rowloss, float* __restrict__ bsum,
    int* __restrict__ bcnt) {
  __shared__ Entries e;
  __shared__ float ex[kMaxEntries + 1];
  const int tid = threadIdx.x, l = tid & 63;
  const long i = blockIdx.x, n = idx ? idx[i] : i;
  int r;
  if (rows_known) {
    r = rows[n];
  } else {
    r = row_counts(a, n, V, r) ? (r < 0 ? V : r) : -1;
    if (tid == 0) rows[n] = r;
  }
  if (r < 0) {
    if (tid == 0) {
      stats[n] = make_float2(0.f, 0.f);
      rowloss[n] = bsum[n] = 0.f;
      bcnt[n] = 0;
    }
    for (int j = tid; j <= a.K; j += 256) xk[n * (a.K + 1) + j] = 0.f;
    return;
  }
  if (live) {  // as in fwd_combine_kernel
    splits = live[1];
    ldp = (long)((live[0] + kBM - 1) / kBM) * kBM;
  }
  const float scale = kLog2e * a.inv_t;
  float m = DU ? kLogitFloor : kNegBig, s = 0.f, s1 = 0.f;
  auto merge = [&](float m2, float s2, float s12) {
    const float mn = fmaxf(m, m2), u = m - mn, v = m2 - mn;
    s = s * fast_exp2(DU ? u * scale : u) + s2 * fast_exp2(DU ? v * scale : v);
    if constexpr (DU) s1 = s1 * fast_exp2(u * kLog2e) + s12 * fast_exp2(v * kLog2e);
    m = mn;
  };
  for (int k = l; k < splits; k += 64) merge(pm[k * ldp + i], ps[k * ldp + i], DU ? ps1[k * ldp + i] : 0.f);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) merge(__shfl_xor(m, o), __shfl_xor(s, o), DU ? __shfl_xor(s1, o) : 0.f);
  const float lse = (DU ? m * scale : m) + log2f(s), lse1 = DU ? m * kLog2e + log2f(s1) : lse;
  const int label = r < V && a.ce != 0.f ? r : -1;
  int col;
  float q, lq;
  load_entries(a, n, V, e, col, q, lq);
  // sixteen lanes per column
  const bf16_t* const h = H + n * (long)d;
  for (int j = tid >> 4; j <= a.K; j += 16) {
    const int c = j < a.K ? e.col[j] : label;
    if (c < 0) {
      if ((tid & 15) == 0) xk[n * (a.K + 1) + j] = 0.f;
      continue;
    }
    const bf16_t* const wr = W + (long)c * d;
    float dot = 0.f;
    for (int k = (tid & 15) * 8; k < d; k += 128) {
      const u32x4 hv = *reinterpret_cast<const u32x4*>(h + k), wv = *reinterpret_cast<const u32x4*>(wr + k);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        dot += bf16_to_f32(hv[p] & 0xffffu) * bf16_to_f32(wv[p] & 0xffffu);
        dot += bf16_to_f32(hv[p] >> 16) * bf16_to_f32(wv[p] >> 16);
      }
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) dot += __shfl_xor(dot, o);
    if ((tid & 15) == 0) {
      dot += bias ? bias[c] : 0.f;
      ex[j] = dot;
      xk[n * (a.K + 1) + j] = dot;
    }
  }
  __syncthreads();
  float term = 0.f;
  if (col >= 0 && q != 0.f && a.kd != 0.f) term = q * (lq + (lse * kLn2 - ex[tid] * a.inv_t));
  const float sum = block_sum(term, e.red);
  if (tid == 0) {
    float loss = a.kd * sum;
    if (a.ce != 0.f) loss += a.ce * (lse1 * kLn2 - (label >= 0 ? ex[a.K] : 0.f));
    stats[n] = make_float2(lse, lse1);
    rowloss[n] = bsum[n] = loss;
    bcnt[n] = 1;
  }
}

struct DistillGrad {
  const float* grad_out;
  const float2* stats;
  const float* xk;
  const int* rows;
  const int32_t* n_valid;
  int reduction, V;
  Teacher a;
};

// The unit of G.  G is held in bf16, and at a row's label it is nearly the same
// number in every row, -ce g (or without labels -kd T g, where one entry has all
// the weight): rounded the same way in every row, half a step of it, up to 2^-8 of
// the label's share, would stay in the sums over the rows.  So G is held over the
// mantissa of that number, in [1, 2), and the products' fp32 sums are multiplied by
// it: the number itself becomes a power of two, no range is lost, and what is
// rounded differs from row to row.
__device__ inline float mantissa(float x) { return __uint_as_float((__float_as_uint(x) & 0x007fffffu) | 0x3f800000u); }
__device__ inline float unit_of(const Teacher& a, float g) { return mantissa(g * (a.ce != 0.f ? a.ce : a.kdg)); }

// *unit where every row has a factor of its own: the largest finite one's, which
// all have where a mean or a masked mean of the rows follows.  One workgroup, bound
// by latency: 5 us for 2048 rows, 10 for 16384.
__global__ __launch_bounds__(1024) void kd_unit_kernel(Teacher a, const float* __restrict__ grad_out, int N,
                                                       float* __restrict__ unit) {
  __shared__ float red[16];
  float g = 0.f;
  for (int n = threadIdx.x; n < N; n += 1024) {
    const float v = fabsf(grad_out[n]);
    if (v < INFINITY) g = fmaxf(g, v);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) g = fmaxf(g, __shfl_xor(g, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = g;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) g = fmaxf(g, red[w]);
  *unit = unit_of(a, g);
}

// One workgroup per GEMM row i of source row idx[i] (idx null: i): its
// coefficients, and the gradient at its K + 1 columns, in units of *unit.
template <bool DU>
__global__ __launch_bounds__(256) void kd_linear_prep_kernel(DistillGrad p, const int* __restrict__ idx,
                                                             float4* __restrict__ rowp, int* __restrict__ rowlab,
                                                             int* __restrict__ cols, float* __restrict__ vals,
                                                             float* __restrict__ unit) {
  __shared__ Entries e;
  const int tid = threadIdx.x, K = p.a.K;
  const long i = blockIdx.x, n = idx ? idx[i] : i;
  const int r = p.rows[n];
  const float g = grad_factor(p.grad_out, p.n_valid, p.reduction, n);
  const float u = p.reduction == CCE_REDUCTION_NONE ? *unit : unit_of(p.a, g);
  if (tid == 0) rowlab[i] = -1;
  if (i == 0 && tid == 0 && p.reduction != CCE_REDUCTION_NONE) *unit = u;
  if (r < 0) {
    if (tid == 0) rowp[i] = make_float4(FLT_MAX, 0.f, 0.f, DU ? FLT_MAX : 0.f);
    for (int j = tid; j <= K; j += 256) cols[i * (K + 1) + j] = -1;
    return;
  }
  int col;
  float q, lq;
  const bool any = load_entries(p.a, n, p.V, e, col, q, lq);
  const float2 st = p.stats[n];
  const float scale = kLog2e * p.a.inv_t, ce = g * p.a.ce / u, kdg = any ? g * p.a.kdg / u : 0.f;
  const float cp = DU ? kdg : kdg + ce;
  const int label = r < p.V && p.a.ce != 0.f ? r : -1;
  if (tid == 0) rowp[i] = make_float4(st.x, cp, DU ? ce : 0.f, DU ? st.y : 0.f);
  auto put = [&](int j, int c) {
    cols[i * (K + 1) + j] = c;
    if (c < 0) return;
    const float x = p.xk[n * (K + 1) + j];
    float v = cp * fast_exp2(__builtin_fmaf(x, scale, -st.x));
    if constexpr (DU) v = __builtin_fmaf(ce, fast_exp2(__builtin_fmaf(x, kLog2e, -st.y)), v);
    v -= kdg * entries_at(e, K, c);
    // entries that share a column, and the label among them, hold the same value
    vals[i * (K + 1) + j] = c == label ? v - ce : v;
  };
  if (tid < K) put(tid, col);
  if (tid == 0) put(K, label);
}

int distill_prep(const SparseGrad& s, const int* idx, long N, float4* rowp, int* rowlab, int* col, float* val,
                 float* unit, hipStream_t st) {
  const DistillGrad& p = *static_cast<const DistillGrad*>(s.args);
  if (p.reduction == CCE_REDUCTION_NONE) {
    hipLaunchKernelGGL(kd_unit_kernel, dim3(1), dim3(1024), 0, st, p.a, p.grad_out, (int)N, unit);
    HIP_TRY(hipGetLastError());
  }
  auto* const prep = s.softmaxes == kTwoSoftmaxes ? kd_linear_prep_kernel<true> : kd_linear_prep_kernel<false>;
  hipLaunchKernelGGL(prep, dim3((unsigned)N), dim3(256), 0, st, p, idx, rowp, rowlab, col, val, unit);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}

struct DistillLayout {
  FwdLayout f;
  float *ps1, *bsum;
  int* bcnt;
  size_t bytes;
};

DistillLayout distill_layout(void* ws, long N, long d, long V, int reduction) {
  DistillLayout L;
  L.f = fwd_layout(ws, N, d, V, reduction, CCE_LSE_LABELLED_ROWS);
  Carver c(ws);
  c.off = L.f.bytes;
  const size_t n = (size_t)std::max<long>(N, 1);
  L.ps1 = c.take<float>((size_t)forward_slots(N, V, L.f.idx != nullptr || fwd_compacts(N, d, CCE_LSE_LABELLED_ROWS)) * kBM);
  L.bsum = c.take<float>(n);
  L.bcnt = c.take<int>(n);
  L.bytes = align_up(c.off, 256);
  return L;
}

int distill_forward_run(const bf16_t* H, const bf16_t* W, const float* bias, long N, long d, long V, const Teacher& a,
                        int reduction, float* loss_out, float2* stats, float* xk, int* rows, int32_t* n_valid,
                        const DistillLayout& L, hipStream_t st) {
  const FwdLayout& F = L.f;
  const bool dual = two_softmaxes(a);
  const int slots = (int)forward_slots(N, V, F.idx != nullptr);
  if (F.idx) {
    hipLaunchKernelGGL(kd_rows_kernel, dim3((unsigned)ceil_div(N, 4)), dim3(256), 0, st, a, (int)N, (int)V, rows);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(compact_rows_kernel, dim3(1), dim3(1024), 0, st, rows, 0, (int)N, -1L, F.idx, F.live, slots,
                       (int)ceil_div(V, kBN), device_cus());
    HIP_TRY(hipGetLastError());
    if (F.Hc) {
      hipLaunchKernelGGL(gather_rows_kernel, dim3((unsigned)std::min<long>(ceil_div(N * (d / 8), 256), 8192)),
                         dim3(256), 0, st, H, (int)d, F.idx, (int)N, F.Hc);
      HIP_TRY(hipGetLastError());
    }
  }
  GemmShape g;
  g.A = F.Hc ? F.Hc : H;
  if (F.idx && !F.Hc) {
    g.arow = F.idx;
    g.arows = N;
  }
  g.lda = d;
  g.B = W;
  g.ldb = d;
  g.M = (int)N;
  g.N = (int)V;
  g.K = (int)d;
  g.live = F.live;
  g.dyn = F.live ? kDynM : kDynNone;
  LseParams ep;
  ep.bias = bias;
  ep.pm = F.pm;
  ep.ps = F.ps;
  ep.ps1 = L.ps1;
  ep.ldp = N;
  ep.splits = forward_splits(N, V);
  ep.tiles_n = (int)ceil_div(V, kBN);
  ep.scale = kLog2e * a.inv_t;
  const int sm = softmaxes_of(a);
  auto* const lse = sm == kOneSoftmax      ? (bias ? launch_lse<EpiLseBias> : launch_lse<EpiLse>)
                    : sm == kAtTemperature ? (bias ? launch_lse<EpiLseBiasTemp> : launch_lse<EpiLseTemp>)
                                           : (bias ? launch_lse<EpiLseBiasTwo> : launch_lse<EpiLseTwo>);
  const int rc = lse(g, ep, slots, st);
  if (rc) return rc;
  float* const rowloss = reduction == CCE_REDUCTION_NONE ? loss_out : F.rowloss;
  auto* const loss = dual ? kd_linear_loss_kernel<true> : kd_linear_loss_kernel<false>;
  hipLaunchKernelGGL(loss, dim3((unsigned)N), dim3(256), 0, st, F.pm, F.ps, L.ps1, ep.splits, (long)N, H, W, bias,
                     (int)d, (int)V, a, rows, F.idx != nullptr, F.idx, F.live, stats, xk, rowloss, L.bsum, L.bcnt);
  HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(fwd_finalize_kernel, dim3(1), dim3(1024), 0, st, L.bsum, L.bcnt, (int)N, reduction, loss_out,
                     n_valid);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}
