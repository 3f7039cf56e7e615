// Token log-probabilities (token_logprobs.h) fused with the head's product: the logits
// H . W^T + b are not kept.  The forward's GEMM gives each row's maximum and two sums,
// the token's logit is a dot product of its own.  The backward is the
// cross-entropy's, band by band, with another form of the epilogue's coefficients.
// With alternatives the logits of a block of rows go through memory in fp32, and the
// row kernels take them from there.
//
// Bound by the MFMA units from some hundred rows on: 8192 x 4096 x 128256 26.1 ms
// forward and backward, 1290 TFLOP/s executed; the entropy's sum costs the forward 1%
// (2048 x 896 x 151936: 477 us, the cross-entropy's 471).  64 x 896 x 32000 takes 93 us
// in seven launches of 2.5 to 38 us: the weight is read three times, its gradient
// written.

// One wave per row: joins the vocabulary splits and takes the token's logit.  Latencies:
// 6 us for 64 rows of d 896 and 250 splits, 27 us for 8192 of d 4096 (the weight's rows).
// stats[n] = {maximum in base 2, log2 of the sum, entropy, 0}.
__global__ __launch_bounds__(256) void lp_linear_join_kernel(const float* __restrict__ pm, const float* __restrict__ ps,
                                                             const float* __restrict__ pw, int splits, long ldp,
                                                             const bf16_t* __restrict__ H, const bf16_t* __restrict__ W,
                                                             const float* __restrict__ bias, int N, int d, int V,
                                                             Tokens a, const int* __restrict__ idx,
                                                             const int* __restrict__ live, LpOut out) {
  const int l = threadIdx.x & 63;
  const long i = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (i >= N) return;
  const long n = idx ? idx[i] : i;
  int col;
  if (!token_of(a, n, V, col)) {
    if (l == 0) {
      out.logprobs[n] = out.entropy[n] = 0.f;
      out.stats[n] = make_float4(0.f, FLT_MAX, 0.f, 0.f);
    }
    return;
  }
  if (live) {  // as in fwd_combine_kernel
    splits = live[1];
    ldp = (long)((live[0] + kBM - 1) / kBM) * kBM;
  }
  typedef EpiLseEntropy<kBN> Epi;
  float m = kLogitFloor, s = 0.f, w = 0.f;
  for (int k = l; k < splits; k += 64) Epi::merge_entropy(m, s, w, pm[k * ldp + i], ps[k * ldp + i], pw[k * ldp + i]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) Epi::merge_entropy(m, s, w, __shfl_xor(m, o), __shfl_xor(s, o), __shfl_xor(w, o));
  float x = 0.f;
  if (col >= 0) {
    const bf16_t *const h = H + n * (long)d, *const wr = W + (long)col * d;
    for (int k = l * 8; k < d; k += 512) {
      const u32x4 hv = *reinterpret_cast<const u32x4*>(h + k), wv = *reinterpret_cast<const u32x4*>(wr + k);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x += bf16_to_f32(hv[q] & 0xffffu) * bf16_to_f32(wv[q] & 0xffffu);
        x += bf16_to_f32(hv[q] >> 16) * bf16_to_f32(wv[q] >> 16);
      }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    if (bias) x += bias[col];
  }
  if (l != 0) return;
  const bool none = s == 0.f;
  // the maximum's logit and the token's are sums in different orders: where they are
  // one, their difference may come out above 0
  const float u = __builtin_fmaf(x, a.scale, -m);
  float lp = none ? -INFINITY : kLn2 * (u - log2f(s));
  // a mask's lowest value: past fp32 in base 2 only
  if (!none && u == -INFINITY) lp = x * a.inv_t;
  if (lp > 0.f) lp = 0.f;
  const float h = none ? 0.f : kLn2 * (log2f(s) - w / s);
  out.logprobs[n] = col >= 0 ? lp : 0.f;
  out.entropy[n] = h;
  out.stats[n] = make_float4(m, none ? FLT_MAX : log2f(s), h, 0.f);
}

struct LpLinearGrad {
  LpGrad p;
  Tokens a;
  const float4* stats;
  int V;
};

// The unit of G (distill_linear.h): at a row's token G is nearly -g / T, so the
// mantissa of the largest one, which all rows have where the gradient is a mean's.
__device__ inline float lp_unit(const LpGrad& p, int N) {
  return mantissa((p.g ? largest_finite(p.g, N) : 0.f) * p.inv_t);
}
__global__ __launch_bounds__(1024) void lp_unit_kernel(LpGrad p, int N, float* __restrict__ unit) {
  const float u = lp_unit(p, N);
  if (threadIdx.x == 0) *unit = u;
}

// Coefficients of GEMM row i, of source row idx[i] (null: i), in units of *unit, which
// every workgroup finds by itself where FIND (few rows: a launch less, 2 to 5 us).
constexpr long kUnitRows = 16384;  // 16 workgroups that read 64 KB each
template <bool FIND>
__global__ __launch_bounds__(1024) void lp_linear_prep_kernel(LpLinearGrad q, const int* __restrict__ idx, int N,
                                                              float4* __restrict__ rowp, int* __restrict__ rowlab,
                                                              float* __restrict__ unit) {
  const int i = blockIdx.x * 1024 + threadIdx.x;
  const float u = FIND ? lp_unit(q.p, N) : *unit;
  if (FIND && i == 0) *unit = u;
  if (i >= N) return;
  const long n = idx ? idx[i] : i;
  int col;
  const bool counts = token_of(q.a, n, q.V, col);
  const float4 st = q.stats[n];
  float4 rp = make_float4(FLT_MAX, 0.f, 0.f, 0.f);
  if (counts && st.y != FLT_MAX) {
    float c, b, at;
    q.p.row(n, col, st.z, c, b, at);
    rp = make_float4(st.x + st.y, c / u, -at / u, b / u);
  } else {
    col = -1;
  }
  rowp[i] = rp;
  rowlab[i] = col;
}

int lp_prep(const SparseGrad& s, const int* idx, long N, float4* rowp, int* rowlab, int*, float*, float* unit,
            hipStream_t st) {
  const LpLinearGrad& q = *static_cast<const LpLinearGrad*>(s.args);
  if (N > kUnitRows) {
    hipLaunchKernelGGL(lp_unit_kernel, dim3(1), dim3(1024), 0, st, q.p, (int)N, unit);
    HIP_TRY(hipGetLastError());
  }
  hipLaunchKernelGGL((N > kUnitRows ? lp_linear_prep_kernel<false> : lp_linear_prep_kernel<true>),
                     dim3((unsigned)ceil_div(N, 1024)), dim3(1024), 0, st, q, idx, (int)N, rowp, rowlab, unit);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}

// Rows of a block whose logits go through memory, with k alternatives: fp32 logits of
// 512 MiB, whole row tiles.  k = 20 of 511 x 1000 x 50257: 77 us for the product (1.5
// rounds of tiles, whose 103 MB of logits leave behind each tile's multiplications),
// 34 us for the rows.  A decoding step is bound by the weight: 8 x 896 x 151936 65 us for
// the product, 11 and 8 for the rows and their join; 8 x 4096 x 128256 209 us in all.
constexpr long kLogitsBudget = 512L << 20;
long logits_ld(long V) { return (long)align_up((size_t)V, 64); }
long logits_block(long N, long V) {
  return std::min<long>(std::max<long>(kLogitsBudget / (4 * logits_ld(V)) / kBM * kBM, kBM), std::max<long>(N, 1));
}

// Columns of the forward's vocabulary tiles: half as wide where twice as many still are
// one round of workgroups (half_tiles).  64 x 896 x 32000 25 -> 19 us; 64 x 896 x 60000,
// two rounds of halves, 33 -> 39.
int lp_tile_width(long N, long V) { return half_tiles(ceil_div(N, kBM) * ceil_div(V, kBN)) ? kTailBN : kBN; }
long lp_slots(long N, long V, bool compact) {
  const int bn = lp_tile_width(N, V);
  return bn == kBN ? forward_slots(N, V, compact) : ceil_div(std::max<long>(N, 1), kBM) * ceil_div(V, bn);
}

struct LpLinearLayout {
  FwdLayout f;
  float *pm, *ps, *pw;  // a slot's maxima and sums
  float* logits;
  void* rows;  // workspace of a block's row kernels
  size_t bytes;
};

LpLinearLayout lp_linear_layout(void* ws, long N, long d, long V, long k) {
  LpLinearLayout L;
  L.f = fwd_layout(ws, N, d, V, CCE_REDUCTION_NONE, CCE_LSE_LABELLED_ROWS);
  Carver c(ws);
  c.off = L.f.bytes;
  if (k > 0) {
    const long R = logits_block(N, V);
    L.pm = L.ps = L.pw = nullptr;
    L.logits = c.take<float>((size_t)(R * logits_ld(V)));
    // the last block has fewer rows, which may be split over more workgroups
    const long last = N > 0 ? (N - 1) % R + 1 : 0;
    L.rows = c.take<char>(std::max(lp_layout(nullptr, R, V, k).bytes, lp_layout(nullptr, last, V, k).bytes));
    L.bytes = align_up(c.off, 256);
    return L;
  }
  const size_t parts = (size_t)lp_slots(N, V, fwd_compacts(N, d, CCE_LSE_LABELLED_ROWS)) * kBM;
  const bool whole = lp_tile_width(N, V) == kBN;  // the cross-entropy's slots
  L.pm = whole ? L.f.pm : c.take<float>(parts);
  L.ps = whole ? L.f.ps : c.take<float>(parts);
  L.pw = c.take<float>(parts);
  L.logits = nullptr;
  L.rows = nullptr;
  L.bytes = align_up(c.off, 256);
  return L;
}

template <template <int> class Epi, int BN>
int launch_out(const GemmShape& g, const OutParams& e, hipStream_t st) {
  const int nb = (int)(ceil_div(g.M, kBM) * ceil_div(g.N, BN));
  constexpr int kKind = CCE_KERNEL_FWD_LSE;
  if (!whole_slabs(g.K)) return launch_gemm<BN, Epi, false, true>(g, e, nb, st, kKind, true);
  if (g.arow) return launch_gemm<BN, Epi, true>(g, e, nb, st, kKind, true);
  return launch_gemm<BN, Epi>(g, e, nb, st, kKind, true);
}

int lp_linear_forward_run(const bf16_t* H, const bf16_t* W, const float* bias, long N, long d, long V, long k,
                          const Tokens& a, LpOut out, const LpLinearLayout& L, hipStream_t st) {
  const FwdLayout& F = L.f;
  const int slots = (int)lp_slots(N, V, F.idx != nullptr), bn = lp_tile_width(N, V);
  int rc = order_rows(a.ids, a.ids64, a.ignore_index, H, N, d, (int)ceil_div(V, bn), slots, F, st);
  if (rc) return rc;
  GemmShape g = forward_shape(H, W, N, d, V, F);
  if (k > 0) {
    const long R = logits_block(N, V), ld = logits_ld(V);
    out.stat_scale = a.scale;
    out.floor = kLogitFloor / a.scale;  // as without alternatives
    const OutParams e = {L.logits, ld, bias};
    for (long m0 = 0; m0 < N; m0 += R) {
      const long rows = std::min(R, N - m0);
      if (F.idx && !F.Hc)
        g.arow = F.idx + m0;
      else
        g.A = (F.Hc ? F.Hc : H) + m0 * d;
      g.M = (int)rows;
      g.live_base = (int)m0;
      if (lp_tile_width(rows, V) == kBN)
        rc = bias ? launch_out<EpiOutBias, kBN>(g, e, st) : launch_out<EpiOut, kBN>(g, e, st);
      else
        rc = bias ? launch_out<EpiOutBias, kTailBN>(g, e, st) : launch_out<EpiOut, kTailBN>(g, e, st);
      if (rc) return rc;
      // without a row order the rows' tokens and outputs start at m0
      Tokens b = a;
      LpOut o = out;
      if (!F.idx && m0 > 0) {
        b.ids = static_cast<const char*>(a.ids) + m0 * (a.ids64 ? 8 : 4);
        o.logprobs += m0;
        o.entropy += m0;
        o.stats += m0;
        o.top_logprobs += m0 * k;
        o.top_indices += m0 * k;
      }
      rc = lp_forward_run(L.logits, ld, rows, V, k, b, F.idx ? F.idx + m0 : nullptr, o,
                          lp_layout(L.rows, rows, V, k), st);
      if (rc) return rc;
    }
    return CCE_OK;
  }
  LseParams ep;
  ep.bias = bias;
  ep.pm = L.pm;
  ep.ps = L.ps;
  ep.ps1 = L.pw;
  ep.ldp = N;
  ep.tiles_n = (int)ceil_div(V, bn);
  ep.splits = bn == kBN ? forward_splits(N, V) : ep.tiles_n;
  ep.scale = a.scale;
  if (bn == kBN)
    rc = bias ? launch_lse<EpiLseBiasEntropy>(g, ep, slots, st) : launch_lse<EpiLseEntropy>(g, ep, slots, st);
  else
    rc = bias ? launch_lse<EpiLseBiasEntropy, kTailBN>(g, ep, slots, st)
              : launch_lse<EpiLseEntropy, kTailBN>(g, ep, slots, st);
  if (rc) return rc;
  hipLaunchKernelGGL(lp_linear_join_kernel, dim3((unsigned)ceil_div(N, 4)), dim3(256), 0, st, L.pm, L.ps, L.pw, ep.splits,
                     (long)N, H, W, bias, (int)N, (int)d, (int)V, a, F.idx, F.live, out);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}
