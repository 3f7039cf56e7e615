// Log-probabilities of given tokens, entropies and top alternatives over logits that
// exist (row kernels, bound by HBM).
//
// With the temperature T, z = x / T, m = max(z), s = sum exp(z - m):
//   logprob = z[t] - m - log s
//   entropy = -sum p log p = log s - sum exp(z - m) (z - m) / s,  p = exp(z - m) / s
//   dx_v = (g ([v == t] - p_v) - h p_v (log p_v + entropy)) / T
// for the gradients g and h of the two.  Both sums of the entropy have one sign, so
// nothing cancels, and one pass with a running maximum gives them: where the maximum
// goes from m to m', s becomes r s and w = sum exp(z - m) (z - m) becomes
// r (w + (m - m') s), r = exp(m - m').
//
// Bound by HBM: the forward reads the logits once and the backward again (the loss in
// between is the caller's) and writes their gradient; 12 operations and an exponential
// per bf16 logit take 80% of the time that its two bytes do.
//
// A row whose token is ignore_index gives zeros (alternatives: column -1) and is not
// read.  A token outside [0, V) has no log-probability: 0, without a gradient.  Where
// every logit is -inf, the log-probability is -inf, the entropy 0 and the gradient 0.

struct Tokens {
  const void* ids;
  int ids64;
  long ignore_index;
  float inv_t;  // 1 / T
  float scale;  // log2(e) / T
};

// Whether row n counts, and its token's column (-1: none).
__device__ inline bool token_of(const Tokens& a, long n, int V, int& col) {
  const long t = load_label(a.ids, a.ids64, n);
  col = t >= 0 && t < V ? (int)t : -1;
  return t != a.ignore_index;
}

// Running maximum of x, sum of exp((x - m) / T), and sum of exp((x - m) / T) times its
// exponent in base 2.
struct LpSums {
  float m = kNegBig, s = 0.f, w = 0.f;
  __device__ inline void rescale(float mn, float scale) {
    const float u = fmaxf((m - mn) * scale, kLeastExponent), r = fast_exp2(u);
    w = r * __builtin_fmaf(u, s, w);
    s *= r;
    m = mn;
  }
  __device__ inline void add(float x, float scale) {
    const float u = (x - m) * scale, e = fast_exp2(u);
    s += e;
    w = __builtin_fmaf(e, fmaxf(u, kLeastExponent), w);  // a NaN stays in e
  }
  // U chunks at once: one change of the maximum for all
  template <typename T, int U>
  __device__ inline void add_chunks(const u32x4 (&raw)[U], float scale) {
    constexpr int E = 16 / sizeof(T);
    float mx = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* v = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) mx = fmaxf(mx, elem_to_f32(v[e]));
    }
    rescale(mx, scale);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* v = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) add(elem_to_f32(v[e]), scale);
    }
  }
  template <typename T>
  __device__ inline void add_chunk(const u32x4& raw, float scale) {
    const u32x4 one[1] = {raw};
    add_chunks<T, 1>(one, scale);
  }
  __device__ inline void add_one(float x, float scale) {
    rescale(fmaxf(m, x), scale);
    add(x, scale);
  }
  __device__ inline void merge(const LpSums& o, float scale) {
    LpSums b = o;
    const float mn = fmaxf(m, b.m);
    rescale(mn, scale);
    b.rescale(mn, scale);
    s += b.s;
    w += b.w;
  }
  __device__ inline void merge_wave(float scale) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      LpSums b;
      b.m = __shfl_xor(m, o);
      b.s = __shfl_xor(s, o);
      b.w = __shfl_xor(w, o);
      merge(b, scale);
    }
  }
  // over a workgroup of 256; every thread gets the sums
  __device__ inline void merge_block(float scale, float (*red)[3]) {
    merge_wave(scale);
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6][0] = m;
      red[threadIdx.x >> 6][1] = s;
      red[threadIdx.x >> 6][2] = w;
    }
    __syncthreads();
    LpSums all;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      LpSums b;
      b.m = red[k][0];
      b.s = red[k][1];
      b.w = red[k][2];
      all.merge(b, scale);
    }
    *this = all;
  }
  // a row whose maximum is below the floor counts as one of -inf alone (a NaN stays)
  __device__ inline void drop_below(float floor) {
    if (m < floor && s == s) s = 0.f;
  }
  __device__ inline float4 packed() const { return make_float4(m, s, w, 0.f); }
  static __device__ inline LpSums of(float4 p) {
    LpSums k;
    k.m = p.x;
    k.s = p.y;
    k.w = p.z;
    return k;
  }
};

// What a forward writes.  stats[n] = {the maximum times stat_scale, log2 of the sum
// (FLT_MAX: nothing to take a gradient of), entropy, 0}.
struct LpOut {
  float *logprobs, *entropy;
  float4* stats;
  float stat_scale;
  float* top_logprobs;  // [N][k]
  int64_t* top_indices;
  float floor = -INFINITY;  // with alternatives: LpSums::drop_below
};

// The row's results, by one thread.  x: the token's logit, where it has one (col >= 0).
__device__ inline void lp_write(const LpOut& o, const Tokens& a, long n, const LpSums& k, int col, float x) {
  const bool none = k.s == 0.f;
  const float ls = logf(k.s), lp = none ? -INFINITY : (x - k.m) * a.inv_t - ls;
  const float h = none ? 0.f : ls - k.w / k.s * kLn2;
  o.logprobs[n] = col >= 0 ? lp : 0.f;
  o.entropy[n] = h;
  o.stats[n] = make_float4(k.m * o.stat_scale, none ? FLT_MAX : log2f(k.s), h, 0.f);
}

// The results of a row that does not count, by a workgroup.
__device__ inline void lp_write_none(const LpOut& o, long n, int k) {
  if (threadIdx.x == 0) {
    o.logprobs[n] = o.entropy[n] = 0.f;
    o.stats[n] = make_float4(0.f, FLT_MAX, 0.f, 0.f);
  }
  for (int j = threadIdx.x; j < k; j += blockDim.x) {
    o.top_logprobs[n * k + j] = 0.f;
    o.top_indices[n * k + j] = -1;
  }
}

__device__ inline float lp_alternative(const Tokens& a, const LpSums& k, float log_s, float x) {
  return k.s == 0.f ? -INFINITY : (x - k.m) * a.inv_t - log_s;
}

// One workgroup per row and split of S; one split: the row's results, more: the sums
// at part[blockIdx.x].  2048 x 151936 bf16: 101 us, 6.2 TB/s (with one change of the
// maximum per chunk instead of per four, 4096 rows of which 60% count 147 us, now 140).
template <typename T>
__global__ __launch_bounds__(256) void lp_stream_kernel(const T* __restrict__ X, long ld, int V, int S, Tokens a,
                                                        LpOut out, float4* __restrict__ part) {
  __shared__ float red[4][3];
  const long n = blockIdx.x / S;
  const int tid = threadIdx.x;
  int col, c0, c1;
  if (!token_of(a, n, V, col)) {
    if (S == 1) lp_write_none(out, n, 0);
    return;
  }
  split_span(V, S, blockIdx.x % S, c0, c1);
  const T* const row = X + n * ld + c0;
  // fetched first, its latency hides under the stream
  const float x = S == 1 && tid == 0 && col >= 0 ? elem_to_f32(row[col]) : 0.f;
  const RowSplit<T> sp(row, c1 - c0);
  LpSums k;
  if (tid < sp.head) k.add_one(elem_to_f32(row[tid]), a.scale);
  if (tid < c1 - c0 - sp.tail_start) k.add_one(elem_to_f32(row[sp.tail_start + tid]), a.scale);
  const u32x4* const body = reinterpret_cast<const u32x4*>(row + sp.head);
  constexpr int U = 4;
  int c = tid;
  for (; c + (U - 1) * 256 < sp.chunks; c += U * 256) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __builtin_nontemporal_load(body + c + u * 256);
    k.template add_chunks<T, U>(raw, a.scale);
  }
  for (; c < sp.chunks; c += 256) k.template add_chunk<T>(__builtin_nontemporal_load(body + c), a.scale);
  k.merge_block(a.scale, red);
  if (tid != 0) return;
  if (S == 1)
    lp_write(out, a, n, k, col, x);
  else
    part[blockIdx.x] = k.packed();
}

// One wave per row: joins its splits (3 us for 16 rows: latencies).
template <typename T>
__global__ __launch_bounds__(256) void lp_join_kernel(const T* __restrict__ X, long ld, int N, int V, int S, Tokens a,
                                                      LpOut out, const float4* __restrict__ part) {
  const int l = threadIdx.x & 63;
  const long n = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (n >= N) return;
  int col;
  if (!token_of(a, n, V, col)) {
    if (l == 0) {
      out.logprobs[n] = out.entropy[n] = 0.f;
      out.stats[n] = make_float4(0.f, FLT_MAX, 0.f, 0.f);
    }
    return;
  }
  const float x = col >= 0 ? elem_to_f32(X[n * ld + col]) : 0.f;
  LpSums k;
  for (int s = l; s < S; s += 64) k.merge(LpSums::of(part[n * S + s]), a.scale);
  k.merge_wave(a.scale);
  if (l == 0) lp_write(out, a, n, k, col, x);
}

// With the k largest logits beside: the sums are taken in the first pass of
// top_of_row, which is the only one over HBM.  One workgroup per row i and split of
// S; the row belongs to token rowmap[i] (null: i).  One split: the row's results,
// more: the sums at part[blockIdx.x] and the split's k largest at
// top_part[blockIdx.x * k], as top_logits_kernel leaves them.
//
// Bound by the vector units where the type has 16 bits: k = 20 of 2048 x 151936 bf16
// 123 us (5.1 TB/s of the rows; the sums alone take 101, the largest alone 101), of
// 1024 x 128256 fp32 88 us (6.0 TB/s).  Short rows end together in a selection that
// nothing hides: k = 5 of 2047 x 50257 56 us, 42 by the sums' time per byte.
template <typename T>
__global__ __launch_bounds__(256) void lp_top_kernel(const T* __restrict__ X, long ld, int V, int S, int k, Tokens a,
                                                     const int* __restrict__ rowmap, LpOut out,
                                                     float4* __restrict__ part, uint64_t* __restrict__ top_part) {
  __shared__ uint32_t hist[256];
  __shared__ uint64_t cands[kTopCandidates];
  __shared__ uint16_t groups[kTopGroups];
  __shared__ int count;
  __shared__ float red[4][3];
  const TopList list = {cands, &count};
  const int tid = threadIdx.x;
  const long i = blockIdx.x / S, n = rowmap ? rowmap[i] : i;
  int col, c0, c1;
  if (!token_of(a, n, V, col)) {
    if (S == 1) lp_write_none(out, n, k);
    return;
  }
  split_span(V, S, blockIdx.x % S, c0, c1);
  const T* const row = X + i * ld + c0;
  const int len = c1 - c0, m = min(k, len);
  LpSums sums;
  if (m > 0) {
    const RowSplit<T> sp(row, len);
    if (tid < sp.head) sums.add_one(elem_to_f32(row[tid]), a.scale);
    if (tid < len - sp.tail_start) sums.add_one(elem_to_f32(row[sp.tail_start + tid]), a.scale);
    auto add = [&](const auto& raw) {
      sums.template add_chunks<T, (int)(sizeof(raw) / sizeof(u32x4))>(raw, a.scale);
    };
    // too few chunks for top_of_row's pass over them
    if (sp.chunks < m)
      for_each_chunk<256, false>(reinterpret_cast<const u32x4*>(row + sp.head), sp.chunks, tid,
                                 [&](int, const u32x4& raw) { sums.template add_chunk<T>(raw, a.scale); });
    top_of_row(row, len, m, hist, groups, list, add);
  }
  sums.merge_block(a.scale, red);
  if (S == 1) {
    sums.drop_below(out.floor);
    const float log_s = logf(sums.s);
    top_ranked(list, k, [&](int rank, uint64_t c) {
      out.top_logprobs[n * k + rank] = lp_alternative(a, sums, log_s, elem_to_f32(row[column(c)]));
      out.top_indices[n * k + rank] = column(c);
    });
    if (tid == 0) lp_write(out, a, n, sums, col, col >= 0 ? elem_to_f32(row[col]) : 0.f);
    return;
  }
  if (tid == 0) part[blockIdx.x] = sums.packed();
  uint64_t* const to = top_part + (long)blockIdx.x * k;
  if (m > 0) top_ranked(list, m, [&](int rank, uint64_t c) { to[rank] = candidate(c >> 32, c0 + column(c)); });
  for (int j = m + tid; j < k; j += 256) to[j] = 0;
}

// One workgroup per row: joins its splits' sums and largest logits (k = 20 of 8 x
// 128256 bf16: 6 us after 12 of lp_top_kernel, latencies both).
template <typename T>
__global__ __launch_bounds__(256) void lp_top_join_kernel(const T* __restrict__ X, long ld, int V, int S, int k,
                                                          Tokens a, const int* __restrict__ rowmap, LpOut out,
                                                          const float4* __restrict__ part,
                                                          const uint64_t* __restrict__ top_part) {
  const int tid = threadIdx.x;
  const long i = blockIdx.x, n = rowmap ? rowmap[i] : i;
  const T* const row = X + i * ld;
  int col;
  if (!token_of(a, n, V, col)) {
    lp_write_none(out, n, k);
    return;
  }
  LpSums sums;  // by every wave
  for (int s = tid & 63; s < S; s += 64) sums.merge(LpSums::of(part[i * S + s]), a.scale);
  sums.merge_wave(a.scale);
  // Lane 0's for all: the lanes of a pair add their two products the other way round, of
  // which one is rounded, and which lane writes which candidate is not the same every run
  sums.m = __shfl(sums.m, 0);
  sums.s = __shfl(sums.s, 0);
  sums.drop_below(out.floor);
  const float log_s = logf(sums.s);
  top_join(top_part + i * S * k, S, k, [&](int rank, uint64_t c) {
    out.top_logprobs[n * k + rank] = lp_alternative(a, sums, log_s, elem_to_f32(row[column(c)]));
    out.top_indices[n * k + rank] = column(c);
  });
  if (tid == 0) lp_write(out, a, n, sums, col, col >= 0 ? elem_to_f32(row[col]) : 0.f);
}

// The coefficients of row n's gradient in base 2, y = log2 p:
//   dx_v = 2^y (c + b y) + [v == t] at
struct LpGrad {
  const float *g, *h;  // gradients of the log-probabilities and of the entropies; null: none
  float inv_t;
  // col: the token's, -1: none
  __device__ inline void row(long n, int col, float entropy, float& c, float& b, float& at) const {
    const float gn = g && col >= 0 ? g[n] : 0.f, hn = h ? h[n] : 0.f;
    c = -(gn + hn * entropy) * inv_t;
    b = -hn * kLn2 * inv_t;
    at = gn * inv_t;
  }
};

// One workgroup per row and split writes the split's columns of dX, the token's
// behind a barrier.  4096 x 151936 bf16, 40% of the rows only zeroed: 411 us for 2.0 GB,
// 4.9 TB/s, the rate of a large copy.
template <typename T>
__global__ __launch_bounds__(256) void lp_grad_kernel(LpGrad p, const T* __restrict__ X, long ld, int V, int S,
                                                      Tokens a, const float4* __restrict__ stats, T* __restrict__ dX,
                                                      long ldg) {
  const long n = blockIdx.x / S;
  const int tid = threadIdx.x;
  int c0, c1, col;
  split_span(V, S, blockIdx.x % S, c0, c1);
  T* const drow = dX + n * ldg + c0;
  const bool counts = token_of(a, n, V, col);
  const float4 st = counts ? stats[n] : make_float4(0.f, FLT_MAX, 0.f, 0.f);
  if (st.y == FLT_MAX) {
    zero_row<256>(drow, c1 - c0, tid);
    return;
  }
  float c, b, at;
  p.row(n, col, st.z, c, b, at);
  auto dense = [&](float x) {
    const float y = __builtin_fmaf(x - st.x, a.scale, -st.y);
    return fast_exp2(y) * __builtin_fmaf(b, fmaxf(y, kLeastExponent), c);
  };
  const T* const row = X + n * ld + c0;
  const RowSplit<T> sp(row, c1 - c0);
  if ((reinterpret_cast<uintptr_t>(drow + sp.head) & 15u) != 0) {
    for (int v = tid; v < c1 - c0; v += 256) drow[v] = f32_to_elem<T>(dense(elem_to_f32(row[v])));
  } else {
    if (tid < sp.head) drow[tid] = f32_to_elem<T>(dense(elem_to_f32(row[tid])));
    if (tid < c1 - c0 - sp.tail_start) {
      const int v = sp.tail_start + tid;
      drow[v] = f32_to_elem<T>(dense(elem_to_f32(row[v])));
    }
    u32x4* const dbody = reinterpret_cast<u32x4*>(drow + sp.head);
    for_each_chunk(reinterpret_cast<const u32x4*>(row + sp.head), sp.chunks, tid, [&](int i, const u32x4& raw) {
      const T* v = reinterpret_cast<const T*>(&raw);
      u32x4 o;
      T* e = reinterpret_cast<T*>(&o);
#pragma unroll
      for (int j = 0; j < RowSplit<T>::E; ++j) e[j] = f32_to_elem<T>(dense(elem_to_f32(v[j])));
      __builtin_nontemporal_store(o, dbody + i);
    });
  }
  if (col < c0 || col >= c1) return;  // for the whole workgroup
  __syncthreads();
  if (tid == 0) drow[col - c0] = f32_to_elem<T>(dense(elem_to_f32(row[col - c0])) + at);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int check_tokens(const void* ids, int ids64, int64_t N, int64_t ignore_index, float temperature, Tokens& a) {
  if (!(temperature >= 1e-2f && temperature <= 1e3f))
    return fail(CCE_ERR_INVALID_ARG, "temperature must be in [0.01, 1000] (got %g)", (double)temperature);
  if (N > 0 && !ids) return fail(CCE_ERR_INVALID_ARG, "tokens must not be null");
  a.ids = ids;
  a.ids64 = ids64;
  a.ignore_index = (long)ignore_index;
  a.inv_t = 1.f / temperature;
  a.scale = kLog2e * a.inv_t;
  return CCE_OK;
}

int check_alternatives(int64_t k, int64_t V, int64_t N, const void* top_logprobs, const void* top_indices) {
  if (k < 0 || k > kTopMax || k > V)
    return fail(CCE_ERR_INVALID_ARG, "top_k must be in [0, min(%d, V = %ld)] (got %ld)", kTopMax, (long)V, (long)k);
  if (k > 0 && N > 0 && (!top_logprobs || !top_indices))
    return fail(CCE_ERR_INVALID_ARG, "top_logprobs_out and top_indices_out must not be null with top_k");
  return CCE_OK;
}

// Workgroups per row.
int lp_splits(long N, long V, long k) { return k > 0 ? top_splits(N, V, k) : kd_splits(N, V); }

struct LpLayout {
  float4* part;
  uint64_t* top;
  size_t bytes;
};

LpLayout lp_layout(void* ws, long N, long V, long k) {
  Carver c(ws);
  LpLayout L;
  const int S = lp_splits(N, V, k);
  const size_t parts = S > 1 ? (size_t)N * S : 0;
  L.part = c.take<float4>(parts);
  L.top = c.take<uint64_t>(parts * k);
  L.bytes = align_up(c.off, 256);
  return L;
}

// Rows [N][ld] of logits; row i's token and outputs are those at rowmap[i] (with k; null: i).
template <typename T>
int lp_forward_run(const T* X, long ld, long N, long V, long k, const Tokens& a, const int* rowmap, const LpOut& out,
                   const LpLayout& L, hipStream_t st) {
  const int S = lp_splits(N, V, k);
  if (k > 0) {
    hipLaunchKernelGGL(lp_top_kernel<T>, dim3((unsigned)(N * S)), dim3(256), 0, st, X, ld, (int)V, S, (int)k, a, rowmap,
                       out, L.part, L.top);
    HIP_TRY(hipGetLastError());
    if (S == 1) return CCE_OK;
    hipLaunchKernelGGL(lp_top_join_kernel<T>, dim3((unsigned)N), dim3(256), 0, st, X, ld, (int)V, S, (int)k, a, rowmap,
                       out, L.part, L.top);
    HIP_TRY(hipGetLastError());
    return CCE_OK;
  }
  hipLaunchKernelGGL(lp_stream_kernel<T>, dim3((unsigned)(N * S)), dim3(256), 0, st, X, ld, (int)V, S, a, out, L.part);
  HIP_TRY(hipGetLastError());
  if (S == 1) return CCE_OK;
  hipLaunchKernelGGL(lp_join_kernel<T>, dim3((unsigned)ceil_div(N, 4)), dim3(256), 0, st, X, ld, (int)N, (int)V, S, a,
                     out, L.part);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}
