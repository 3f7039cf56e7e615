// Distillation from a teacher's top logits, over student logits that exist
// (row kernels, bound by HBM) and fused with the head's product (the GEMM core).
//
// A row has K entries: the teacher's logit t_k at column i_k.  An entry is
// usable where 0 <= i_k < V and t_k is not -inf.  With temperature T
//   q = softmax(t / T) over the usable entries, p_T = softmax(x / T)
//   loss = kd T^2 sum_k q_k (log q_k - log p_T[i_k]) + ce (lse(x) - x[label])
//   dloss/dx_v = kd T (p_T[v] - sum of q_k with i_k = v) + ce (p_1[v] - [v == label])
// where a row without a usable entry has no first term and a label outside
// [0, V) no x[label].  A row counts where its label is not ignore_index, or,
// without labels, where it has a usable entry; other rows give no loss and a
// zero gradient, whatever they hold.
//
// So the gradient is dense in p (one fused multiply-add and one or two
// exponentials per logit) except at the K + 1 columns of a row's entries and
// label.  Those are computed in fp32 and written over the dense values: one
// rounding each, also where p and q nearly cancel.

constexpr int kMaxEntries = CCE_MAX_TEACHER_ENTRIES;

struct Teacher {
  const void* t;
  int tdtype;
  const void* index;
  int index64;
  int K;
  const void* labels;  // null: none
  int labels64;
  long ignore_index;
  float inv_t;  // 1 / T
  float kd;     // kd T^2, the loss's factor
  float kdg;    // kd T, the gradient's
  float ce;
  int squares;  // T = 2^squares for 1 and 2: exp(x) is exp(x / T) squared so often; 0: T is another
};

__device__ inline float load_teacher(const Teacher& a, long i) {
  if (a.tdtype == CCE_DTYPE_F32) return static_cast<const float*>(a.t)[i];
  if (a.tdtype == CCE_DTYPE_F16) return (float)static_cast<const _Float16*>(a.t)[i];
  return bf16_to_f32(static_cast<const uint16_t*>(a.t)[i]);
}

// Entry k of row n: its logit, and its column or -1 where it is not usable.
__device__ inline int load_entry(const Teacher& a, long n, int k, int V, float& t) {
  t = -INFINITY;
  if (k >= a.K) return -1;
  const long c = load_label(a.index, a.index64, n * a.K + k);
  if (c < 0 || c >= V) return -1;
  const float v = load_teacher(a, n * a.K + k);
  if (v == -INFINITY) return -1;
  t = v;
  return (int)c;
}

// Whether row n counts (by a workgroup of 256, all of whose threads call this),
// and its label (-1: no target).
__device__ inline bool row_counts(const Teacher& a, long n, int V, int& label) {
  label = -1;
  if (a.labels) {
    const long lab = load_label(a.labels, a.labels64, n);
    if (lab == a.ignore_index) return false;
    if (lab >= 0 && lab < V) label = (int)lab;
    return true;
  }
  float t;
  return __syncthreads_or(load_entry(a, n, threadIdx.x, V, t) >= 0);
}

// A row's entries in LDS.
struct Entries {
  int col[kMaxEntries];
  float q[kMaxEntries];
  float red[4];
};

// Thread k of a workgroup of 256 takes entry k: its column (-1: none), q_k and
// log q_k; every thread gets whether the row has a usable entry.
__device__ inline bool load_entries(const Teacher& a, long n, int V, Entries& e, int& col, float& q, float& lq) {
  float t;
  col = load_entry(a, n, threadIdx.x, V, t);
  float mx = t;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  if ((threadIdx.x & 63) == 0) e.red[threadIdx.x >> 6] = mx;
  const bool any = __syncthreads_or(col >= 0);
  mx = fmaxf(fmaxf(e.red[0], e.red[1]), fmaxf(e.red[2], e.red[3]));
  // differences before the division by T: no overflow at a small T
  const float u = col >= 0 ? (t - mx) * a.inv_t : -INFINITY;
  const float p = fast_exp2(u * kLog2e);
  const float s = block_sum(p, e.red);
  q = col >= 0 ? p / s : 0.f;
  lq = u - logf(s);
  e.col[threadIdx.x] = col;
  e.q[threadIdx.x] = q;
  __syncthreads();
  return any;
}

// The teacher's share of column c: the q of every entry there, in order.
__device__ inline float entries_at(const Entries& e, int K, int c) {
  float s = 0.f;
  for (int j = 0; j < K; ++j) s += e.col[j] == c ? e.q[j] : 0.f;
  return s;
}

// ---------------------------------------------------------------------------
// Over logits that exist
// ---------------------------------------------------------------------------

// Running maximum of x and sums of exp((x - m) / T) and, with DU, exp(x - m).
// The differences are taken before they are scaled: with x at its type's lowest
// value, m * log2(e) would pass the range of fp32.
template <bool DU>
struct KdSums {
  float m = kNegBig, st = 0.f, s1 = 0.f;
  __device__ inline void rescale(float mn, float scale) {
    st *= fast_exp2((m - mn) * scale);
    if constexpr (DU) s1 *= fast_exp2((m - mn) * kLog2e);
    m = mn;
  }
  // SQ: Teacher::squares
  template <int SQ>
  __device__ inline void add(float x, float scale) {
    const float e = fast_exp2((x - m) * scale);
    st += e;
    if constexpr (DU) {
      if constexpr (SQ == 0)
        s1 += fast_exp2((x - m) * kLog2e);
      else if constexpr (SQ == 1)
        s1 = __builtin_fmaf(e, e, s1);
      else
        s1 = __builtin_fmaf(e * e, e * e, s1);
    }
  }
  __device__ inline void merge(float m2, float st2, float s12, float scale) {
    const float mn = fmaxf(m, m2);
    rescale(mn, scale);
    st += st2 * fast_exp2((m2 - mn) * scale);
    if constexpr (DU) s1 += s12 * fast_exp2((m2 - mn) * kLog2e);
  }
  __device__ inline void merge_wave(float scale) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      merge(__shfl_xor(m, o), __shfl_xor(st, o), DU ? __shfl_xor(s1, o) : 0.f, scale);
  }
};

// One workgroup per row and split: part[n * S + s] = {m, sum at T, sum at 1}.
// DU: both sums (a cross-entropy term beside a temperature other than 1).
// 4096 x 151936 bf16, 5% ignored, both sums: 195 us, 6.1 TB/s; bound by the vector
// units before the second exponential became a square (223 us), now by HBM.
template <typename T, bool DU>
__global__ __launch_bounds__(256) void kd_stream_kernel(const T* __restrict__ X, long ld, int V, int S, Teacher a,
                                                        float4* __restrict__ part) {
  __shared__ float red[4][3];
  const long n = blockIdx.x / S;
  const int s = blockIdx.x % S;
  int label;
  if (!row_counts(a, n, V, label)) return;
  int c0, c1;
  split_span(V, S, s, c0, c1);
  const T* const row = X + n * ld + c0;
  const RowSplit<T> sp(row, c1 - c0);
  const float scale = kLog2e * a.inv_t;
  const int tid = threadIdx.x;
  KdSums<DU> k;
  auto add1 = [&](float x) {
    k.rescale(fmaxf(k.m, x), scale);
    k.template add<0>(x, scale);
  };
  if (tid < sp.head) add1(elem_to_f32(row[tid]));
  if (tid < c1 - c0 - sp.tail_start) add1(elem_to_f32(row[sp.tail_start + tid]));
  for_each_chunk(reinterpret_cast<const u32x4*>(row + sp.head), sp.chunks, tid, [&](int, const u32x4& raw) {
    const T* v = reinterpret_cast<const T*>(&raw);
    float x[RowSplit<T>::E], mx = k.m;
#pragma unroll
    for (int e = 0; e < RowSplit<T>::E; ++e) {
      x[e] = elem_to_f32(v[e]);
      mx = fmaxf(mx, x[e]);
    }
    k.rescale(mx, scale);
    auto all = [&](auto SQ) {
#pragma unroll
      for (int e = 0; e < RowSplit<T>::E; ++e) k.template add<decltype(SQ)::value>(x[e], scale);
    };
    if (!DU || a.squares == 0)
      all(std::integral_constant<int, 0>{});
    else if (a.squares == 1)
      all(std::integral_constant<int, 1>{});
    else
      all(std::integral_constant<int, 2>{});
  });
  k.merge_wave(scale);
  if ((tid & 63) == 0) {
    red[tid >> 6][0] = k.m;
    red[tid >> 6][1] = k.st;
    red[tid >> 6][2] = k.s1;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 4; ++w) k.merge(red[w][0], red[w][1], red[w][2], scale);
    part[blockIdx.x] = make_float4(k.m, k.st, k.s1, 0.f);
  }
}

// One workgroup per row: joins the splits and forms the row's loss (K scattered
// reads a row, 15 us for 4096 rows of K = 64).
// stats[n] = {m, log2 of the sum at T, log2 of the sum at 1, 0}.
template <typename T, bool DU>
__global__ __launch_bounds__(256) void kd_loss_kernel(const T* __restrict__ X, long ld, int V, int S, Teacher a,
                                                      const float4* __restrict__ part, float4* __restrict__ stats,
                                                      float* __restrict__ rowloss, float* __restrict__ bsum,
                                                      int* __restrict__ bcnt) {
  __shared__ Entries e;
  const long n = blockIdx.x;
  const int tid = threadIdx.x;
  int label, col;
  if (!row_counts(a, n, V, label)) {
    if (tid == 0) {
      stats[n] = make_float4(0.f, 0.f, 0.f, 0.f);
      rowloss[n] = bsum[n] = 0.f;
      bcnt[n] = 0;
    }
    return;
  }
  const float scale = kLog2e * a.inv_t;
  KdSums<DU> k;
  for (int s = tid & 63; s < S; s += 64) {
    const float4 p = part[n * S + s];
    k.merge(p.x, p.y, p.z, scale);
  }
  k.merge_wave(scale);
  const float s1 = DU ? k.s1 : k.st;  // T == 1, or not used
  float q, lq;
  load_entries(a, n, V, e, col, q, lq);
  // an entry without weight adds nothing, also where the student gives its column nothing
  float term = 0.f;
  if (col >= 0 && q != 0.f && a.kd != 0.f) term = q * (lq + (logf(k.st) - (elem_to_f32(X[n * ld + col]) - k.m) * a.inv_t));
  const float sum = block_sum(term, e.red);
  if (tid == 0) {
    float loss = a.kd * sum;
    if (a.ce != 0.f) loss += a.ce * (logf(s1) + (label >= 0 ? k.m - elem_to_f32(X[n * ld + label]) : k.m));
    stats[n] = make_float4(k.m, log2f(k.st), log2f(s1), 0.f);
    rowloss[n] = bsum[n] = loss;
    bcnt[n] = 1;
  }
}

// The factor of row n's gradient.
__device__ inline float grad_factor(const float* grad_out, const int32_t* n_valid, int reduction, long n) {
  const float g = reduction == CCE_REDUCTION_NONE ? grad_out[n] : grad_out[0];
  return reduction == CCE_REDUCTION_MEAN ? g / (float)(n_valid[0] > 1 ? n_valid[0] : 1) : g;
}

// One workgroup per row and split writes the split's columns of dX: the dense
// part, then, behind a barrier, the columns of the entries and of the label.
// 4096 x 151936 bf16: 489 us for 2.43 GB, the rate of a large copy.
template <typename T, bool DU>
__global__ __launch_bounds__(256) void kd_grad_kernel(const float* __restrict__ grad_out, const T* __restrict__ X,
                                                      long ld, int V, int S, Teacher a,
                                                      const float4* __restrict__ stats,
                                                      const int32_t* __restrict__ n_valid, int reduction,
                                                      T* __restrict__ dX, long ldg) {
  __shared__ Entries e;
  const long n = blockIdx.x / S;
  const int tid = threadIdx.x;
  int c0, c1, label, col;
  split_span(V, S, blockIdx.x % S, c0, c1);
  T* const drow = dX + n * ldg + c0;
  if (!row_counts(a, n, V, label)) {
    zero_row<256>(drow, c1 - c0, tid);
    return;
  }
  float q, lq;
  const bool any = load_entries(a, n, V, e, col, q, lq);
  const float g = grad_factor(grad_out, n_valid, reduction, n);
  const float4 st = stats[n];
  const float scale = kLog2e * a.inv_t;
  const float ce = g * a.ce, kdg = any ? g * a.kdg : 0.f;
  const float cp = DU ? kdg : kdg + ce;  // without DU both softmaxes are one, or ce is 0
  auto dense = [&](float x) {
    const float u = x - st.x;
    float v = cp * fast_exp2(__builtin_fmaf(u, scale, -st.y));
    if constexpr (DU) v = __builtin_fmaf(ce, fast_exp2(__builtin_fmaf(u, kLog2e, -st.z)), v);
    return v;
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
    for_each_chunk(reinterpret_cast<const u32x4*>(row + sp.head), sp.chunks, tid, [&](int c, const u32x4& raw) {
      const T* v = reinterpret_cast<const T*>(&raw);
      u32x4 out;
      T* o = reinterpret_cast<T*>(&out);
#pragma unroll
      for (int i = 0; i < RowSplit<T>::E; ++i) o[i] = f32_to_elem<T>(dense(elem_to_f32(v[i])));
      __builtin_nontemporal_store(out, dbody + c);
    });
  }
  __syncthreads();
  auto sparse = [&](int c) {
    if (c < c0 || c >= c1) return;
    float v = dense(elem_to_f32(row[c - c0])) - kdg * entries_at(e, a.K, c);
    if (c == label) v -= ce;
    drow[c - c0] = f32_to_elem<T>(v);
  };
  // entries that share a column, and the label among them, write the same value
  if (col >= 0) sparse(col);
  if (tid == 0 && label >= 0 && ce != 0.f) sparse(label);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int check_teacher(const cce_teacher* t, long N, const void* labels, int64_t ignore_index, int labels_int64,
                  Teacher& a) {
  if (!t) return fail(CCE_ERR_INVALID_ARG, "teacher must not be null");
  if (t->entries < 1 || t->entries > kMaxEntries)
    return fail(CCE_ERR_INVALID_ARG, "a teacher has 1 to %d entries per row (got %ld)", kMaxEntries,
                (long)t->entries);
  if (!logits_elem_size(t->logits_dtype))
    return fail(CCE_ERR_INVALID_ARG, "the teacher's logits must be CCE_DTYPE_BF16, CCE_DTYPE_F16 or CCE_DTYPE_F32");
  if (!(t->temperature >= 1e-2f && t->temperature <= 1e3f))
    return fail(CCE_ERR_INVALID_ARG, "temperature must be in [0.01, 1000] (got %g)", (double)t->temperature);
  if (!(fabsf(t->distill_weight) < INFINITY) || !(fabsf(t->ce_weight) < INFINITY))
    return fail(CCE_ERR_INVALID_ARG, "distill_weight and ce_weight must be finite");
  // without rows, labels that were given may well be at a null address
  if (N > 0 && t->ce_weight != 0.f && !labels) return fail(CCE_ERR_INVALID_ARG, "ce_weight needs labels");
  if (N > 0 && (!t->logits || !t->indices))
    return fail(CCE_ERR_INVALID_ARG, "the teacher's logits and indices must not be null");
  a.t = t->logits;
  a.tdtype = t->logits_dtype;
  a.index = t->indices;
  a.index64 = t->indices_int64;
  a.K = (int)t->entries;
  a.labels = labels;
  a.labels64 = labels_int64;
  a.ignore_index = (long)ignore_index;
  a.inv_t = 1.f / t->temperature;
  a.kd = t->distill_weight * t->temperature * t->temperature;
  a.kdg = t->distill_weight * t->temperature;
  a.ce = t->ce_weight;
  a.squares = t->temperature == 2.f ? 1 : t->temperature == 4.f ? 2 : 0;
  return CCE_OK;
}

// Both softmaxes are needed: at the temperature and, for the labels, at 1.
bool two_softmaxes(const Teacher& a) { return a.ce != 0.f && a.inv_t != 1.f; }

// What the GEMM epilogues compute for it.
int softmaxes_of(const Teacher& a) {
  return two_softmaxes(a) ? kTwoSoftmaxes : a.inv_t == 1.f ? kOneSoftmax : kAtTemperature;
}

// Workgroups per row: enough for the card's CUs where there are few rows, with at
// least 4096 columns each.
int kd_splits(long N, long V) {
  const long s = std::min(ceil_div(4096, std::max<long>(N, 1)), V / 4096);
  return (int)std::max<long>(s, 1);
}

struct KdLayout {
  float4* part;
  float *rowloss, *bsum;
  int* bcnt;
  size_t bytes;
};

KdLayout kd_layout(void* ws, long N, long V) {
  Carver c(ws);
  KdLayout L;
  const size_t n = (size_t)std::max<long>(N, 1);
  L.part = c.take<float4>(n * kd_splits(N, V));
  L.rowloss = c.take<float>(n);
  L.bsum = c.take<float>(n);
  L.bcnt = c.take<int>(n);
  L.bytes = align_up(c.off, 256);
  return L;
}

// Calls f(T()) for a type of logits.
template <typename F>
int logits_type(int dtype, F&& f) {
  if (dtype == CCE_DTYPE_BF16) return f((uint16_t)0);
  if (dtype == CCE_DTYPE_F16) return f((_Float16)0);
  return f(0.f);
}

template <typename T, bool DU>
int kd_forward_run(const T* X, long ld, long N, long V, const Teacher& a, int reduction, float* loss_out,
                   float4* stats, int32_t* n_valid, const KdLayout& L, hipStream_t st) {
  const int S = kd_splits(N, V);
  float* const rowloss = reduction == CCE_REDUCTION_NONE ? loss_out : L.rowloss;
  if (N > 0) {
    hipLaunchKernelGGL((kd_stream_kernel<T, DU>), dim3((unsigned)(N * S)), dim3(256), 0, st, X, ld, (int)V, S, a, L.part);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((kd_loss_kernel<T, DU>), dim3((unsigned)N), dim3(256), 0, st, X, ld, (int)V, S, a, L.part,
                       stats, rowloss, L.bsum, L.bcnt);
    HIP_TRY(hipGetLastError());
  }
  hipLaunchKernelGGL(fwd_finalize_kernel, dim3(1), dim3(1024), 0, st, L.bsum, L.bcnt, (int)N, reduction, loss_out,
                     n_valid);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}

template <typename T, bool DU>
int kd_backward_run(const float* grad_out, const T* X, long ld, long N, long V, const Teacher& a, const float4* stats,
                    const int32_t* n_valid, int reduction, T* dX, long ldg, hipStream_t st) {
  const int S = kd_splits(N, V);
  hipLaunchKernelGGL((kd_grad_kernel<T, DU>), dim3((unsigned)(N * S)), dim3(256), 0, st, grad_out, X, ld, (int)V, S, a,
                     stats, n_valid, reduction, dX, ldg);
  HIP_TRY(hipGetLastError());
  return CCE_OK;
}
