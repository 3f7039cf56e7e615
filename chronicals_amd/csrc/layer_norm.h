// Layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / D;  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)
//   n = (x - mean) * rstd;  y = n * w + b
//   a = dy * w;  dx = rstd * (a - sum(a) / D - n * sum(a * n) / D)
//   dw = sum over rows of dy * n;  db = sum over rows of dy
//
// Statistics, sums and every intermediate are fp32; y and dx are rounded once
// to the type of x, dw and db to the type of w.  All of it is bound by HBM: the
// forward reads x and writes y, the backward reads x and dy and writes dx.

// One workgroup per row: three passes over the row (its second and third reads
// come from the caches).
template <typename T, typename W>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(const T* __restrict__ X, long ldx, const W* __restrict__ w,
                                                             const W* __restrict__ b, int D, float eps,
                                                             T* __restrict__ Y, float* __restrict__ mean_out,
                                                             float* __restrict__ rstd_out) {
  __shared__ float red[4];
  const long n = blockIdx.x;
  const T* const x = X + n * ldx;
  float s = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) s += elem_to_f32(x[c]);
  const float mean = block_sum(s, red) / (float)D;
  s = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float v = elem_to_f32(x[c]) - mean;
    s += v * v;
  }
  const float rstd = 1.f / sqrtf(block_sum(s, red) / (float)D + eps);
  T* const y = Y + n * D;
  for (int c = threadIdx.x; c < D; c += 256) {
    float v = (elem_to_f32(x[c]) - mean) * rstd;
    if (w) v *= elem_to_f32(w[c]);
    if (b) v += elem_to_f32(b[c]);
    y[c] = f32_to_elem<T>(v);
  }
  if (threadIdx.x == 0) {
    mean_out[n] = mean;
    rstd_out[n] = rstd;
  }
}

// dx: one workgroup per row.
template <typename T, typename W>
__global__ __launch_bounds__(256) void layer_norm_dx_kernel(const T* __restrict__ dY, const T* __restrict__ X, long ldx,
                                                            const W* __restrict__ w, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, int D,
                                                            T* __restrict__ dX) {
  __shared__ float red[4];
  const long n = blockIdx.x;
  const T* const x = X + n * ldx;
  const T* const dy = dY + n * D;
  const float mu = mean[n], r = rstd[n];
  float sa = 0.f, san = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float a = elem_to_f32(dy[c]) * (w ? elem_to_f32(w[c]) : 1.f);
    sa += a;
    san += a * ((elem_to_f32(x[c]) - mu) * r);
  }
  sa = block_sum(sa, red) / (float)D;
  san = block_sum(san, red) / (float)D;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float a = elem_to_f32(dy[c]) * (w ? elem_to_f32(w[c]) : 1.f);
    dX[n * D + c] = f32_to_elem<T>(r * (a - sa - (elem_to_f32(x[c]) - mu) * r * san));
  }
}

// dw and db over the rows [part * rows, (part + 1) * rows), part = blockIdx.y,
// one column per thread.
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_parts_kernel(const T* __restrict__ dY, const T* __restrict__ X,
                                                               long ldx, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, long N, int D, long rows,
                                                               float* __restrict__ dw, float* __restrict__ db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  const long n0 = blockIdx.y * rows, n1 = min(n0 + rows, N);
  float sw = 0.f, sb = 0.f;
  for (long n = n0; n < n1; ++n) {
    const float g = elem_to_f32(dY[n * D + c]);
    sw += g * ((elem_to_f32(X[n * ldx + c]) - mean[n]) * rstd[n]);
    sb += g;
  }
  dw[(long)blockIdx.y * D + c] = sw;
  db[(long)blockIdx.y * D + c] = sb;
}

// The parts' sums, in order, rounded to the parameters' type.
template <typename W>
__global__ __launch_bounds__(256) void layer_norm_join_kernel(const float* __restrict__ pw, const float* __restrict__ pb,
                                                              int parts, int D, W* __restrict__ dw,
                                                              W* __restrict__ db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  float sw = 0.f, sb = 0.f;
  for (int p = 0; p < parts; ++p) {
    sw += pw[(long)p * D + c];
    sb += pb[(long)p * D + c];
  }
  if (dw) dw[c] = f32_to_elem<W>(sw);
  if (db) db[c] = f32_to_elem<W>(sb);
}

constexpr long kNormMaxD = 1L << 20;

int check_norm(int64_t N, int64_t D, int dtype, int64_t ldx, int wdtype) {
  if (N < 0 || N > 0x7fffffffL) return fail(CCE_ERR_INVALID_ARG, "N must be in [0, 2^31) (got %ld)", (long)N);
  if (D <= 0 || D > kNormMaxD) return fail(CCE_ERR_INVALID_ARG, "D must be in [1, 2^20] (got %ld)", (long)D);
  if (!logits_elem_size(dtype))
    return fail(CCE_ERR_INVALID_ARG, "dtype must be CCE_DTYPE_BF16, CCE_DTYPE_F16 or CCE_DTYPE_F32");
  if (wdtype != dtype && wdtype != CCE_DTYPE_F32)
    return fail(CCE_ERR_INVALID_ARG, "the parameters' dtype must be the input's or CCE_DTYPE_F32, got %d", wdtype);
  if (N > 1 && ldx < D) return fail(CCE_ERR_INVALID_ARG, "row stride %ld is smaller than D = %ld", (long)ldx, (long)D);
  return CCE_OK;
}

struct NormLayout {
  int parts;
  long rows;
  float *dw, *db;
  size_t bytes;
};

NormLayout norm_layout(void* ws, long N, long D) {
  Carver c(ws);
  NormLayout L;
  L.rows = std::max<long>(64, ceil_div(std::max<long>(N, 1), 256));
  L.parts = (int)ceil_div(std::max<long>(N, 1), L.rows);
  L.dw = c.take<float>((size_t)L.parts * D);
  L.db = c.take<float>((size_t)L.parts * D);
  L.bytes = align_up(c.off, 256);
  return L;
}

// Calls f(T(), W()) for the types of the input and of the parameters.
template <typename F>
int norm_types(int dtype, int wdtype, F&& f) {
  if (dtype == CCE_DTYPE_BF16) return wdtype == dtype ? f((uint16_t)0, (uint16_t)0) : f((uint16_t)0, 0.f);
  if (dtype == CCE_DTYPE_F16) return wdtype == dtype ? f((_Float16)0, (_Float16)0) : f((_Float16)0, 0.f);
  return f(0.f, 0.f);
}

int norm_forward(const void* x, int dtype, int64_t ldx, const void* weight, const void* bias, int wdtype, int64_t N,
                 int64_t D, float eps, void* y, float* mean, float* rstd, hipStream_t st) {
  return norm_types(dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W>), dim3((unsigned)N), dim3(256), 0, st, static_cast<const T*>(x),
                       (long)ldx, static_cast<const W*>(weight), static_cast<const W*>(bias), (int)D, eps,
                       static_cast<T*>(y), mean, rstd);
    HIP_TRY(hipGetLastError());
    return CCE_OK;
  });
}

int norm_backward(const void* dy, const void* x, int dtype, int64_t ldx, const void* weight, int wdtype,
                  const float* mean, const float* rstd, int64_t N, int64_t D, void* dx, void* dw, void* db,
                  const NormLayout& L, hipStream_t st) {
  return norm_types(dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    if (dx && N > 0) {
      hipLaunchKernelGGL((layer_norm_dx_kernel<T, W>), dim3((unsigned)N), dim3(256), 0, st, static_cast<const T*>(dy),
                         static_cast<const T*>(x), (long)ldx, static_cast<const W*>(weight), mean, rstd, (int)D,
                         static_cast<T*>(dx));
      HIP_TRY(hipGetLastError());
    }
    if (!dw && !db) return CCE_OK;
    hipLaunchKernelGGL(layer_norm_parts_kernel<T>, dim3((unsigned)ceil_div(D, 256), (unsigned)L.parts), dim3(256), 0,
                       st, static_cast<const T*>(dy), static_cast<const T*>(x), (long)ldx, mean, rstd, (long)N, (int)D,
                       L.rows, L.dw, L.db);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(layer_norm_join_kernel<W>, dim3((unsigned)ceil_div(D, 256)), dim3(256), 0, st, L.dw, L.db,
                       L.parts, (int)D, static_cast<W*>(dw), static_cast<W*>(db));
    HIP_TRY(hipGetLastError());
    return CCE_OK;
  });
}
