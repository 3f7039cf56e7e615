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
//
// The mean m of the first sum is off by its rounding, which for rows far from 0
// is no little part of sqrt(eps) or of the variation.  So the second pass sums
// x - m beside its square: their mean e completes the first, x - m - e is what is
// normalised, and the variance is mean((x - m)^2) - e^2.  fp32 rows of 1000.1 came
// out as 0.013 at D = 896 and 0.26 at D = 20000, and come out as 0.  The second sum
// costs the forward 0.4 us of 13.4 (16384 x 896 bf16) to 3 of 37 (2048 x 16384).
//
// Rows stay in registers: TR threads hold up to C chunks of 16 bytes each, a wave
// per row up to 256 chunks, then a workgroup of 256 or 1024.  A workgroup goes on
// to further rows with the parameters in its registers, and in the backward with
// its share of dw and db there too.  Rows need no alignment (16-byte accesses at
// the element's), and a last chunk that is not whole goes element by element.
// Longer rows go by the kernels below, which read them two or three times.
//
// Forward / backward with the join of its parts (TB/s of what has to move): 16384 x
// 896 bf16 14 / 26 us (4.1 / 3.4), 65536 x 896 44 / 71 us (5.4 / 5.0), 8192 x 4096
// fp32 47 / 79 us (5.8 / 5.1), 8192 x 1001 bf16 13 / 26 us.  Reading each row two or
// three times, a column per thread for dw and db: 16384 x 896 48 / 137 us.

// Sixteen bytes at any element.
typedef u32x4 loose_u32x4 __attribute__((aligned(2)));
typedef f32x4 loose_f32x4 __attribute__((aligned(4)));

// Sums of two values over the TR threads of a row (fixed order).
template <int TR>
__device__ inline void row_sums(float& a, float& b, float (*red)[2]) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  if constexpr (TR > 64) {
    __syncthreads();  // red may still be read by the sum before
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6][0] = a;
      red[threadIdx.x >> 6][1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < TR / 64; ++w) {
      a += red[w][0];
      b += red[w][1];
    }
  }
}

// The chunks of a row of D elements that thread t of TR holds, as fp32: chunk t +
// c * TR.  Elements past the row's end are 0.
template <typename T, int TR, int C>
struct RowRegs {
  static constexpr int E = 16 / sizeof(T);
  float v[C][E];
  static __device__ inline int first(int c, int t) { return (t + c * TR) * E; }
  // a row's whole chunks on their way
  struct Raw {
    u32x4 v[C];
    __device__ inline void issue(const T* row, int D, int t) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        v[c] = u32x4{0u, 0u, 0u, 0u};
        if (first(c, t) + E <= D)
          v[c] = __builtin_nontemporal_load(reinterpret_cast<const loose_u32x4*>(row + first(c, t)));
      }
    }
  };
  __device__ inline void take(const Raw& raw, const T* row, int D, int t) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const T* e = reinterpret_cast<const T*>(&raw.v[c]);
#pragma unroll
      for (int i = 0; i < E; ++i) v[c][i] = elem_to_f32(e[i]);
    }
    tail(D, t, [&](float& x, int at) { x = elem_to_f32(row[at]); });
  }
  // f(value, position) for the elements of a last chunk that is not whole
  template <typename F>
  __device__ inline void tail(int D, int t, F&& f) {
    if (D % E == 0) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (first(c, t) >= D || first(c, t) + E <= D) continue;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (first(c, t) + i < D) f(v[c][i], first(c, t) + i);
    }
  }
  // parameters, fp32 or of type T (null: `none`)
  __device__ inline void load_params(const void* p, int f32, int D, int t, float none) {
    if (p && !f32) {
      Raw raw;
      raw.issue(static_cast<const T*>(p), D, t);
      take(raw, static_cast<const T*>(p), D, t);
      return;
    }
    const float* const q = static_cast<const float*>(p);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; i += 4) {
        f32x4 e = {none, none, none, none};
        if (p && first(c, t) + E <= D) e = *reinterpret_cast<const loose_f32x4*>(q + first(c, t) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[c][i + k] = e[k];
      }
    if (p) tail(D, t, [&](float& x, int at) { x = q[at]; });
  }
  __device__ inline void store(T* row, int D, int t) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      u32x4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < E; ++i) e[i] = f32_to_elem<T>(v[c][i]);
      if (first(c, t) + E <= D) __builtin_nontemporal_store(raw, reinterpret_cast<loose_u32x4*>(row + first(c, t)));
    }
    tail(D, t, [&](float& x, int at) { row[at] = f32_to_elem<T>(x); });
  }
};

// 1 / sqrt(var + eps) from the mean of the squared differences and that of the
// differences.  Rounding may leave less than 0 of a row without variation.
__device__ inline float norm_rstd(float square, float rest, float eps) {
  const float var = __builtin_fmaf(-rest, rest, square);
  return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);
}

template <typename T, int TR, int C>
__global__ __launch_bounds__(TR < 256 ? 256 : TR) void layer_norm_fwd_rows_kernel(
    const T* __restrict__ X, long ldx, const void* __restrict__ w, const void* __restrict__ b, int param_f32, long N,
    int D, float eps, T* __restrict__ Y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  typedef RowRegs<T, TR, C> Row;
  constexpr int kRows = TR < 256 ? 256 / TR : 1;  // rows of a workgroup at a time
  __shared__ float red[TR / 64][2];
  const int t = threadIdx.x % TR;
  const float inv = 1.f / (float)D;
  Row wr, br;
  wr.load_params(w, param_f32, D, t, 1.f);
  br.load_params(b, param_f32, D, t, 0.f);
  for (long n = (long)blockIdx.x * kRows + threadIdx.x / TR; n < N; n += (long)gridDim.x * kRows) {
#pragma clang fp contract(off)  // the mean is subtracted as it is rounded and kept, not as a product fused
    Row x;
    typename Row::Raw raw;
    raw.issue(X + n * ldx, D, t);
    x.take(raw, X + n * ldx, D, t);
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < Row::E; ++i) s += x.v[c][i];
    row_sums<TR>(s, q, red);
    const float mean = s * inv;
    s = q = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < Row::E; ++i) {
        x.v[c][i] = Row::first(c, t) + i < D ? x.v[c][i] - mean : 0.f;
        s += x.v[c][i];
        q = __builtin_fmaf(x.v[c][i], x.v[c][i], q);
      }
    row_sums<TR>(s, q, red);
    const float rest = s * inv, rstd = norm_rstd(q * inv, rest, eps), off = -rest * rstd;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < Row::E; ++i) x.v[c][i] = __builtin_fmaf(__builtin_fmaf(x.v[c][i], rstd, off), wr.v[c][i], br.v[c][i]);
    x.store(Y + n * D, D, t);
    if (t == 0) {
      mean_out[n] = mean + rest;
      rstd_out[n] = rstd;
    }
  }
}

// dx, and the workgroup's sums of dw and db over its rows at part[blockIdx.x].
template <typename T, int TR, int C>
__global__ __launch_bounds__(TR < 256 ? 256 : TR) void layer_norm_bwd_rows_kernel(
    const T* __restrict__ dY, const T* __restrict__ X, long ldx, const void* __restrict__ w, int param_f32,
    const float* __restrict__ mean, const float* __restrict__ rstd, long N, int D, T* __restrict__ dX,
    float* __restrict__ dw, float* __restrict__ db) {
  typedef RowRegs<T, TR, C> Row;
  constexpr int kRows = TR < 256 ? 256 / TR : 1, E = Row::E;
  __shared__ float red[TR / 64][2];
  const int t = threadIdx.x % TR;
  const float inv = 1.f / (float)D;
  Row wr;
  wr.load_params(w, param_f32, D, t, 1.f);
  float sw[C][E] = {}, sb[C][E] = {};
  const long step = (long)gridDim.x * kRows;
  long n = (long)blockIdx.x * kRows + threadIdx.x / TR;
  typename Row::Raw raw_x, raw_g;
  float next_mu = 0.f, next_r = 0.f;
  auto issue = [&](long m) {
    raw_x.issue(X + m * ldx, D, t);
    raw_g.issue(dY + m * D, D, t);
    next_mu = mean[m];
    next_r = rstd[m];
  };
  constexpr bool kAhead = TR < 1024;  // 1024 threads have no registers for it
  if (kAhead && n < N) issue(n);
  for (; n < N; n += step) {
    if (!kAhead) issue(n);
    Row x, g;
    x.take(raw_x, X + n * ldx, D, t);
    g.take(raw_g, dY + n * D, D, t);
    const float mu = next_mu, r = next_r;
    if (kAhead && n + step < N) issue(n + step);  // the next row, while this one is worked on
    float sa = 0.f, san = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        // past the row's end g is 0, so x there does not count
        x.v[c][i] = (x.v[c][i] - mu) * r;
        sw[c][i] = __builtin_fmaf(g.v[c][i], x.v[c][i], sw[c][i]);
        sb[c][i] += g.v[c][i];
        g.v[c][i] *= wr.v[c][i];
        sa += g.v[c][i];
        san = __builtin_fmaf(g.v[c][i], x.v[c][i], san);
      }
    if (!dX) continue;
    row_sums<TR>(sa, san, red);
    sa *= inv;
    san *= inv;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; ++i) x.v[c][i] = r * (g.v[c][i] - sa - x.v[c][i] * san);
    x.store(dX + n * D, D, t);
  }
  if (!dw) return;
  // the rows' sums within the workgroup, one after the other
  if constexpr (kRows > 1) {
    __shared__ float sums[2][TR * C * E];
    for (int k = 0; k < kRows; ++k) {
      if (threadIdx.x / TR == k) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const int at = (c * E + i) * TR + t;
            sums[0][at] = sw[c][i] = k ? sums[0][at] + sw[c][i] : sw[c][i];
            sums[1][at] = sb[c][i] = k ? sums[1][at] + sb[c][i] : sb[c][i];
          }
      }
      __syncthreads();
    }
    if (threadIdx.x / TR != kRows - 1) return;
  }
  dw += (long)blockIdx.x * D;
  db += (long)blockIdx.x * D;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const int at = Row::first(c, t) + i;
      if (at + 4 <= D) {
        *reinterpret_cast<loose_f32x4*>(dw + at) = f32x4{sw[c][i], sw[c][i + 1], sw[c][i + 2], sw[c][i + 3]};
        *reinterpret_cast<loose_f32x4*>(db + at) = f32x4{sb[c][i], sb[c][i + 1], sb[c][i + 2], sb[c][i + 3]};
        continue;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + k < D) {
          dw[at + k] = sw[c][i + k];
          db[at + k] = sb[c][i + k];
        }
    }
}

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
  float q = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float v = elem_to_f32(x[c]) - mean;
    s += v;
    q += v * v;
  }
  const float rest = block_sum(s, red) / (float)D;
  const float rstd = norm_rstd(block_sum(q, red) / (float)D, rest, eps);
  T* const y = Y + n * D;
  for (int c = threadIdx.x; c < D; c += 256) {
    float v = (elem_to_f32(x[c]) - mean - rest) * rstd;
    if (w) v *= elem_to_f32(w[c]);
    if (b) v += elem_to_f32(b[c]);
    y[c] = f32_to_elem<T>(v);
  }
  if (threadIdx.x == 0) {
    mean_out[n] = mean + rest;
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

// The parts' sums, rounded to the parameters' type: blockIdx.y 0: dw, 1: db.  16
// columns per workgroup, each by 16 threads that take every 16th part.
template <typename W>
__global__ __launch_bounds__(256) void layer_norm_join_kernel(const float* __restrict__ pw, const float* __restrict__ pb,
                                                              int parts, int D, W* __restrict__ dw,
                                                              W* __restrict__ db) {
  __shared__ float sums[16][17];
  W* const out = blockIdx.y ? db : dw;
  if (!out) return;
  const float* const p = blockIdx.y ? pb : pw;
  const int x = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int k = g; k < parts; k += 16) s += p[(long)k * D + c];
  }
  sums[g][x] = s;
  __syncthreads();
  if (g != 0 || c >= D) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += sums[k][x];
  out[c] = f32_to_elem<W>(s);
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

// Workgroups of a forward.
constexpr long kNormGroups = 1024;

// Workgroups of a backward, each with a part of dw and db: enough to fill the
// card, few enough that the parts are little next to the rows, which with a wave
// per row they are from 32 rows each on (8192 x 2048 bf16: 256 parts 31 us, 512
// 37; 16384 x 896: 34, 26; 65536 x 896 with 256, 512, 768: 118, 81, 73; a
// workgroup per row, 8192 x 4096: 69, 53, 51, and of 1024 threads, 2048 x 16384:
// 60, 78, 78).
constexpr long kNormParts = 768;
long most_norm_parts(long N, long D) {  // and no more than 128 MiB of them
  return std::max<long>(1, std::min({N, kNormParts, (1L << 24) / D}));
}
long norm_parts(long N, long D, int threads) {
  const long parts = threads == 64 ? std::min(std::max(N / 32, 256L), kNormParts) : threads == 256 ? 512 : 256;
  return std::max<long>(1, std::min({parts, threads == 64 ? ceil_div(N, 4) : N, most_norm_parts(N, D)}));
}

struct NormLayout {
  float *dw, *db;
  size_t bytes;
};

NormLayout norm_layout(void* ws, long parts, long D) {
  Carver c(ws);
  NormLayout L;
  L.dw = c.take<float>((size_t)(parts * D));
  L.db = c.take<float>((size_t)(parts * D));
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

// Calls f(TR, C) as integral constants for rows of D elements of E to a chunk;
// false: more than kMost.
template <int E, int kMost, typename F>
bool norm_shape(long D, F&& f) {
  const long chunks = ceil_div(D, E);
  auto by = [&](auto tr) {
    constexpr int TR = decltype(tr)::value;
    if constexpr (TR * 2 * E < kMost) {
      if (chunks > TR * 2) return f(tr, std::integral_constant<int, 4>{});
    }
    f(tr, std::integral_constant<int, 2>{});
  };
  if (D > kMost) return false;
  if (chunks <= 64 * 4)
    by(std::integral_constant<int, 64>{});
  else if (chunks <= 256 * 4)
    by(std::integral_constant<int, 256>{});
  else
    by(std::integral_constant<int, 1024>{});
  return true;
}

// The longest rows that stay in registers, forward and backward: 16 elements in
// each of 1024 threads, past which both spill.  It is the backward's limit: 1024 x
// 20000 bf16 took 175 us with 370 registers in memory, and takes 134 to 152 by the
// kernels for longer rows.  The forward has no limit of its own: with 18 registers
// in memory it took 36 us there, and takes 98 by those kernels.
constexpr int kNormRegD = 1024 * 16;

// Threads of a row of D elements in registers; 256 for longer ones, whose parts
// are as many.
int norm_threads(int dtype, long D) {
  int threads = 256;
  auto shape = [&](auto tr, auto) { threads = decltype(tr)::value; };
  if (dtype == CCE_DTYPE_F32)
    norm_shape<4, kNormRegD>(D, shape);
  else
    norm_shape<8, kNormRegD>(D, shape);
  return threads;
}

// What one backward uses: nothing where neither dw nor db is wanted.
size_t norm_bytes(int dtype, long N, long D, bool params) {
  return params ? norm_layout(nullptr, norm_parts(N, D, norm_threads(dtype, D)), D).bytes : 0;
}

int norm_forward(const void* x, int dtype, int64_t ldx, const void* weight, const void* bias, int wdtype, int64_t N,
                 int64_t D, float eps, void* y, float* mean, float* rstd, hipStream_t st) {
  return norm_types(dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    const bool in_registers = norm_shape<16 / sizeof(T), kNormRegD>(D, [&](auto tr, auto c) {
      constexpr int TR = decltype(tr)::value, kRows = TR < 256 ? 256 / TR : 1;
      const unsigned grid = (unsigned)std::min<long>(ceil_div(N, kRows), kNormGroups);
      hipLaunchKernelGGL((layer_norm_fwd_rows_kernel<T, TR, decltype(c)::value>), dim3(grid), dim3(std::max(TR, 256)), 0,
                         st, static_cast<const T*>(x), (long)ldx, weight, bias, (int)(wdtype == CCE_DTYPE_F32), (long)N,
                         (int)D, eps, static_cast<T*>(y), mean, rstd);
    });
    if (!in_registers)
      hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W>), dim3((unsigned)N), dim3(256), 0, st, static_cast<const T*>(x),
                         (long)ldx, static_cast<const W*>(weight), static_cast<const W*>(bias), (int)D, eps,
                         static_cast<T*>(y), mean, rstd);
    HIP_TRY(hipGetLastError());
    return CCE_OK;
  });
}

int norm_backward(const void* dy, const void* x, int dtype, int64_t ldx, const void* weight, int wdtype,
                  const float* mean, const float* rstd, int64_t N, int64_t D, void* dx, void* dw, void* db,
                  void* workspace, hipStream_t st) {
  return norm_types(dtype, wdtype, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    const bool params = dw || db;
    if (!dx && !params) return CCE_OK;
    const long parts = norm_parts(N, D, norm_threads(dtype, D));
    const NormLayout L = norm_layout(params ? workspace : nullptr, parts, D);
    const bool in_registers = norm_shape<16 / sizeof(T), kNormRegD>(D, [&](auto tr, auto c) {
      constexpr int TR = decltype(tr)::value;
      hipLaunchKernelGGL((layer_norm_bwd_rows_kernel<T, TR, decltype(c)::value>), dim3((unsigned)parts),
                         dim3(std::max(TR, 256)), 0, st, static_cast<const T*>(dy), static_cast<const T*>(x), (long)ldx,
                         weight, (int)(wdtype == CCE_DTYPE_F32), mean, rstd, (long)N, (int)D, static_cast<T*>(dx),
                         L.dw, L.db);
    });
    HIP_TRY(hipGetLastError());
    if (!in_registers && dx && N > 0) {
      hipLaunchKernelGGL((layer_norm_dx_kernel<T, W>), dim3((unsigned)N), dim3(256), 0, st, static_cast<const T*>(dy),
                         static_cast<const T*>(x), (long)ldx, static_cast<const W*>(weight), mean, rstd, (int)D,
                         static_cast<T*>(dx));
      HIP_TRY(hipGetLastError());
    }
    if (!params) return CCE_OK;
    if (!in_registers) {
      hipLaunchKernelGGL(layer_norm_parts_kernel<T>, dim3((unsigned)ceil_div(D, 256), (unsigned)parts), dim3(256), 0,
                         st, static_cast<const T*>(dy), static_cast<const T*>(x), (long)ldx, mean, rstd, (long)N, (int)D,
                         ceil_div(N, parts), L.dw, L.db);
      HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(layer_norm_join_kernel<W>, dim3((unsigned)ceil_div(D, 16), 2), dim3(256), 0, st, L.dw, L.db,
                       (int)parts, (int)D, static_cast<W*>(dw), static_cast<W*>(db));
    HIP_TRY(hipGetLastError());
    return CCE_OK;
  });
}
