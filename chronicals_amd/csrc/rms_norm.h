// Root-mean-square norm over the last dimension with the residual's addition, forward,
// backward, and with an 8-bit output and its scales.
//
//   s = x + r (or x);  rstd = 1 / sqrt(sum(s^2) / D + eps);  n = s * rstd;  y = n * w
//   a = dy * w;  ds' = rstd * (a - n * sum(a * n) / D) + ds;  dx = dr = ds'
//   dw = sum over rows of dy * n
//   8 bits: scale = max(amax(|y|), 1e-30) / M over a row or a group of its columns,
//   q = round(y / scale), M = 448 (e4m3) or 127 (int8), y and the quotient in fp32
//
// s is rounded to the residual's type first, and what is normalised is the rounded
// one: it is what the caller keeps as the stream, what the backward reads, and what a
// model that adds and normalises in two steps would see.  Statistics, sums and all
// else are fp32; y, q and the gradients are rounded once.
//
// Rows stay in registers as in layer_norm.h, whose shapes these are; longer rows go by
// the kernels further below, which read them two or three times.
//
// Bound by HBM.  bf16 with a bf16 residual, forward / backward with both gradients and
// the join of its parts (TB/s of what has to move; a large copy reaches 4.8): 16384 x
// 896 24 / 29 us (4.9 / 4.1), 65536 x 896 81 / 88 (5.8 / 5.3), 8192 x 4096 48 / 53 (5.6 /
// 5.1), fp32 91 / 92 (5.9 / 5.8).  In 8 bits 8192 x 3584 40 to 42 us (5.0), by rows
// and by groups of 128 alike.  The backward without the next row's loads ahead: 16384 x 896 35.

// A row of type S on its way, in the chunks that RowRegs<T, TR, C> holds: 16 bytes of
// T, so fp32 beside a 16-bit T takes two loads a chunk.
template <typename T, typename S, int TR, int C>
struct RawChunks {
  static constexpr int E = 16 / sizeof(T), ES = 16 / sizeof(S);
  u32x4 v[C][E / ES];
  __device__ inline void issue(const S* row, int D, int t) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = RowRegs<T, TR, C>::first(c, t);
#pragma unroll
      for (int i = 0; i < E / ES; ++i) {
        v[c][i] = u32x4{0u, 0u, 0u, 0u};
        if (at + E <= D) v[c][i] = __builtin_nontemporal_load(reinterpret_cast<const loose_u32x4*>(row + at + i * ES));
      }
    }
  }
  // as fp32; 0 past the row's end
  __device__ inline void take(float (&x)[C][E], const S* row, int D, int t) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const S* e = reinterpret_cast<const S*>(v[c]);
#pragma unroll
      for (int i = 0; i < E; ++i) x[c][i] = elem_to_f32(e[i]);
    }
    if (D % E == 0) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = RowRegs<T, TR, C>::first(c, t);
      if (at >= D || at + E <= D) continue;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (at + i < D) x[c][i] = elem_to_f32(row[at + i]);
    }
  }
};

template <typename T, typename S, int TR, int C>
__device__ inline void load_chunks(float (&v)[C][16 / sizeof(T)], const S* row, int D, int t) {
  RawChunks<T, S, TR, C> raw;
  raw.issue(row, D, t);
  raw.take(v, row, D, t);
}

template <typename T, typename S, int TR, int C>
__device__ inline void store_chunks(const float (&v)[C][16 / sizeof(T)], S* row, int D, int t) {
  constexpr int E = 16 / sizeof(T), ES = 16 / sizeof(S);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = RowRegs<T, TR, C>::first(c, t);
    if (at + E <= D) {
#pragma unroll
      for (int i = 0; i < E / ES; ++i) {
        u32x4 raw;
        S* e = reinterpret_cast<S*>(&raw);
#pragma unroll
        for (int k = 0; k < ES; ++k) e[k] = f32_to_elem<S>(v[c][i * ES + k]);
        __builtin_nontemporal_store(raw, reinterpret_cast<loose_u32x4*>(row + at + i * ES));
      }
    } else if (at < D) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (at + i < D) row[at + i] = f32_to_elem<S>(v[c][i]);
    }
  }
}

// An 8-bit output.
struct RmsQuant {
  uint8_t* q;     // [N][D]
  float* scales;  // [N][groups]
  int group;      // columns that share a scale: 32, 64, 128, 256, or 0: a row's
  int shift;      // its base-2 logarithm
  int groups;     // of a row
  int int8;
  // whether a chunk's first column starts a group, and which
  __device__ inline bool starts(int at) const { return group && (at & (group - 1)) == 0; }
  __device__ inline long place(long n, int at) const { return n * groups + (at >> shift); }
};

// The scale of a group of largest magnitude amax, given as its bits: ordered as
// integers a NaN's are the largest, so that one in the group makes the scale a NaN.
__device__ inline float quant_scale(const RmsQuant& o, uint32_t amax) {
  const float a = __uint_as_float(amax);
  return (a < 1e-30f ? 1e-30f : a) / (o.int8 ? 127.f : 448.f);
}

// Quotients by a scale, from its reciprocal r and what that lacks, e = 1 - r scale (exact):
// v / scale = v r / (1 - e) is rounded once, from a value that is off by at most 2^-22 of
// a step of fp32 (e^2, and u's rounding).  v r alone is off by up to 1.5 steps, which takes
// values beside a midpoint of the 8-bit type to the wrong code.  8192 x 3584 bf16 into e4m3
// with a scale per row: v r alone 41 us, this 42, the compiler's division 47.
struct Quotient {
  float r, e;
  __device__ inline explicit Quotient(float scale) {
    r = 1.f / scale;
    // an infinite scale takes finite values to 0
    e = scale < INFINITY ? __builtin_fmaf(-r, scale, 1.f) : 0.f;
  }
  __device__ inline float of(float v) const {
    const float u = v * r * e;
    return __builtin_fmaf(v, r, u);
  }
};

__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values over their scale, rounded to nearest even: the quotients are at most M and
// a few 2^-24 of it, which round to M in either type (e4m3's midpoint above 448 is 464).
__device__ inline uint32_t quant4(const RmsQuant& o, const Quotient& by, const float* v) {
  const float a = by.of(v[0]), b = by.of(v[1]), c = by.of(v[2]), d = by.of(v[3]);
  if (o.int8) {
    // within the type also where a NaN has no integer (its group's scale is a NaN)
    auto whole = [](float v) { return (uint32_t)(int)rintf(__builtin_amdgcn_fmed3f(v, -127.f, 127.f)) & 255u; };
    return whole(a) | whole(b) << 8 | whole(c) << 16 | whole(d) << 24;
  }
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// The maximum over L neighbouring lanes (a power of two).
__device__ inline uint32_t lanes_max(uint32_t v, int L) {
  for (int o = 1; o < L; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// Eight bytes at any address.
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// Sum over the TR threads of a row (fixed order).
template <int TR>
__device__ inline float row_sum(float a, float (*red)[2]) {
  float none = 0.f;
  row_sums<TR>(a, none, red);
  return a;
}

// y, or with Q its 8 bits, and s and rstd where they are wanted.  S: the residual's
// type, T's where there is none.
template <typename T, typename S, int TR, int C, bool Q>
__global__ __launch_bounds__(TR < 256 ? 256 : TR) void rms_fwd_rows_kernel(
    const T* __restrict__ X, long ldx, const S* __restrict__ R, long ldr, const void* __restrict__ w, int param_f32,
    long N, int D, float eps, T* __restrict__ Y, S* __restrict__ sum_out, float* __restrict__ rstd_out, RmsQuant o) {
  typedef RowRegs<T, TR, C> Row;
  constexpr int kRows = TR < 256 ? 256 / TR : 1, E = Row::E;
  __shared__ float red[TR / 64][2];
  __shared__ uint32_t redmax[TR / 64];
  const int t = threadIdx.x % TR;
  const float inv = 1.f / (float)D;
  Row wr;
  wr.load_params(w, param_f32, D, t, 1.f);
  for (long n = (long)blockIdx.x * kRows + threadIdx.x / TR; n < N; n += (long)gridDim.x * kRows) {
    float v[C][E];
    load_chunks<T, T, TR, C>(v, X + n * ldx, D, t);
    if (R) {
      float r[C][E];
      load_chunks<T, S, TR, C>(r, R + n * ldr, D, t);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < E; ++i) v[c][i] = elem_to_f32(f32_to_elem<S>(v[c][i] + r[c][i]));
      store_chunks<T, S, TR, C>(v, sum_out + n * D, D, t);
    }
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; ++i) q = __builtin_fmaf(v[c][i], v[c][i], q);
    const float rstd = 1.f / sqrtf(row_sum<TR>(q, red) * inv + eps);
    if (rstd_out && t == 0) rstd_out[n] = rstd;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; ++i) v[c][i] = v[c][i] * rstd * wr.v[c][i];
    if constexpr (!Q) {
      store_chunks<T, T, TR, C>(v, Y + n * D, D, t);
    } else {
      uint32_t mx[C], all = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        mx[c] = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) mx[c] = max(mx[c], magnitude(v[c][i]));
        all = max(all, mx[c]);
      }
      if (o.group) {
#pragma unroll
        for (int c = 0; c < C; ++c) mx[c] = lanes_max(mx[c], o.group / E);
      } else {
        all = lanes_max(all, 64);
        if constexpr (TR > 64) {
          if ((threadIdx.x & 63) == 0) redmax[threadIdx.x >> 6] = all;
          __syncthreads();
#pragma unroll
          for (int k = 0; k < TR / 64; ++k) all = max(all, redmax[k]);
        }
        if (t == 0) o.scales[n] = quant_scale(o, all);
      }
      uint8_t* const row = o.q + n * D;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int at = Row::first(c, t);
        const float scale = quant_scale(o, o.group ? mx[c] : all);
        const Quotient by(scale);
        if (o.starts(at) && at < D) o.scales[o.place(n, at)] = scale;
        uint32_t b[E / 4];
#pragma unroll
        for (int i = 0; i < E; i += 4) b[i / 4] = quant4(o, by, &v[c][i]);
        if (at + E <= D) {
          if constexpr (E == 8)
            *reinterpret_cast<u32x2_any*>(row + at) = u32x2_any{b[0], b[1]};
          else
            *reinterpret_cast<u32_any*>(row + at) = b[0];
        } else if (at < D) {
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (at + i < D) row[at + i] = (uint8_t)(b[i / 4] >> (i % 4 * 8));
        }
      }
    }
  }
}

// The gradient of s and the workgroup's sums of dw over its rows at
// dw[blockIdx.x * D].  dS: null where there is none; dR: null where dx is the
// residual's gradient too.
template <typename T, typename S, int TR, int C>
__global__ __launch_bounds__(TR < 256 ? 256 : TR) void rms_bwd_rows_kernel(
    const T* __restrict__ dY, const S* __restrict__ dS, const S* __restrict__ sum, long lds, const void* __restrict__ w,
    int param_f32, const float* __restrict__ rstd, long N, int D, T* __restrict__ dX, S* __restrict__ dR,
    float* __restrict__ dw) {
  typedef RowRegs<T, TR, C> Row;
  constexpr int kRows = TR < 256 ? 256 / TR : 1, E = Row::E;
  __shared__ float red[TR / 64][2];
  const int t = threadIdx.x % TR;
  const float inv = 1.f / (float)D;
  Row wr;
  wr.load_params(w, param_f32, D, t, 1.f);
  float sw[C][E] = {};
  const long step = (long)gridDim.x * kRows;
  long n = (long)blockIdx.x * kRows + threadIdx.x / TR;
  RawChunks<T, S, TR, C> raw_x;
  RawChunks<T, T, TR, C> raw_g;
  float next_r = 0.f;
  auto issue = [&](long m) {
    raw_x.issue(sum + m * lds, D, t);
    raw_g.issue(dY + m * D, D, t);
    next_r = rstd[m];
  };
  constexpr bool kAhead = TR < 1024;  // as in layer_norm_bwd_rows_kernel
  if (kAhead && n < N) issue(n);
  for (; n < N; n += step) {
    if (!kAhead) issue(n);
    float x[C][E], g[C][E];
    raw_x.take(x, sum + n * lds, D, t);
    raw_g.take(g, dY + n * D, D, t);
    const float r = next_r;
    RawChunks<T, S, TR, C> raw_s;
    if (dS) raw_s.issue(dS + n * D, D, t);
    if (kAhead && n + step < N) issue(n + step);  // the next row, while this one is worked on
    float san = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[c][i] *= r;
        sw[c][i] = __builtin_fmaf(g[c][i], x[c][i], sw[c][i]);
        g[c][i] *= wr.v[c][i];
        san = __builtin_fmaf(g[c][i], x[c][i], san);
      }
    if (!dX && !dR) continue;
    san = row_sum<TR>(san, red) * inv;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < E; ++i) x[c][i] = r * __builtin_fmaf(-x[c][i], san, g[c][i]);
    if (dS) {
      raw_s.take(g, dS + n * D, D, t);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < E; ++i) x[c][i] += g[c][i];
    }
    if (dX) store_chunks<T, T, TR, C>(x, dX + n * D, D, t);
    if (dR) store_chunks<T, S, TR, C>(x, dR + n * D, D, t);
  }
  if (!dw) return;
  // the rows' sums within the workgroup, one after the other
  if constexpr (kRows > 1) {
    __shared__ float sums[TR * C * E];
    for (int k = 0; k < kRows; ++k) {
      if (threadIdx.x / TR == k) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const int at = (c * E + i) * TR + t;
            sums[at] = sw[c][i] = k ? sums[at] + sw[c][i] : sw[c][i];
          }
      }
      __syncthreads();
    }
    if (threadIdx.x / TR != kRows - 1) return;
  }
  dw += (long)blockIdx.x * D;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const int at = Row::first(c, t) + i;
      if (at + 4 <= D) {
        *reinterpret_cast<loose_f32x4*>(dw + at) = f32x4{sw[c][i], sw[c][i + 1], sw[c][i + 2], sw[c][i + 3]};
        continue;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + k < D) dw[at + k] = sw[c][i + k];
    }
}

// A parameter's element, fp32 or of type T (null: 1).
template <typename T>
__device__ inline float param_at(const void* w, int f32, int c) {
  return !w ? 1.f : f32 ? static_cast<const float*>(w)[c] : elem_to_f32(static_cast<const T*>(w)[c]);
}

// Longer rows, one workgroup per row: s and its sum of squares, then (Q: the scales,
// with the row's largest magnitude, then) the output.  Element by element, each pass adding
// x and r again: 2048 x 20000 bf16 with a bf16 residual 132 us (2.5 TB/s of what has to
// move), in 8 bits 170 us with group scales and 238 with a row's; backward 187 us and 242
// with dw.  Rows of 16384, in registers: 54, 53, 54; 49 and 61.
template <typename T, typename S, bool Q>
__global__ __launch_bounds__(256) void rms_fwd_kernel(const T* __restrict__ X, long ldx, const S* __restrict__ R, long ldr,
                                                      const void* __restrict__ w, int param_f32, int D, float eps,
                                                      T* __restrict__ Y, S* __restrict__ sum_out,
                                                      float* __restrict__ rstd_out, RmsQuant o) {
  __shared__ float red[4];
  __shared__ uint32_t redmax[4];
  const long n = blockIdx.x;
  const int tid = threadIdx.x;
  const T* const x = X + n * ldx;
  auto at = [&](int c) {
    const float v = elem_to_f32(x[c]);
    return R ? elem_to_f32(f32_to_elem<S>(v + elem_to_f32(R[n * ldr + c]))) : v;
  };
  float q = 0.f;
  for (int c = tid; c < D; c += 256) {
    const float v = at(c);
    if (R) sum_out[n * D + c] = f32_to_elem<S>(v);
    q = __builtin_fmaf(v, v, q);
  }
  const float rstd = 1.f / sqrtf(block_sum(q, red) / (float)D + eps);
  if (rstd_out && tid == 0) rstd_out[n] = rstd;
  auto y = [&](int c) { return at(c) * rstd * param_at<T>(w, param_f32, c); };
  if constexpr (!Q) {
    for (int c = tid; c < D; c += 256) Y[n * D + c] = f32_to_elem<T>(y(c));
  } else {
    uint32_t all = 0;
    if (!o.group) {
      for (int c = tid; c < D; c += 256) all = max(all, magnitude(y(c)));
      all = lanes_max(all, 64);
      if ((tid & 63) == 0) redmax[tid >> 6] = all;
      __syncthreads();
      all = max(max(redmax[0], redmax[1]), max(redmax[2], redmax[3]));
      if (tid == 0) o.scales[n] = quant_scale(o, all);
    }
    // eight columns a thread, so that a group is at most half a wave's
    for (int c0 = 0; c0 < D; c0 += 2048) {
      const int c = c0 + tid * 8;
      float v[8];
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = c + i < D ? y(c + i) : 0.f;
        mx = max(mx, magnitude(v[i]));
      }
      if (o.group) mx = lanes_max(mx, o.group / 8);
      const float scale = quant_scale(o, o.group ? mx : all);
      const Quotient by(scale);
      if (o.starts(c) && c < D) o.scales[o.place(n, c)] = scale;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const uint32_t b = quant4(o, by, &v[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + i + k < D) o.q[n * D + c + i + k] = (uint8_t)(b >> (k * 8));
      }
    }
  }
}

template <typename T, typename S>
__global__ __launch_bounds__(256) void rms_dx_kernel(const T* __restrict__ dY, const S* __restrict__ dS,
                                                     const S* __restrict__ sum, long lds, const void* __restrict__ w,
                                                     int param_f32, const float* __restrict__ rstd, int D,
                                                     T* __restrict__ dX, S* __restrict__ dR) {
  __shared__ float red[4];
  const long n = blockIdx.x;
  const S* const x = sum + n * lds;
  const T* const dy = dY + n * D;
  const float r = rstd[n];
  float san = 0.f;
  for (int c = threadIdx.x; c < D; c += 256)
    san += elem_to_f32(dy[c]) * param_at<T>(w, param_f32, c) * (elem_to_f32(x[c]) * r);
  san = block_sum(san, red) / (float)D;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float a = elem_to_f32(dy[c]) * param_at<T>(w, param_f32, c);
    float v = r * (a - elem_to_f32(x[c]) * r * san);
    if (dS) v += elem_to_f32(dS[n * D + c]);
    if (dX) dX[n * D + c] = f32_to_elem<T>(v);
    if (dR) dR[n * D + c] = f32_to_elem<S>(v);
  }
}

// dw over the rows [part * rows, (part + 1) * rows), part = blockIdx.y, one column per
// thread.
template <typename T, typename S>
__global__ __launch_bounds__(256) void rms_parts_kernel(const T* __restrict__ dY, const S* __restrict__ sum, long lds,
                                                        const float* __restrict__ rstd, long N, int D, long rows,
                                                        float* __restrict__ dw) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  const long n0 = blockIdx.y * rows, n1 = min(n0 + rows, N);
  float sw = 0.f;
  for (long n = n0; n < n1; ++n) sw += elem_to_f32(dY[n * D + c]) * (elem_to_f32(sum[n * lds + c]) * rstd[n]);
  dw[(long)blockIdx.y * D + c] = sw;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// Calls f(T(), S()) for the types of the input and of the residual.
template <typename F>
int rms_types(int dtype, int rdtype, F&& f) {
  if (dtype == CCE_DTYPE_BF16) return rdtype == dtype ? f((uint16_t)0, (uint16_t)0) : f((uint16_t)0, 0.f);
  if (dtype == CCE_DTYPE_F16) return rdtype == dtype ? f((_Float16)0, (_Float16)0) : f((_Float16)0, 0.f);
  return f(0.f, 0.f);
}

int check_rms(int64_t N, int64_t D, int dtype, int64_t ldx, int rdtype, int64_t ldr, int wdtype, float eps) {
  const int rc = check_norm(N, D, dtype, ldx, wdtype);
  if (rc) return rc;
  if (rdtype != dtype && rdtype != CCE_DTYPE_F32)
    return fail(CCE_ERR_INVALID_ARG, "the residual's dtype must be the input's or CCE_DTYPE_F32, got %d", rdtype);
  if (N > 1 && ldr < D)
    return fail(CCE_ERR_INVALID_ARG, "the residual's row stride %ld is smaller than D = %ld", (long)ldr, (long)D);
  if (!(eps >= 0.f && eps < INFINITY)) return fail(CCE_ERR_INVALID_ARG, "eps must be finite and at least 0");
  return CCE_OK;
}

// The backward's shapes are layer norm's, but for rows of a workgroup that would hold
// 32 elements a thread (16-bit types past 4096): with the next row's loads beside they
// take 250 registers, and the barriers of a row find one other workgroup on the CU.
// 1024 threads of 16 elements, 4096 x 8192 bf16: 70 -> 63 us.  Waves of 32 elements
// stay (16384 x 2048 63 us, by 256 threads of 16 70), and 256 threads of 16 (8192 x
// 4096 fp32 92 us, by 1024 98).
template <int E, int kMost, typename F>
bool rms_bwd_shape(long D, F&& f) {
  if (E == 8 && D > 256 * 2 * E && D <= 1024 * 2 * E) {
    f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
    return true;
  }
  return norm_shape<E, kMost>(D, f);
}

// Parts of dw, one per workgroup of the backward.
long rms_parts(int dtype, long N, long D) {
  int threads = 256;
  auto shape = [&](auto tr, auto) { threads = decltype(tr)::value; };
  if (dtype == CCE_DTYPE_F32)
    rms_bwd_shape<4, kNormRegD>(D, shape);
  else
    rms_bwd_shape<8, kNormRegD>(D, shape);
  return norm_parts(N, D, threads);
}
size_t rms_bytes(int dtype, long N, long D, bool need_dw) {
  return need_dw ? align_up((size_t)(rms_parts(dtype, N, D) * D) * sizeof(float), 256) : 0;
}

template <bool Q>
int rms_forward(const void* x, int dtype, int64_t ldx, const void* residual, int rdtype, int64_t ldr, const void* weight,
                int wdtype, int64_t N, int64_t D, float eps, void* y, void* sum, float* rstd, const RmsQuant& o,
                hipStream_t st) {
  return rms_types(dtype, rdtype, [&](auto t, auto s) {
    typedef decltype(t) T;
    typedef decltype(s) S;
    const int f32 = wdtype == CCE_DTYPE_F32;
    const bool in_registers = norm_shape<16 / sizeof(T), kNormRegD>(D, [&](auto tr, auto c) {
      constexpr int TR = decltype(tr)::value, kRows = TR < 256 ? 256 / TR : 1;
      const unsigned grid = (unsigned)std::min<long>(ceil_div(N, kRows), kNormGroups);
      hipLaunchKernelGGL((rms_fwd_rows_kernel<T, S, TR, decltype(c)::value, Q>), dim3(grid), dim3(std::max(TR, 256)), 0,
                         st, static_cast<const T*>(x), (long)ldx, static_cast<const S*>(residual), (long)ldr, weight, f32,
                         (long)N, (int)D, eps, static_cast<T*>(y), static_cast<S*>(sum), rstd, o);
    });
    if (!in_registers)
      hipLaunchKernelGGL((rms_fwd_kernel<T, S, Q>), dim3((unsigned)N), dim3(256), 0, st, static_cast<const T*>(x),
                         (long)ldx, static_cast<const S*>(residual), (long)ldr, weight, f32, (int)D, eps,
                         static_cast<T*>(y), static_cast<S*>(sum), rstd, o);
    HIP_TRY(hipGetLastError());
    return CCE_OK;
  });
}

int rms_backward(const void* dy, const void* ds, const void* sum, int dtype, int rdtype, int64_t lds, const void* weight,
                 int wdtype, const float* rstd, int64_t N, int64_t D, void* dx, void* dr, void* dw, float* parts_dw,
                 hipStream_t st) {
  return rms_types(dtype, rdtype, [&](auto t, auto s) {
    typedef decltype(t) T;
    typedef decltype(s) S;
    if (!dx && !dr && !dw) return CCE_OK;
    const int f32 = wdtype == CCE_DTYPE_F32;
    const long parts = rms_parts(dtype, N, D);
    const bool in_registers = rms_bwd_shape<16 / sizeof(T), kNormRegD>(D, [&](auto tr, auto c) {
      constexpr int TR = decltype(tr)::value;
      hipLaunchKernelGGL((rms_bwd_rows_kernel<T, S, TR, decltype(c)::value>), dim3((unsigned)parts),
                         dim3(std::max(TR, 256)), 0, st, static_cast<const T*>(dy), static_cast<const S*>(ds),
                         static_cast<const S*>(sum), (long)lds, weight, f32, rstd, (long)N, (int)D, static_cast<T*>(dx),
                         static_cast<S*>(dr), dw ? parts_dw : nullptr);
    });
    HIP_TRY(hipGetLastError());
    if (!in_registers && (dx || dr) && N > 0) {
      hipLaunchKernelGGL((rms_dx_kernel<T, S>), dim3((unsigned)N), dim3(256), 0, st, static_cast<const T*>(dy),
                         static_cast<const S*>(ds), static_cast<const S*>(sum), (long)lds, weight, f32, rstd, (int)D,
                         static_cast<T*>(dx), static_cast<S*>(dr));
      HIP_TRY(hipGetLastError());
    }
    if (!dw) return CCE_OK;
    if (!in_registers) {
      hipLaunchKernelGGL((rms_parts_kernel<T, S>), dim3((unsigned)ceil_div(D, 256), (unsigned)parts), dim3(256), 0, st,
                         static_cast<const T*>(dy), static_cast<const S*>(sum), (long)lds, rstd, (long)N, (int)D,
                         ceil_div(N, parts), parts_dw);
      HIP_TRY(hipGetLastError());
    }
    return norm_types(dtype, wdtype, [&](auto, auto w) {
      typedef decltype(w) W;
      hipLaunchKernelGGL(layer_norm_join_kernel<W>, dim3((unsigned)ceil_div(D, 16), 1), dim3(256), 0, st, parts_dw,
                         nullptr, (int)parts, (int)D, static_cast<W*>(dw), nullptr);
      HIP_TRY(hipGetLastError());
      return CCE_OK;
    });
  });
}
