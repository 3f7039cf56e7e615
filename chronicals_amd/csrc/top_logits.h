// The k largest logits of each row, largest first, and their columns; among
// equal values the lower column first.  A NaN counts as larger than any number
// (as torch orders it), and -0 equals +0.  What is chosen is copied bit by bit.

constexpr int kTopMax = CCE_MAX_TEACHER_ENTRIES;  // entries per row

// A 32-bit key that orders as the values do.
__device__ inline uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 becomes +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The bits of a type's keys that tell values apart: bf16 has 16 (the others of a
// negative value's key are ones, and cleared).
template <typename T>
constexpr int kKeyBits = std::is_same<T, uint16_t>::value ? 16 : 32;
template <typename T>
__device__ inline uint32_t key_of(T x) {
  return order_key(elem_to_f32(x)) & (~0u << (32 - kKeyBits<T>));
}

// The k-th largest of m keys (1 <= k <= m) by a workgroup of 256: eight bits at
// a time from the top, the count of each value among the keys that agree so far.
// Returns how many keys equal to `tau` belong to the k largest.
template <int BITS, typename F>
__device__ int kth_key(F&& key, int m, int k, uint32_t* hist, uint32_t& tau) {
  __shared__ int found[2];
  const int tid = threadIdx.x;
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 32 - BITS; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < m; i += 256) {
      const uint32_t v = key(i);
      if ((v & mask) == prefix) atomicAdd(&hist[v >> shift & 255], 1u);
    }
    __syncthreads();
    // keys whose digit is tid or more
    int above = (int)hist[tid];
    for (int o = 1; o < 256; o <<= 1) {
      const int more = tid + o < 256 ? (int)hist[tid + o] : 0;
      __syncthreads();
      above += more;
      hist[tid] = (uint32_t)above;
      __syncthreads();
    }
    const int next = tid < 255 ? (int)hist[tid + 1] : 0;
    if (above >= k && next < k) {
      found[0] = tid;
      found[1] = next;
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    mask |= 255u << shift;
    k -= found[1];
    __syncthreads();
  }
  tau = prefix;
  return k;
}

// A candidate: its key above the complement of its column, so that a larger one
// comes first and among equal keys the lower column.  All are different.
__device__ inline uint64_t candidate(uint32_t key, int at) { return (uint64_t)key << 32 | (uint32_t)~at; }
__device__ inline int column(uint64_t c) { return (int)~(uint32_t)c; }

// Candidates in LDS.
struct TopList {
  uint64_t* c;
  int* count;
};

// The first `need` of the m keys that equal tau, by position, into list.c[at..]
// (at least so many are there).  Eight neighbouring keys per thread at a time.
template <typename F>
__device__ void take_equal(F&& key, int m, uint32_t tau, int need, int at, const TopList& list) {
  __shared__ int wave_count[4];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  int done = 0;
  for (int i0 = 0; i0 < m && done < need; i0 += 256 * 8) {
    unsigned eq = 0;
    for (int e = 0; e < 8; ++e) {
      const int i = i0 + tid * 8 + e;
      if (i < m && key(i) == tau) eq |= 1u << e;
    }
    int upto = __popc(eq);  // an inclusive scan over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      if (l >= o) upto += v;
    }
    __syncthreads();
    if (l == 63) wave_count[w] = upto;
    __syncthreads();
    int p = done + upto - __popc(eq);
    for (int v = 0; v < 4; ++v) {
      if (v < w) p += wave_count[v];
      done += wave_count[v];
    }
    for (int e = 0; e < 8; ++e)
      if (eq >> e & 1) {
        if (p < need) list.c[at + p] = candidate(tau, i0 + tid * 8 + e);
        ++p;
      }
  }
  __syncthreads();
}

// The k largest of m keys into `list`, in no order.
template <int BITS, typename F>
__device__ void top_exact(F&& key, int m, int k, uint32_t* hist, const TopList& list) {
  const int tid = threadIdx.x;
  uint32_t tau;
  const int equal = kth_key<BITS>(key, m, k, hist, tau);
  if (tid == 0) *list.count = 0;
  __syncthreads();
  for (int i = tid; i < m; i += 256) {
    const uint32_t v = key(i);
    if (v > tau) list.c[atomicAdd(list.count, 1)] = candidate(v, i);
  }
  take_equal(key, m, tau, equal, k - equal, list);
  if (tid == 0) *list.count = k;
  __syncthreads();
}

// Calls f(rank, candidate) for the candidates of rank below k, one thread each.
template <typename F>
__device__ void top_ranked(const TopList& list, int k, F&& f) {
  const int m = *list.count;
  for (int i = threadIdx.x; i < m; i += 256) {
    const uint64_t v = list.c[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < m; ++j) rank += list.c[j] > v;
    if (rank < k) f(rank, v);
  }
}

// The largest of some elements, as unsigned integers that order as the values do:
// 0 for -inf, past +inf's the NaN of either sign, -0 one below +0.  From the bits
// b: b ^ 0x7f.. for negative ones, less -inf's.  The 16-bit types keep two, of the
// even and the odd elements (packed operations).
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short w16x2 __attribute__((ext_vector_type(2)));
template <typename T>
struct GroupMax {
  static constexpr int kParts = 2, kBits = 16;
  static constexpr uint32_t kInf = std::is_same<T, uint16_t>::value ? 0x7f80 : 0x7c00;  // +inf's bits
  static constexpr uint32_t kZero = kInf + 1;                                          // +0
  w16x2 v = {0, 0};
  __device__ inline void add(const u32x4& raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = raw[i];  // a bit_cast of the vector's element itself takes element 0
      const s16x2 b = __builtin_bit_cast(s16x2, r);
      const w16x2 p = __builtin_bit_cast(w16x2, (s16x2)(b ^ (s16x2)((b >> 15) & (short)0x7fff))) + (unsigned short)kZero;
      v = __builtin_elementwise_max(v, p);
    }
  }
  __device__ inline void merge(const GroupMax& o) { v = __builtin_elementwise_max(v, o.v); }
  __device__ inline uint32_t part(int i) const { return v[i]; }
  static __device__ inline T value(uint32_t p) {
    const short b = (short)(p - kZero);
    return __builtin_bit_cast(T, (short)(b ^ ((b >> 15) & 0x7fff)));
  }
};
template <>
struct GroupMax<float> {
  static constexpr int kParts = 1, kBits = 32;
  static constexpr uint32_t kInf = 0x7f800000u, kZero = kInf + 1;
  uint32_t v = 0;
  __device__ inline void add(const u32x4& raw) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v = max(v, (raw[i] ^ (uint32_t)((int)raw[i] >> 31) >> 1) + kZero);
  }
  __device__ inline void merge(const GroupMax& o) { v = max(v, o.v); }
  __device__ inline uint32_t part(int) const { return v; }
  static __device__ inline float value(uint32_t p) {
    const uint32_t b = p - kZero;
    return __uint_as_float(b ^ (uint32_t)((int)b >> 31) >> 1);
  }
};

constexpr int kTopCandidates = 2048, kTopGroups = 1024;

// The k largest of row[0, V) into `list` (at least those k, at most
// kTopCandidates), by one pass over HBM and a second look at a few of its lines.
//
// Pass 1 keeps the largest of groups of chunks: a thread's chunks at each place of
// its four loads in flight, by their round modulo four.  Four such groups together
// (1024 or, of the 16-bit types, 2048 fours) have a largest element each, so at
// least k elements reach the k-th largest of these, tau.  Pass 2 reads the groups
// that reach tau again and collects their elements from it on: for values in no
// particular order about k groups and k elements, 66 to 300 for k = 64 to 256.
// A chunk of 16 bytes brings a whole line: with the four groups as one, 42% of the
// row was read again (now 12%), and 128 us taken for 107.
//
// With more than kTopCandidates there (a mask's value fills the row up to k), the
// elements above tau are collected alone and the first ones that equal it added.
// What overflows then too, or has fewer chunks than k, goes by top_exact, whose
// passes over the row are three to five.
//
// Bound by HBM: k = 64 of 2048 x 151936 bf16 takes 107 us, 5.8 TB/s of the rows (a
// large copy reaches 4.9, half of it reads); by top_exact alone it took 1550 us.
// 144 -> 136 us came from non-temporal loads in pass 1 and 136 -> 128 from eight
// workgroups per CU instead of seven.  With all but 20 columns of a row at a mask's
// value 390 us, and by top_exact after the overflow 2510.
template <typename T>
__device__ void top_of_row(const T* row, int V, int k, uint32_t* hist, uint16_t* groups, const TopList& list) {
  constexpr int U = 4, NP = GroupMax<T>::kParts;
  __shared__ int counts[2][4], ngroups;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const RowSplit<T> sp(row, V);
  if (sp.chunks >= k) {
    const u32x4* const body = reinterpret_cast<const u32x4*>(row + sp.head);
    constexpr int R = 4;
    GroupMax<T> part[R][U], g[U];
    for (int c0 = tid; c0 < sp.chunks; c0 += R * U * 256) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int c = c0 + r * U * 256;
        if (c + (U - 1) * 256 < sp.chunks) {
          u32x4 raw[U];
#pragma unroll
          for (int u = 0; u < U; ++u) raw[u] = __builtin_nontemporal_load(body + c + u * 256);
#pragma unroll
          for (int u = 0; u < U; ++u) part[r][u].add(raw[u]);
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c + u * 256 < sp.chunks) part[r][u].add(body[c + u * 256]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      g[u] = part[0][u];
#pragma unroll
      for (int r = 1; r < R; ++r) g[u].merge(part[r][u]);
    }
    // tau: the largest integer that k groups reach, bit by bit from the top
    uint32_t tau = 0;
    auto search = [&](int high, int low) {
      for (int bit = high; bit >= low; --bit) {
        const uint32_t next = tau | 1u << bit;
        int n = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < NP; ++i) n += __popcll(__ballot(g[u].part(i) >= next));
        int* const at = counts[bit & 1];
        if (l == 0) at[w] = n;
        __syncthreads();
        if (at[0] + at[1] + at[2] + at[3] >= k) tau = next;
      }
      __syncthreads();
    };
    const int rounds = (sp.chunks + R * U * 256 - 1) / (R * U * 256);  // of a group
    // The elements of keys from `from` on (above it: with `above`) into the list, as
    // far as they fit; returns how many there are.
    auto collect = [&](uint32_t from, bool above) {
      // the lowest integer of the same key: NaN are equal, and so are zeros
      constexpr uint32_t kInf = GroupMax<T>::kInf + GroupMax<T>::kZero;
      const uint32_t reach = tau > kInf ? kInf + 1 : tau == GroupMax<T>::kZero ? tau - 1 : tau;
      if (tid == 0) *list.count = ngroups = 0;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          bool some = false;
#pragma unroll
          for (int i = 0; i < NP; ++i) some = some || part[r][u].part(i) >= reach;
          if (!some) continue;
          const int p = atomicAdd(&ngroups, 1);
          if (p < kTopGroups) groups[p] = (uint16_t)((r * U + u) * 256 + tid);
        }
      __syncthreads();
      auto take = [&](T x, int at) {
        const uint32_t key = key_of(x);
        if (key < from || (above && key == from)) return;
        const int p = atomicAdd(list.count, 1);
        if (p < kTopCandidates) list.c[p] = candidate(key, at);
      };
      // with more groups than the list holds: every chunk
      const bool listed = ngroups <= kTopGroups;
      const int items = listed ? ngroups * rounds : sp.chunks;
      for (int i0 = 0; i0 < items; i0 += U * 256) {
        u32x4 raw[U];
        int at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * 256 + tid;
          at[u] = -1;
          if (i < items) {
            // neighbouring threads take neighbouring groups of one round
            const int chunk = listed ? (i / ngroups) * (R * U * 256) + groups[i % ngroups] : i;
            if (chunk < sp.chunks) {
              at[u] = sp.head + chunk * RowSplit<T>::E;
              raw[u] = body[chunk];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (at[u] < 0) continue;
          const T* v = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
          for (int e = 0; e < RowSplit<T>::E; ++e) take(v[e], at[u] + e);
        }
      }
      if (tid < sp.head) take(row[tid], tid);
      if (tid < V - sp.tail_start) take(row[sp.tail_start + tid], sp.tail_start + tid);
      __syncthreads();
      const int n = *list.count;
      __syncthreads();
      return n;
    };
    // Of fp32's bits the lowest 12 stay 0 at first: what lies in between is hardly
    // ever a candidate more, and each bit costs a barrier
    constexpr int kBits = GroupMax<T>::kBits, kFirst = kBits == 32 ? 12 : 0;
    search(kBits - 1, kFirst);
    if (collect(key_of(GroupMax<T>::value(tau)), false) <= kTopCandidates) return;
    search(kFirst - 1, 0);
    const uint32_t from = key_of(GroupMax<T>::value(tau));
    const int above = collect(from, true);
    if (above <= kTopCandidates) {
      if (above >= k) return;
      take_equal([&](int i) { return key_of(row[i]); }, V, from, k - above, above, list);
      if (tid == 0) *list.count = k;
      __syncthreads();
      return;
    }
  }
  top_exact<kKeyBits<T>>([&](int i) { return key_of(row[i]); }, V, k, hist, list);
}

// Columns of split s of S of a row of V: whole multiples of 64, so that every
// split starts on the row's alignment.
__device__ inline void split_span(int V, int S, int s, int& c0, int& c1) {
  const int per = ((V + S - 1) / S + 63) / 64 * 64;
  c0 = min((int)min((long)s * per, (long)V), V);
  c1 = (int)min((long)c0 + per, (long)V);
}

// One workgroup per row and split of S.  One split: the row's answer.  More: the
// split's k largest, in order, at part[(n * S + s) * k], or all of it where it has
// no more than k columns, and zeros (less than any candidate) behind.
template <typename T>
__global__ __launch_bounds__(256) void top_logits_kernel(const T* __restrict__ X, long ld, int V, int S, int k,
                                                         T* __restrict__ values, int64_t* __restrict__ indices,
                                                         uint64_t* __restrict__ part) {
  __shared__ uint32_t hist[256];
  __shared__ uint64_t cands[kTopCandidates];
  __shared__ uint16_t groups[kTopGroups];  // 16 bits: eight workgroups per CU fit with 20 KB each
  __shared__ int count;
  const TopList list = {cands, &count};
  const long n = blockIdx.x / S;
  int c0, c1;
  split_span(V, S, blockIdx.x % S, c0, c1);
  const T* const row = X + n * ld + c0;
  const int m = min(k, c1 - c0);
  if (m > 0) top_of_row(row, c1 - c0, m, hist, groups, list);
  if (S == 1) {
    top_ranked(list, k, [&](int rank, uint64_t c) {
      values[n * k + rank] = row[column(c)];
      indices[n * k + rank] = column(c);
    });
    return;
  }
  uint64_t* const out = part + (long)blockIdx.x * k;
  if (m > 0) top_ranked(list, m, [&](int rank, uint64_t c) { out[rank] = candidate(c >> 32, c0 + column(c)); });
  for (int i = m + threadIdx.x; i < k; i += 256) out[i] = 0;
}

// The k largest of a row from those of its S splits.  S * ceil(k / S) candidates
// reach the smallest of the splits' ceil(k / S)-th ones, so no other counts.
template <typename T>
__global__ __launch_bounds__(256) void top_join_kernel(const T* __restrict__ X, long ld, int S, int k,
                                                       const uint64_t* __restrict__ part, T* __restrict__ values,
                                                       int64_t* __restrict__ indices) {
  constexpr int kE = kTopCandidates / 256;
  __shared__ uint64_t cands[kTopCandidates], low[4];
  __shared__ int count;
  const TopList list = {cands, &count};
  const long n = blockIdx.x;
  const int tid = threadIdx.x;
  const uint64_t* const p = part + n * S * k;
  uint64_t c[kE], tau = ~0ull;
  for (int s = tid; s < S; s += 256) tau = min(tau, p[s * k + (k + S - 1) / S - 1]);
#pragma unroll
  for (int e = 0; e < kE; ++e) c[e] = e * 256 + tid < S * k ? p[e * 256 + tid] : 0;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) tau = min(tau, (uint64_t)__shfl_xor((unsigned long long)tau, o));
  if ((tid & 63) == 0) low[tid >> 6] = tau;
  if (tid == 0) count = 0;
  __syncthreads();
  tau = min(min(low[0], low[1]), min(low[2], low[3]));
#pragma unroll
  for (int e = 0; e < kE; ++e)
    if (c[e] >= tau && c[e] != 0) cands[atomicAdd(&count, 1)] = c[e];
  __syncthreads();
  top_ranked(list, k, [&](int rank, uint64_t v) {
    values[n * k + rank] = X[n * ld + column(v)];
    indices[n * k + rank] = column(v);
  });
}

// Workgroups per row: about four per CU where there are few rows, with at least
// 2048 columns each, and no more candidates than one workgroup can join.  k = 128
// of 16 x 128256 fp32: one workgroup per row by top_exact 528 us, 16 of them and
// their join 22 us (11 each, most of it latencies).
int top_splits(long N, long V, long k) {
  const long s = std::min({ceil_div(1024, std::max<long>(N, 1)), V / 2048, kTopCandidates / std::max<long>(k, 1)});
  return (int)std::max<long>(s, 1);
}

size_t top_bytes(long N, long V, long k) {
  const int S = top_splits(N, V, k);
  return S > 1 ? (size_t)N * S * k * sizeof(uint64_t) : 0;
}

template <typename T>
int top_run(const T* X, long ld, long N, long V, long k, T* values, int64_t* indices, uint64_t* part, hipStream_t st) {
  const int S = top_splits(N, V, k);
  hipLaunchKernelGGL(top_logits_kernel<T>, dim3((unsigned)(N * S)), dim3(256), 0, st, X, ld, (int)V, S, (int)k, values,
                     indices, part);
  HIP_TRY(hipGetLastError());
  if (S > 1) {
    hipLaunchKernelGGL(top_join_kernel<T>, dim3((unsigned)N), dim3(256), 0, st, X, ld, S, (int)k, part, values, indices);
    HIP_TRY(hipGetLastError());
  }
  return CCE_OK;
}

int check_top(int64_t N, int64_t V, int64_t k, int dtype, int64_t ld) {
  const int rc = check_logits_args(N, V, dtype, ld, CCE_REDUCTION_NONE, 0.f, CCE_SMOOTH_LOGV);
  if (rc) return rc;
  if (k < 1 || k > kTopMax || k > V)
    return fail(CCE_ERR_INVALID_ARG, "k must be in [1, min(%d, V = %ld)] (got %ld)", kTopMax, (long)V, (long)k);
  return CCE_OK;
}
