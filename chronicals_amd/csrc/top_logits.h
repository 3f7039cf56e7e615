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

// Candidates in LDS, as (key, position) pairs that are all different.
struct TopList {
  uint32_t* key;
  int* at;
  int* count;
};

// The k largest of m keys into `list`, in no order; equal keys by the lower
// position first.
template <int BITS, typename F>
__device__ void top_exact(F&& key, int m, int k, uint32_t* hist, const TopList& list) {
  __shared__ int wave_count[4];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  uint32_t tau;
  const int equal = kth_key<BITS>(key, m, k, hist, tau);
  if (tid == 0) *list.count = 0;
  __syncthreads();
  for (int i = tid; i < m; i += 256) {
    const uint32_t v = key(i);
    if (v > tau) {
      const int p = atomicAdd(list.count, 1);
      list.key[p] = v;
      list.at[p] = i;
    }
  }
  // those equal to tau in order of their positions, 256 at a time
  int done = 0;
  for (int i0 = 0; i0 < m && done < equal; i0 += 256) {
    const int i = i0 + tid;
    const bool eq = i < m && key(i) == tau;
    const uint64_t mine = __ballot(eq);
    __syncthreads();
    if (l == 0) wave_count[w] = __popcll(mine);
    __syncthreads();
    int p = done + __popcll(mine & ((1ull << l) - 1));
    for (int v = 0; v < 4; ++v) {
      if (v < w) p += wave_count[v];
      done += wave_count[v];
    }
    if (eq && p < equal) {
      list.key[k - equal + p] = tau;
      list.at[k - equal + p] = i;
    }
  }
  __syncthreads();
  if (tid == 0) *list.count = k;
  __syncthreads();
}

// Calls f(rank, position) for the candidates of rank below k, one thread each.
template <typename F>
__device__ void top_ranked(const TopList& list, int k, F&& f) {
  const int m = *list.count;
  for (int i = threadIdx.x; i < m; i += 256) {
    const uint32_t v = list.key[i];
    const int at = list.at[i];
    int rank = 0;
    for (int j = 0; j < m; ++j) rank += list.key[j] > v || (list.key[j] == v && list.at[j] < at);
    if (rank < k) f(rank, at);
  }
}

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(256) void top_logits_kernel(const T* __restrict__ X, long ld, int V, int k,
                                                         T* __restrict__ values, int64_t* __restrict__ indices) {
  __shared__ uint32_t hist[256], ckey[kTopMax];
  __shared__ int cat[kTopMax], count;
  const TopList list = {ckey, cat, &count};
  const long n = blockIdx.x;
  const T* const row = X + n * ld;
  top_exact<kKeyBits<T>>([&](int i) { return key_of(row[i]); }, V, k, hist, list);
  top_ranked(list, k, [&](int rank, int at) {
    values[n * k + rank] = row[at];
    indices[n * k + rank] = at;
  });
}

int check_top(int64_t N, int64_t V, int64_t k, int dtype, int64_t ld) {
  const int rc = check_logits_args(N, V, dtype, ld, CCE_REDUCTION_NONE, 0.f, CCE_SMOOTH_LOGV);
  if (rc) return rc;
  if (k < 1 || k > kTopMax || k > V)
    return fail(CCE_ERR_INVALID_ARG, "k must be in [1, min(%d, V = %ld)] (got %ld)", kTopMax, (long)V, (long)k);
  return CCE_OK;
}
