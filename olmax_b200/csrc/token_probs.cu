// The distribution of an LM head: log probabilities of given tokens, entropy and top classes; distillation from a teacher's top
// classes; the gradients of both with respect to the logits.  See token_probs.h for the definitions.
//
// Everything here reads long rows of logits and is bound by HBM (a byte of logits costs 1.5 instructions at most if it is to be
// read at full rate), so that a row is read once per direction: statistics are kept as (maximum, sums of exponentials relative to
// it; token_stats.cuh), and the top classes are found on the way.
#include "token_probs.h"
#include "host_common.h"

#include <limits.h>
#include <type_traits>
#include "token_stats.cuh"

namespace ob {

constexpr int TP_THREADS = 256;
template <class T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16(x); }

__device__ __forceinline__ Stats block_combine(Stats a, Stats* red, float c) {
  a = shuffle_combine(a, 16, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
  return shuffle_combine(red[threadIdx.x % (TP_THREADS / 32)], TP_THREADS / 64, c);
}

// A row as 16-byte vectors between a head and a tail of single classes: rows start at any multiple of the element size.
template <class T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  const T* z;
  int head, nvec, tail;   // classes, vectors, classes
  __device__ __forceinline__ Row(const T* row, int V) : z(row) {
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    head = min(V, lead);
    nvec = (V - head) / N;
    tail = V - head - nvec * N;
  }
  __device__ __forceinline__ int class_of(int vec) const { return head + vec * N; }
  __device__ __forceinline__ uint4 load(int vec) const { return reinterpret_cast<const uint4*>(z + head)[vec]; }
  // the single class of thread t in the head (t < head) or the tail, or -1
  __device__ __forceinline__ int single(int t, bool first, bool last) const {
    if (t < N) return first && t < head ? t : -1;
    t -= N;
    return last && t < tail ? head + nvec * N + t : -1;
  }
};
template <class T>
__device__ __forceinline__ void unpack(uint4 v, float* f);
template <>
__device__ __forceinline__ void unpack<float>(uint4 v, float* f) {
  f[0] = __uint_as_float(v.x);
  f[1] = __uint_as_float(v.y);
  f[2] = __uint_as_float(v.z);
  f[3] = __uint_as_float(v.w);
}
template <>
__device__ __forceinline__ void unpack<bf16>(uint4 v, float* f) {
  const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
// sixteen bytes of -inf: classes that are not there
template <class T>
__device__ __forceinline__ uint4 no_vector() {
  const unsigned u = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  return make_uint4(u, u, u, u);
}
// the vectors first, first + TP_THREADS, ... below `end`; `whole`: the batch has all of them, for every thread
template <class T, int U>
__device__ __forceinline__ void load_batch(const Row<T>& r, int first, bool whole, int end, uint4 (&v)[U]) {
  if (whole) {
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = r.load(first + k * TP_THREADS);
  } else {
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = first + k * TP_THREADS < end ? r.load(first + k * TP_THREADS) : no_vector<T>();
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Top classes.  Order of the classes: larger logits first (NaN before all, -0 equal to 0), then lower classes.
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned order_key(float z) {
  if (z != z) return 0xffffffffu;
  const unsigned u = __float_as_uint(z + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_logit(unsigned key) {
  return key == 0xffffffffu ? NAN : __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
// Every class has a key above 0.

// What a row's (or slice's) top classes are found from, in shared memory.  The row is read in batches; what a thread reads of a batch is a group,
// known by its largest logit.  Group g is the batch g / TP_THREADS of thread g % TP_THREADS.
struct TopWork {
  static constexpr int EVERY = 4;                          // batches between two looks at the number of groups, but for the first ones
  static constexpr int LIMIT = 1536;                       // groups kept from one look to the next
  static constexpr int GROUPS = LIMIT + EVERY * TP_THREADS;   // ... and those that come until then
  static constexpr int STEP = 128;
  static constexpr int CLASSES = 512;
  unsigned group_key[GROUPS];
  int group[GROUPS];
  unsigned long long code[CLASSES];   // in order of the classes: order_code
  int groups, classes, kept;
  int red[2][TP_THREADS / 32];
};
static_assert(TopWork::LIMIT >= TP_THREADS + OB_TOP_K_MAX && TopWork::CLASSES > OB_TOP_K_MAX, "what drop_groups and collect_classes leave");

// Larger codes come first.
__device__ __forceinline__ unsigned long long order_code(unsigned key, int cls) {
  return (unsigned long long)key << 32 | (unsigned)~cls;
}

__device__ __forceinline__ int block_sum(int c, int* red) {
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = c;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, (threadIdx.x & 31) < TP_THREADS / 32 ? red[threadIdx.x & 31] : 0);
}

// The k-th in order of the members that count(pred) counts with pred(key, place): its key and the last place of that key among the first k.
// There are k of them.  All threads call it.
template <class F>
__device__ void kth_in_order(F count, int k, unsigned& key, int& place) {
  key = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned next = key | (1u << bit);
    if (count([&](unsigned q, int) { return q >= next; }) >= k) key = next;
  }
  const int above = count([&](unsigned q, int) { return q > key; });
  place = 0;
  for (int bit = 30; bit >= 0; --bit) {
    const int next = place | (1 << bit);
    if (count([&](unsigned q, int i) { return q == key && i < next; }) < k - above) place = next;
  }
}

// The groups of a batch have been too many (rising logits, or the same ones over and over): drops those that hold none of the first k classes.  The
// k-th largest of the groups' maxima is a bound that k classes reach, none of them behind the batch up to which k groups reach it;
// groups of later batches have to be above it.  What stays are fewer than k groups above, fewer than k at the bound of earlier batches
// and the groups of one batch; their number is returned.
__device__ __noinline__ int drop_groups(TopWork& w, int k, unsigned& cut) {
  const int n = w.groups;
  int turn = 0;
  unsigned key;
  int batch;
  kth_in_order(
      [&](auto pred) {
        int x = 0;
        for (int i = threadIdx.x; i < n; i += TP_THREADS) x += pred(w.group_key[i], w.group[i] / TP_THREADS);
        turn ^= 1;   // (two buffers: a thread is at most one sum ahead of the slowest reader)
        return block_sum(x, w.red[turn]);
      },
      k, key, batch);
  if (threadIdx.x == 0) w.kept = 0;
  // in place: a group moves to where an earlier chunk, or its own, has been read
  for (int i0 = 0; i0 < n; i0 += TP_THREADS) {
    const int i = i0 + threadIdx.x;
    const unsigned q = i < n ? w.group_key[i] : 0u;
    const int g = i < n ? w.group[i] : 0;
    __syncthreads();
    if (i < n && (q > key || (q == key && g / TP_THREADS <= batch))) {
      const int at = atomicAdd(&w.kept, 1);
      w.group_key[at] = q;
      w.group[at] = g;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) w.groups = w.kept;
  cut = max(cut, key);
  __syncthreads();
  return w.kept;
}

// A lower bound of the k-th largest of one key per thread (0: none), exact in its upper 16 bits.
__device__ __forceinline__ unsigned kth_of_threads(unsigned key, int k) {
  unsigned cut = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const unsigned next = cut | (1u << bit);
    if (__syncthreads_count(key >= next) >= k) cut = next;
  }
  return cut;
}

// The classes of the groups at or above `cut` that reach it themselves, and those of the row's head and tail (`single` of this thread, or -1), as
// w.code: at most CLASSES, and the first k among them.  Returns how many.
template <class T, int U>
__device__ int collect_classes(TopWork& w, const Row<T>& r, int v0, int v1, int single, int k, unsigned cut) {
  constexpr int N = Row<T>::N;
  const int n = w.groups;
  // visit(key, class) for this thread's share of the classes
  auto each = [&](auto visit) {
    for (int t = threadIdx.x; t < n * U; t += TP_THREADS) {
      if (w.group_key[t / U] < cut) continue;
      const int g = w.group[t / U], vec = v0 + (g / TP_THREADS * U + t % U) * TP_THREADS + g % TP_THREADS;
      if (vec >= v1) continue;
      float f[N];
      unpack<T>(r.load(vec), f);
#pragma unroll
      for (int j = 0; j < N; ++j) visit(order_key(f[j]), r.class_of(vec) + j);
    }
    if (single >= 0) visit(order_key(to_f(r.z[single])), single);
  };
  if (threadIdx.x == 0) w.classes = 0;
  __syncthreads();
  each([&](unsigned key, int i) {
    if (key < cut) return;
    const int at = atomicAdd(&w.classes, 1);
    if (at < TopWork::CLASSES) w.code[at] = order_code(key, i);
  });
  __syncthreads();
  int found = w.classes;
  if (found <= TopWork::CLASSES) return found;
  // more equal or nearly equal logits than there is room for: the k-th class exactly, then the first k
  unsigned key;
  int cls, turn = 0;
  kth_in_order(
      [&](auto pred) {
        int x = 0;
        each([&](unsigned q, int i) { x += pred(q, i); });
        turn ^= 1;
        return block_sum(x, w.red[turn]);
      },
      k, key, cls);
  if (threadIdx.x == 0) w.classes = 0;
  __syncthreads();
  each([&](unsigned q, int i) {
    if (q < key || (q == key && i > cls)) return;
    w.code[atomicAdd(&w.classes, 1)] = order_code(q, i);
  });
  __syncthreads();
  return w.classes;
}

// log p of a class with capped logit y, and the entropy.  Neither passes 0 by the roundings of a soft-capped maximum; a NaN stays.
__device__ __forceinline__ float log_prob(float y, float m, float log_s, const Scaling& sc) {
  if (y == -INFINITY) return log_s == log_s ? y : log_s;
  const float lp = LN2 * ((y - m) * sc.c - log_s);
  return lp > 0.f ? 0.f : lp;
}
__device__ __forceinline__ float entropy_of(Stats a, float log_s) {
  const float h = LN2 * (log_s - a.w / a.s);
  return no_class(a) || h < 0.f ? 0.f : h;
}

struct ScoreArgs {
  const long long* ids;
  float *log_probs, *entropy, *norm;
  int top_k;
  float* top_log_probs;
  long long* top_ids;
  int V, ignore_index;
  Scaling sc;
};

// What a CTA of a row's cluster leaves with the first one.
struct Slice {
  unsigned long long code[OB_TOP_K_MAX];   // 0: no class
};

// (forms that do not ask for a converged warp)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void store_cluster(uint32_t addr, float x) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, unsigned long long x) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(x) : "memory");
}

// Log probabilities, entropy and top classes.  A row belongs to a cluster of C CTAs (C = 1 but for few rows), a slice of its vectors to
// each; the first CTA joins the slices' statistics and top classes through distributed shared memory.  Every thread has U 16-byte
// loads in flight (AHEAD: those of the next batch) and takes the maximum of the batch before its exponentials.
// Top classes in the same pass, at one comparison per thread and batch: a group (TopWork) is kept if its largest logit is above `cut`, a
// lower bound of the row's k-th largest logit that k classes of earlier batches reach, so that no class of a later one at the bound is among the
// first k.  The bound is the k-th largest of the threads' maxima so far, which some 256 ln(256 / (256 - k)) classes reach if they are spread over
// the threads by chance (1.15 k at 64, 1.4 k at 128; more by the bound's upper 16 bits only, and any number in a bad order: more than CLASSES are
// sorted out exactly); it is looked for at the first batch, whenever STEP more groups have come together, and at the end if there are many.  Then the
// classes of the groups above it are read again and put in order.
// Bound by HBM in fp32 (2048 x 100352: 132 us, 6.2 TB/s), by loads and the special-function unit in bf16 (80 us, 5.1 TB/s), by instructions with a
// soft-cap (118 us; 184 us where an eighth of the logits lie beyond 3/4 of the cap); the 64 top classes add 42 us to the first (instructions and barriers of the selection).
template <class T, int U, bool CAP, bool TOP>
__global__ void __launch_bounds__(TP_THREADS, TOP || CAP ? 4 : sizeof(T) == 2 ? 5 : 6)
    token_log_probs_fwd_kernel(const T* __restrict__ logits, long long ld, int C, ScoreArgs p) {
  constexpr int N = Row<T>::N, E = U * N;
  constexpr bool AHEAD = TOP || CAP || sizeof(T) == 2;
  extern __shared__ __align__(16) char shared_bytes[];
  TopWork& work = *reinterpret_cast<TopWork*>(shared_bytes);                     // TOP
  Slice* slices = reinterpret_cast<Slice*>(shared_bytes + sizeof(TopWork));      // TOP, one per CTA of the cluster
  __shared__ Stats red[TP_THREADS / 32], parts[8];
  if (C > 1) cluster_arrive();
  const long long row = blockIdx.x / (unsigned)C;
  const int part = (int)(blockIdx.x - row * C);
  const Row<T> r(logits + row * ld, p.V);
  const int v0 = (int)((long long)r.nvec * part / C), v1 = (int)((long long)r.nvec * (part + 1) / C);
  uint4 v[U];
  auto load = [&](int b) { load_batch<T, U>(r, b + threadIdx.x, b + TP_THREADS * U <= v1, v1, v); };
  load(v0);
  float taken = 0.f;
  bool known = false;
  if (part == 0 && threadIdx.x == 0 && p.log_probs != nullptr) {
    const long long id = p.ids[row];
    known = id != (long long)p.ignore_index && id >= 0 && id < p.V;
    if (known) taken = to_f(r.z[id]);
  }
  Stats a = empty_stats();
  unsigned cut = 0, best = 0;
  int limit = TopWork::STEP, end = 0;
  if (TOP && threadIdx.x == 0) work.groups = 0;
  if (TOP) __syncthreads();
  const int single = r.single(threadIdx.x, part == 0, part == C - 1);
  if (single >= 0) add_class(a, p.sc.capped(to_f(r.z[single])), p.sc);
  for (int b = v0, batch = 0; b < v1; b += TP_THREADS * U, ++batch) {
    float f[E];
    if (!AHEAD && b > v0) load(b);
#pragma unroll
    for (int k = 0; k < U; ++k) unpack<T>(v[k], f + k * N);
    if (AHEAD) load(b + TP_THREADS * U);
    const float mx = largest(f);
    if (CAP) {
      float y[E];
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = f[j];
      p.sc.cap_logits(y);
      if (b + TP_THREADS * U > v1) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (b + j / N * TP_THREADS + (int)threadIdx.x >= v1) y[j] = ABSENT;
      }
      add_capped<true, E>(a, y, p.sc);
    } else {
      add_classes<false, true, E>(a, f, mx, p.sc);
    }
    if (TOP) {
      const int first = b + threadIdx.x;
      unsigned key = first < v1 ? order_key(mx) : 0u;
      if (a.s != a.s) {   // a NaN, in this batch or before, comes first but is no maximum
        for (int k = 0; k < U && first + k * TP_THREADS < v1; ++k) {
          float x[N];
          unpack<T>(r.load(first + k * TP_THREADS), x);
          for (int j = 0; j < N; ++j)
            if (x[j] != x[j]) key = 0xffffffffu;
        }
      }
      best = max(best, key);
      if (b == v0) cut = kth_of_threads(best, p.top_k);
      if (b == v0 ? key != 0u && key >= cut : key > cut) {
        const int at = atomicAdd(&work.groups, 1);
        work.group_key[at] = key;
        work.group[at] = batch * TP_THREADS + threadIdx.x;
        end = at + 1;
      }
      // (every thread's last group, not the counter: a faster thread may already be adding to that)
      if ((batch < TopWork::EVERY || batch % TopWork::EVERY == TopWork::EVERY - 1) && __syncthreads_or(end > limit)) {
        int n = work.groups;
        if (n > TopWork::LIMIT) {
          n = drop_groups(work, p.top_k, cut);
          end = 0;
        } else {
          cut = max(cut, kth_of_threads(best, p.top_k));
        }
        limit = min(n + TopWork::STEP, TopWork::LIMIT);
      }
    }
  }
  a = block_combine(a, red, p.sc.c);
  if (C > 1) cluster_wait();   // the first CTA runs
  if (TOP) {
    // the slice's first k classes in order; few groups are not worth a better bound
    if (work.groups > TopWork::STEP) cut = max(cut, kth_of_threads(best, p.top_k));
    const int n = collect_classes<T, U>(work, r, v0, v1, single, p.top_k, cut);
    uint32_t codes = smem_u32(slices[part].code);
    if (C > 1) codes = mapa_shared(codes, 0);
    for (int t = threadIdx.x; t < n; t += TP_THREADS) {
      const unsigned long long code = work.code[t];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += work.code[j] > code;
      if (rank < p.top_k) store_cluster(codes + rank * 8, code);
    }
    for (int t = n + threadIdx.x; t < p.top_k; t += TP_THREADS) store_cluster(codes + t * 8, 0ull);
  }
  if (C > 1) {
    if (threadIdx.x == 0) {
      const uint32_t at = mapa_shared(smem_u32(&parts[part]), 0);
      store_cluster(at, a.m);
      store_cluster(at + 4, a.s);
      store_cluster(at + 8, a.w);
    }
    cluster_arrive();
    cluster_wait();
    if (part != 0) return;
    a = parts[0];
    for (int i = 1; i < C; ++i) a = combine(a, parts[i], p.sc.c);
  } else if (TOP) {
    __syncthreads();
  }
  const float log_s = log2f(a.s);
  auto log_p = [&](float z) { return log_prob(CAP ? p.sc.capped(z) : z, a.m, log_s, p.sc); };
  if (threadIdx.x == 0) {
    if (p.log_probs != nullptr) p.log_probs[row] = known ? log_p(taken) : 0.f;
    if (p.entropy != nullptr) p.entropy[row] = entropy_of(a, log_s);
    if (p.norm != nullptr) *reinterpret_cast<float2*>(p.norm + row * 2) = make_float2(a.m, log_s);
  }
  if (TOP) {
    // the place of a class among all slices: its own in its list and, of every other, the number of classes before it
    for (int t = threadIdx.x; t < C * p.top_k; t += TP_THREADS) {
      const int own = t / p.top_k;
      int rank = t - own * p.top_k;
      const unsigned long long code = slices[own].code[rank];
      if (code == 0) continue;
      for (int s = 0; s < C; ++s) {
        if (s == own) continue;
        int lo = 0, hi = p.top_k;   // classes [0, lo) of the list come before, [hi, k) after
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (slices[s].code[mid] > code) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      if (rank < p.top_k) {
        p.top_log_probs[row * p.top_k + rank] = log_p(key_logit((unsigned)(code >> 32)));
        p.top_ids[row * p.top_k + rank] = ~(unsigned)code;
      }
    }
  }
}

// The scores of rows whose statistics lie in `n` parts, parts[i * stride + row] = (m, s, w, -).  A block has 32 rows: a warp reads every 32nd part of
// them, row by lane, and joins one row, part by lane.  Bound by latency: 7.7 us with cold caches for 1024 rows of the 50304-class head.
__global__ void __launch_bounds__(1024)
    join_scores_kernel(const float4* __restrict__ parts, const float* __restrict__ target, long long stride, int n, long long rows,
                       ScoreArgs p) {
  __shared__ Stats red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row0 = (long long)blockIdx.x * 32, row = row0 + warp;
  constexpr int U = 4;
  Stats a = empty_stats();
  if (row0 + lane < rows) {
    for (int i0 = warp; i0 < n; i0 += 32 * U) {
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        x[u] = i0 + u * 32 < n ? parts[(i0 + u * 32) * stride + row0 + lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) a = combine(a, Stats{x[u].x, x[u].y, x[u].z}, p.sc.c);
    }
  }
  red[warp][lane] = a;
  __syncthreads();
  a = shuffle_combine(red[lane][warp], 16, p.sc.c);
  if (lane != 0 || row >= rows) return;
  const float log_s = log2f(a.s);
  if (p.log_probs != nullptr) {
    const long long id = p.ids[row];
    float lp = 0.f;
    if (id != (long long)p.ignore_index && id >= 0 && id < p.V) {
      lp = log_prob(p.sc.capped(target[row]), a.m, log_s, p.sc);
    }
    p.log_probs[row] = lp;
  }
  p.entropy[row] = entropy_of(a, log_s);
  if (p.norm != nullptr) *reinterpret_cast<float2*>(p.norm + row * 2) = make_float2(a.m, log_s);
}

// ---------------------------------------------------------------------------------------------------------------------
// Gradients: every class's from its logit and a few numbers of the row.  A block takes a span of a row, blocks in launch order.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int GRAD_THREADS = 256, GRAD_UNROLL = 2;

// N gradients to where they lie side by side, N * sizeof(D) bytes aligned alike
template <class D, int N>
__device__ __forceinline__ void store_vector(D* d, const float (&g)[N]);
template <>
__device__ __forceinline__ void store_vector<float, 4>(float* d, const float (&g)[4]) {
  *reinterpret_cast<float4*>(d) = make_float4(g[0], g[1], g[2], g[3]);
}
template <>
__device__ __forceinline__ void store_vector<bf16, 4>(bf16* d, const float (&g)[4]) {
  *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]));
}
template <>
__device__ __forceinline__ void store_vector<bf16, 8>(bf16* d, const float (&g)[8]) {
  *reinterpret_cast<uint4*>(d) = make_uint4(pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3]), pack_bf16x2(g[4], g[5]), pack_bf16x2(g[6], g[7]));
}

// The span `part` of `per_block` vectors of a row and its gradient, for the classes [lo, hi), which it returns: grad(f, i) turns
// an array f of the logits of classes i, i + 1, ... into their gradients.
// The gradient is written in vectors where its row is aligned like the logits', else class by class.
template <class T, class D, class F>
__device__ __forceinline__ int2 map_span(const T* z, D* d, int V, int part, int parts, int per_block, F grad) {
  constexpr int N = Row<T>::N;
  const Row<T> r(z, V);
  const int v0 = min(r.nvec, part * per_block), v1 = part == parts - 1 ? r.nvec : min(r.nvec, v0 + per_block);
  const int lo = part == 0 ? 0 : r.class_of(v0), hi = part == parts - 1 ? V : r.class_of(v1);
  if ((reinterpret_cast<uintptr_t>(d + r.head) & (N * sizeof(D) - 1)) != 0) {
    for (int i = lo + threadIdx.x; i < hi; i += GRAD_THREADS) {
      float f[1] = {to_f(z[i])};
      grad(f, i);
      d[i] = from_f<D>(f[0]);
    }
    return make_int2(lo, hi);
  }
  uint4 next[GRAD_UNROLL];
  auto load = [&](int b) {
#pragma unroll
    for (int k = 0; k < GRAD_UNROLL; ++k)
      if (b + k * GRAD_THREADS < v1) next[k] = r.load(b + k * GRAD_THREADS);
  };
  load(v0 + threadIdx.x);
  for (int b = v0 + threadIdx.x; b < v1; b += GRAD_THREADS * GRAD_UNROLL) {
    uint4 v[GRAD_UNROLL];
#pragma unroll
    for (int k = 0; k < GRAD_UNROLL; ++k) v[k] = next[k];
    load(b + GRAD_THREADS * GRAD_UNROLL);
#pragma unroll
    for (int k = 0; k < GRAD_UNROLL; ++k) {
      const int i = b + k * GRAD_THREADS;
      if (i >= v1) break;
      float f[N];
      unpack<T>(v[k], f);
      const int cls = r.class_of(i);
      grad(f, cls);
      store_vector<D, N>(d + cls, f);
    }
  }
  const int single = r.single(threadIdx.x, part == 0, part == parts - 1);
  if (single >= 0) {
    float f[1] = {to_f(z[single])};
    grad(f, single);
    d[single] = from_f<D>(f[0]);
  }
  return make_int2(lo, hi);
}

struct ScoreGradArgs {
  const long long* ids;
  const float2* norm;
  const float *entropy, *g_log_probs, *g_entropy;
  long long stride_lp, stride_ent;
  int V, ignore_index;
  Scaling sc;
};

// dz = dy/dz (g_lp (onehot - p) - g_H p (log p + H)) = dy/dz (g_lp onehot - p (k0 + k1 t)) with t = log2 p.
// One read and one write of a class: 2048 x 100352 fp32 243 us, bf16 131 us (6.8 and 6.3 TB/s, HBM), with a soft-cap 153 us (instructions; 231 us
// where an eighth of the logits lie beyond 3/4 of the cap).
template <class T, class D, bool CAP>
__global__ void __launch_bounds__(GRAD_THREADS, CAP && sizeof(T) == 2 ? 5 : 6)
    token_log_probs_bwd_kernel(const T* __restrict__ logits, long long ld, D* __restrict__ dlogits, long long ld_d, int parts,
                               int per_block, ScoreGradArgs p) {
  const long long row = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - row * parts);
  float2 norm = p.norm[row];
  const float ge = p.g_entropy != nullptr ? p.g_entropy[row * p.stride_ent] : 0.f;
  float gl = 0.f;
  int id = -1;
  if (p.g_log_probs != nullptr) {
    const long long i = p.ids[row];
    if (i != (long long)p.ignore_index && i >= 0 && i < p.V) {
      gl = p.g_log_probs[row * p.stride_lp];
      id = (int)i;
    }
  }
  float k0 = (gl + ge * (ge != 0.f ? p.entropy[row] : 0.f)) * p.sc.inv_temp, k1 = ge * LN2 * p.sc.inv_temp;
  gl *= p.sc.inv_temp;
  if (norm.x == -INFINITY && norm.y == -INFINITY) {   // no class: exponents of -inf and factors of 0
    norm = make_float2(0.f, 0.f);
    k0 = k1 = gl = 0.f;
  }
  k0 = -k0, k1 = -k1;
  const float t0 = fmaf(-norm.x, p.sc.c, -norm.y);   // (capped logits are small: one rounding of this is no more than theirs)
  map_span<T, D>(logits + row * ld, dlogits + row * ld_d, p.V, part, parts, per_block, [&](auto& f, int i) {
    constexpr int M = sizeof(f) / sizeof(float);
    float slope[M];
    if (CAP) p.sc.template cap_logits<true>(f, slope);
    auto pair = [&](float2 x) {
      const float2 t = CAP ? fma2(x, make_float2(p.sc.c, p.sc.c), make_float2(t0, t0))
                           : fma2(add2(x, make_float2(-norm.x, -norm.x)), make_float2(p.sc.c, p.sc.c), make_float2(-norm.y, -norm.y));
      // (2^t is 0 from -150 on; what it is multiplied by stays finite)
      const float2 u = CAP ? t : make_float2(fmaxf(t.x, -1024.f), fmaxf(t.y, -1024.f));
      return mul2(make_float2(exp2_fast(t.x), exp2_fast(t.y)), fma2(u, make_float2(k1, k1), make_float2(k0, k0)));
    };
    float g[M + 1];
#pragma unroll
    for (int j = 0; j < M; j += 2) {
      const float2 o = pair(make_float2(f[j], j + 1 < M ? f[j + 1] : f[j]));
      g[j] = o.x;
      g[j + 1] = o.y;
    }
    if ((unsigned)(id - i) < (unsigned)M) {
#pragma unroll
      for (int j = 0; j < M; ++j)
        if (i + j == id) g[j] += gl;
    }
#pragma unroll
    for (int j = 0; j < M; ++j) f[j] = CAP ? g[j] * slope[j] : g[j];
  });
}

// ---------------------------------------------------------------------------------------------------------------------
// Distillation.  S: the classes that the teacher names, t_i its values, q_i its masses; L the log-sum-exp of the student's other classes.
//   loss = sum_S q (log q - log p) + rest_q (log rest_q - (L - lse)),   M = sum_S q + rest_q
//   d/dy_j = M p_j - q_j in S,   e^(y_j - L) (M e^(L - lse) - rest_q) outside
// L has its own maximum and sum over the classes outside S: 1 - sum_S p would lose what a confident student leaves to the rest.
// The teacher's masses are summed in 64 bits for the same reason, and lse is L joined with the named classes in 64 bits, so that L's own error is the
// same in both and leaves the loss where the rest has most of the mass (2e-9 of a loss of 1e-5; 1.5e-7 with a join in 32).
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ long long teacher_id(const void* ids, int ids_64, long long at) {
  return ids_64 ? reinterpret_cast<const long long*>(ids)[at] : (long long)reinterpret_cast<const int*>(ids)[at];
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

struct DistillArgs {
  const void* teacher_ids;
  const float* teacher_log_probs;
  int ids_64, k, renormalize;
  long long ld_t;
  float *row_loss, *row_stats, *q;
  int V;
  double inv_temp;
  Scaling sc;
};

// f <- gradients of classes outside the teacher's with logits f: coef * 2^((cap(f) - m) c - log_s) [* slope]; zeros whatever f is if `zero`.
template <bool CAP, int M>
__device__ __forceinline__ void rest_gradient(float (&f)[M], bool zero, float m, float log_s, float coef, const Scaling& sc) {
  if (zero) {
#pragma unroll
    for (int j = 0; j < M; ++j) f[j] = 0.f;
    return;
  }
  float slope[M];
  if (CAP) sc.template cap_logits<true>(f, slope);
  const float t0 = fmaf(-m, sc.c, -log_s);   // (as in the gradient of the scores)
  float g[M + 1];
#pragma unroll
  for (int j = 0; j < M; j += 2) {
    const float2 x = make_float2(f[j], j + 1 < M ? f[j + 1] : f[j]);
    const float2 t = CAP ? fma2(x, make_float2(sc.c, sc.c), make_float2(t0, t0))
                         : fma2(add2(x, make_float2(-m, -m)), make_float2(sc.c, sc.c), make_float2(-log_s, -log_s));
    const float2 o = mul2(make_float2(exp2_fast(t.x), exp2_fast(t.y)), make_float2(coef, coef));
    g[j] = o.x;
    g[j + 1] = o.y;
  }
#pragma unroll
  for (int j = 0; j < M; ++j) f[j] = CAP ? g[j] * slope[j] : g[j];
}

// Sums over the block, the same in every thread.
__device__ __forceinline__ double block_sum(double x, double* red) {
  x = warp_sum(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < TP_THREADS / 32; ++i) t += red[i];
  return t;
}

// A row belongs to a cluster of C CTAs as in the log probabilities.  Thread t holds the teacher's pair t.  One bit of shared memory per vector, the
// bits of a thread's batch side by side, says whether the teacher names one of its classes, one bit per class which: a batch without one, and
// that is most of them, costs one look.
// With 64 classes named, 2048 x 100352: fp32 140 us (5.9 TB/s, HBM), bf16 100 us (loads), with a soft-cap 133 us (instructions; 145 with five CTAs per SM
// and no batch ahead).
template <class T, int U, bool CAP>
__global__ void __launch_bounds__(TP_THREADS, CAP ? 4 : 6)
    distill_fwd_kernel(const T* __restrict__ logits, long long ld, int C, int slice_vectors, DistillArgs p) {
  constexpr int N = Row<T>::N, E = U * N;
  extern __shared__ __align__(16) char shared_bytes[];
  unsigned* flags = reinterpret_cast<unsigned*>(shared_bytes);   // a bit per vector, whole batches
  const int flag_words = (slice_vectors + TP_THREADS * U - 1) / (TP_THREADS * U) * (TP_THREADS * U / 32);
  unsigned* named = flags + flag_words;                          // a bit per class
  __shared__ Stats red[TP_THREADS / 32], parts[8];
  __shared__ double red_d[TP_THREADS / 32];
  __shared__ int cls_s[OB_TOP_K_MAX];
  if (C > 1) cluster_arrive();
  const long long row = blockIdx.x / (unsigned)C;
  const int part = (int)(blockIdx.x - row * C);
  const Row<T> r(logits + row * ld, p.V);
  const int v0 = (int)((long long)r.nvec * part / C), v1 = (int)((long long)r.nvec * (part + 1) / C);
  const int c0 = r.class_of(v0), c1 = r.class_of(v1);
  const int lo = part == 0 ? 0 : c0, hi = part == C - 1 ? p.V : c1;
  const int shift = N - c0;   // the bit of class i is i + shift: vectors begin at multiples of N, the row's head lies in front of the first

  // ---- the classes that the teacher names
  int id = -1;
  float t = -INFINITY, y = -INFINITY;
  if ((int)threadIdx.x < p.k) {
    const long long i = teacher_id(p.teacher_ids, p.ids_64, row * p.ld_t + threadIdx.x);
    if (i >= 0 && i < p.V) {
      id = (int)i;
      t = p.teacher_log_probs[row * p.ld_t + threadIdx.x];
      y = to_f(r.z[i]);   // (waited for at the end)
    }
  }
  if (threadIdx.x < OB_TOP_K_MAX) cls_s[threadIdx.x] = id;
  for (int i = threadIdx.x; i < flag_words; i += TP_THREADS) flags[i] = 0;
  for (int i = threadIdx.x; i < (hi + shift + 31) / 32; i += TP_THREADS) named[i] = 0;
  __syncthreads();
  bool again = C > 1 && id >= 0;   // (another slice's bits are not here to tell)
  if (id >= lo && id < hi) {
    const unsigned bit = 1u << ((id + shift) & 31);
    again |= (atomicOr(&named[(id + shift) >> 5], bit) & bit) != 0;
    if (id >= c0 && id < c1) {
      const int vec = (id - c0) / N, at = (vec / (TP_THREADS * U) * TP_THREADS + vec % TP_THREADS) * U + vec / TP_THREADS % U;
      atomicOr(&flags[at >> 5], 1u << (at & 31));
    }
  }
  bool in = id >= 0;
  if (__syncthreads_or(again) && in) {   // of several pairs with one class the first counts
    for (int j = 0; j < (int)threadIdx.x; ++j) in &= cls_s[j] != id;
  }

  // ---- the statistics of the others
  Stats a = empty_stats();
  auto is_named = [&](int i) { return (named[(i + shift) >> 5] >> ((i + shift) & 31)) & 1; };
  const int single = r.single(threadIdx.x, part == 0, part == C - 1);
  if (single >= 0 && !is_named(single)) add_class(a, p.sc.capped(to_f(r.z[single])), p.sc);
  uint4 v[U];
  auto load = [&](int b) { load_batch<T, U>(r, b + threadIdx.x, b + TP_THREADS * U <= v1, v1, v); };
  if (CAP) load(v0);   // (the next batch ahead: the instructions of this one hide it)
  for (int b = v0, batch = 0; b < v1; b += TP_THREADS * U, ++batch) {
    if (!CAP) load(b);
    float f[E];
#pragma unroll
    for (int k = 0; k < U; ++k) unpack<T>(v[k], f + k * N);
    if (CAP) load(b + TP_THREADS * U);
    if (CAP) p.sc.cap_logits(f);
    const int bit = (batch * TP_THREADS + threadIdx.x) * U;
    const unsigned some = (flags[bit >> 5] >> (bit & 31)) & ((1u << U) - 1);
    if (some) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int at = (b - v0 + k * TP_THREADS + threadIdx.x + 1) * N;
        const unsigned out = (some >> k) & 1 ? named[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int j = 0; j < N; ++j)
          if ((out >> j) & 1) f[k * N + j] = CAP ? ABSENT : -INFINITY;
      }
    }
    if (CAP && b + TP_THREADS * U > v1) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (b + j / N * TP_THREADS + (int)threadIdx.x >= v1) f[j] = ABSENT;
    }
    if (CAP) {
      add_capped<false, E>(a, f, p.sc);
    } else {
      add_classes<false, false, E>(a, f, largest(f), p.sc);
    }
  }
  a = block_combine(a, red, p.sc.c);
  if (C > 1) {
    cluster_wait();   // the first CTA runs
    if (threadIdx.x == 0) {
      const uint32_t at = mapa_shared(smem_u32(&parts[part]), 0);
      store_cluster(at, a.m);
      store_cluster(at + 4, a.s);
    }
    cluster_arrive();
    cluster_wait();
    if (part != 0) return;
    a = Stats{parts[0].m, parts[0].s, 0.f};
    for (int i = 1; i < C; ++i) a = combine(a, Stats{parts[i].m, parts[i].s, 0.f}, p.sc.c);
  }

  // ---- the teacher and the row
  if (!in) t = -INFINITY;
  y = in ? p.sc.capped(y) : -INFINITY;
  Stats st = empty_stats();
  if (in) add_class(st, y, p.sc);
  st = block_combine(st, red, p.sc.c);
  const Stats all = combine(st, a, p.sc.c);
  double t_shift = 0.0;
  if (p.renormalize) {
    float t_max = t;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) t_max = fmaxf(t_max, __shfl_xor_sync(0xffffffffu, t_max, off));
    if ((threadIdx.x & 31) == 0) red_d[threadIdx.x >> 5] = (double)t_max;
    __syncthreads();
    for (int i = 0; i < OB_TOP_K_MAX / 32; ++i) t_max = fmaxf(t_max, (float)red_d[i]);
    if (t_max > -INFINITY) t_shift = (double)t_max;
  }
  const bool any = __syncthreads_or(in && !(p.renormalize && t == -INFINITY));
  double q = in ? exp((double)t - t_shift) : 0.0;
  const double sum = block_sum(q, red_d);
  const bool others = !no_class(a);
  double mass = sum, rest = 0.0, log_norm = t_shift;
  if (p.renormalize) {
    log_norm += log(sum);
    mass = 1.0;
    q /= sum;
  } else if (others) {
    rest = fmax(0.0, 1.0 - sum);
  }
  // sum q (log q - log p), but for log p's common part; in 64 bits, the temperature too, for a loss that is a small difference of logarithms
  const bool none = no_class(all);
  const double log_p0 = y == -INFINITY ? -INFINITY : ((double)y - all.m) * p.inv_temp;
  double loss = block_sum(in && q != 0.0 ? q * ((double)t - log_norm - log_p0) : 0.0, red_d);
  if ((int)threadIdx.x < p.k) p.q[row * p.k + threadIdx.x] = in && any ? (float)q : -1.f;
  if (threadIdx.x == 0) {
    // (not all.s: joined in 32 bits, with a rounded c and an exponential that is low, it would differ from a.s by more than a small loss holds)
    auto share = [&](Stats x) { return x.s == 0.f ? 0.0 : x.s * exp(((double)x.m - all.m) * p.inv_temp); };
    const double log_s = none ? 0.0 : log(share(st) + share(a)), rest_log_s = others ? log((double)a.s) : 0.0;
    const double total = mass + rest, rest_lp = ((double)a.m - all.m) * p.inv_temp + rest_log_s - log_s;
    loss += mass * log_s;
    if (rest > 0.0) loss += rest * (log(rest) - rest_lp);
    p.row_loss[row] = any ? (float)loss : 0.f;
    float4* o = reinterpret_cast<float4*>(p.row_stats + row * 8);
    o[0] = make_float4(any ? (float)total : -1.f, others && any ? (float)(total * exp(rest_lp) - rest) : 0.f, 0.f, 0.f);
    o[1] = make_float4(all.m, log2f(all.s), a.m, log2f(a.s));
  }
}
static_assert(OB_TOP_K_MAX <= TP_THREADS, "one thread per class of the teacher");

struct DistillGradArgs {
  const void* teacher_ids;
  int ids_64, k;
  long long ld_t;
  const float *row_stats, *q, *g;
  long long stride_g;
  const float* inv_count;
  float scale;
  int V;
  Scaling sc;
};

// Every class as one outside the teacher's, then the teacher's anew.  2048 x 100352, 64 of the teacher's: fp32 244 us, bf16 131 us (6.7 and 6.3 TB/s,
// HBM), with a soft-cap 157 us (instructions).
template <class T, class D, bool CAP>
__global__ void __launch_bounds__(GRAD_THREADS, CAP && sizeof(T) == 2 ? 5 : 6)
    distill_bwd_kernel(const T* __restrict__ logits, long long ld, D* __restrict__ dlogits, long long ld_d, int parts, int per_block,
                       DistillGradArgs p) {
  const long long row = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - row * parts);
  const T* z = logits + row * ld;
  D* d = dlogits + row * ld_d;
  const float2 st = *reinterpret_cast<const float2*>(p.row_stats + row * 8);
  const float4 norm = *reinterpret_cast<const float4*>(p.row_stats + row * 8 + 4);
  long long id = -1;
  float q = -1.f;
  auto teacher = [&] {
    if ((int)threadIdx.x >= p.k) return;
    q = p.q[row * p.k + threadIdx.x];
    id = teacher_id(p.teacher_ids, p.ids_64, row * p.ld_t + threadIdx.x);
  };
  if (!CAP) teacher();   // (with a soft-cap the registers are short)
  const float gs = (p.g != nullptr ? p.g[row * p.stride_g] : 1.f) * p.scale * (p.inv_count != nullptr ? *p.inv_count : 1.f);
  const bool nothing = st.x < 0.f || (norm.x == -INFINITY && norm.y == -INFINITY);
  const bool zero = nothing || (norm.z == -INFINITY && norm.w == -INFINITY);   // no class outside the teacher's
  const float coef = st.y * gs * p.sc.inv_temp;
  const int2 span = map_span<T, D>(z, d, p.V, part, parts, per_block, [&](auto& f, int) {
    rest_gradient<CAP>(f, zero, norm.z, norm.w, coef, p.sc);
  });
  // the teacher's classes, over what has just been written for them
  __syncthreads();
  if (CAP) teacher();
  if (!nothing && !(q < 0.f) && id >= span.x && id < span.y) {
    float slope;
    const float x = p.sc.capped(to_f(z[id]), &slope);
    d[id] = from_f<D>((st.x * exp2_fast((x - norm.x) * p.sc.c - norm.y) - q) * gs * slope);
  }
}
static_assert(OB_TOP_K_MAX <= GRAD_THREADS, "one thread per class of the teacher");

// One block: the order of the sum does not depend on the launch.
__global__ void __launch_bounds__(1024)
    distill_reduce_kernel(const float* __restrict__ row_loss, const float* __restrict__ row_stats, long long rows, int mean,
                          float* __restrict__ loss, float* __restrict__ inv_count) {
  __shared__ double red[32];
  __shared__ int redi[32];
  double sum = 0.0;
  int n = 0;
  for (long long r = threadIdx.x; r < rows; r += 1024) {
    const bool counted = !(row_stats[r * 8] < 0.f);
    if (counted) sum += (double)row_loss[r];
    n += counted;
  }
  sum = warp_sum(sum);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = sum;
    redi[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = warp_sum(red[threadIdx.x]);
    n = __reduce_add_sync(0xffffffffu, redi[threadIdx.x]);
    if (threadIdx.x == 0) {
      const double inv = 1.0 / (double)(n > 0 ? n : 1);
      *loss = (float)(mean ? sum * inv : sum);
      if (inv_count != nullptr) *inv_count = (float)inv;
    }
  }
}

__global__ void __launch_bounds__(1024)
    distill_count_kernel(const void* __restrict__ teacher_ids, int ids_64, const float* __restrict__ teacher_log_probs,
                         long long ld_t, int k, int renormalize, long long rows, int V, float* __restrict__ inv_count) {
  __shared__ int redi[32];
  int n = 0;
  for (long long r = threadIdx.x; r < rows; r += 1024) {
    bool any = false;
    for (int i = 0; i < k && !any; ++i) {
      const long long id = teacher_id(teacher_ids, ids_64, r * ld_t + i);
      any = id >= 0 && id < V && !(renormalize && teacher_log_probs[r * ld_t + i] == -INFINITY);
      for (int j = 0; j < i && any && renormalize; ++j) any = teacher_id(teacher_ids, ids_64, r * ld_t + j) != id;   // (the first of a class counts)
    }
    n += any;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) redi[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) n = __reduce_add_sync(0xffffffffu, redi[threadIdx.x]);
  if (threadIdx.x == 0) *inv_count = 1.f / (float)(n > 0 ? n : 1);
}

static inline int check_logits(const char* what, const void* logits, int dtype, long long ld, long long rows, int V) {
  if (logits == nullptr) OB_FAIL(-1, "%s: no logits", what);
  if (dtype != OB_F32 && dtype != OB_BF16) OB_FAIL(-2, "%s: unknown type of logits %d", what, dtype);
  if (V < 1 || rows > INT_MAX || ld < 0) OB_FAIL(-3, "%s: %lld rows of %d classes, %lld apart", what, rows, V, ld);
  return 0;
}

// Shared memory beyond 48 KB is an attribute of a kernel on a device: set once for each.
template <class K>
static inline int allow_shared(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  OB_CUDA_OK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) OB_FAIL(-7, "device ordinal %d outside the supported range [0, 64)", dev);
  if (!done[dev]) {
    OB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev] = true;
  }
  return 0;
}

// CTAs per row: a power of two up to the portable cluster size, as long as there are no more than two CTAs per SM and a slice keeps a batch
// or more of every thread.  Device time at 1, 2, 4, 8 CTAs: 1 x 50304 fp32, top 5, 11.6, 10.2, 9.0, 9.2 us; 1 x 256000 bf16, top 64, 36.9, 27.2, 20.5,
// 20.8 us; 8 x 128256 bf16, top 20, 21.1, 17.4, 14.0, 12.5 us.  With up to four per SM 64 x 128256 takes 41.5 (fp32, top 128) and 17.0 us (bf16, top
// 20), with two 26.8 and 15.8.
static inline int ctas_per_row(long long rows, int V, int per_batch) {
  int C = 1;
  while (C < 8 && rows * C * 2 <= 2ll * sm_count() && V / (2 * C) >= per_batch) C *= 2;
  return C;
}

template <class K, class... Args>
static int launch_clusters(K kernel, long long blocks, int C, int shared, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(TP_THREADS);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  OB_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
  return 0;
}

template <class T, int U, bool CAP, bool TOP>
static int launch_scores(const T* logits, long long ld, long long rows, const ScoreArgs& args, cudaStream_t stream) {
  constexpr int per_batch = TP_THREADS * U * Row<T>::N;
  auto kernel = token_log_probs_fwd_kernel<T, U, CAP, TOP>;
  const int C = ctas_per_row(rows, args.V, per_batch);
  static_assert(sizeof(TopWork) + 8 * sizeof(Slice) + 1024 <= 48 * 1024, "shared memory that needs no attribute, with the static part");
  const int shared = TOP ? (int)(sizeof(TopWork) + C * sizeof(Slice)) : 0;
  return launch_clusters(kernel, rows * C, C, shared, stream, logits, ld, C, args);
}

template <class T, int U, bool CAP>
static int launch_distill(const T* logits, long long ld, long long rows, const DistillArgs& args, cudaStream_t stream) {
  constexpr int N = Row<T>::N, LIMIT = 160 * 1024;
  auto kernel = distill_fwd_kernel<T, U, CAP>;
  // a bit for each vector of whole batches and a bit for each class, with the row's head and tail; more CTAs where they do not fit
  int C = ctas_per_row(rows, args.V, TP_THREADS * U * N), vectors;
  long long bytes;
  for (;; C *= 2) {
    vectors = args.V / N / C + 1;
    bytes = (vectors + TP_THREADS * U - 1) / (TP_THREADS * U) * (TP_THREADS * U / 8) + ((long long)vectors * N + 4 * N + 31) / 32 * 4;
    if (bytes <= LIMIT) break;
    if (C == 8) OB_FAIL(-6, "distillation: no room in shared memory for the bits of %d classes", args.V);
  }
  if (rows > INT_MAX / C) OB_FAIL(-3, "distillation: %lld rows of %d classes", rows, args.V);
  static bool done[64] = {};
  if (int rc = allow_shared(kernel, LIMIT, done)) return rc;
  return launch_clusters(kernel, rows * C, C, (int)bytes, stream, logits, ld, C, vectors, args);
}

// Calls launch(z, d, parts, per_block) with the types of the logits and of their gradient and the spans of a row.
template <class F>
static int launch_gradient(const char* what, const void* z, int dtype, long long ld, void* d, int dtype_d, long long ld_d,
                           long long rows, int V, cudaStream_t stream, F launch) {
  const int N = dtype == OB_F32 ? 4 : 8;
  // four batches of every thread to a block, more where the grid would not hold the blocks
  long long per_block = 4ll * GRAD_THREADS * GRAD_UNROLL, parts = 0;
  for (;; per_block *= 2) {
    parts = (V / N + per_block - 1) / per_block;
    if (parts < 1) parts = 1;
    if (rows * parts <= INT_MAX) break;
  }
  if (dtype == OB_F32 && dtype_d == OB_F32) launch((const float*)z, (float*)d, (int)parts, (int)per_block);
  else if (dtype == OB_F32 && dtype_d == OB_BF16) launch((const float*)z, (bf16*)d, (int)parts, (int)per_block);
  else if (dtype == OB_BF16 && dtype_d == OB_BF16) launch((const bf16*)z, (bf16*)d, (int)parts, (int)per_block);
  else OB_FAIL(-2, "%s: no gradient of type %d for logits of type %d", what, dtype_d, dtype);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace ob

using namespace ob;

extern "C" int ob_token_log_probs_fwd(const void* logits, int dtype, long long ld, const long long* ids, float* log_probs,
                                      float* entropy, float* norm, int top_k, float* top_log_probs, long long* top_ids,
                                      long long rows, int V, int ignore_index, float softcap, double inv_temp,
                                      cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("token_log_probs", logits, dtype, ld, rows, V)) return rc;
  if (top_k < 0 || top_k > OB_TOP_K_MAX || top_k > V) OB_FAIL(-4, "token_log_probs: top_k %d outside [0, min(%d, %d)]", top_k, OB_TOP_K_MAX, V);
  if ((log_probs != nullptr && ids == nullptr) || (top_k > 0 && (top_log_probs == nullptr || top_ids == nullptr)))
    OB_FAIL(-5, "token_log_probs: missing tensor");
  const ScoreArgs args{ids, log_probs, entropy, norm, top_k, top_log_probs, top_ids, V, ignore_index, scaling(softcap, inv_temp)};
  const bool cap = softcap > 0.f, top = top_k > 0;
  if (dtype == OB_F32) {
    auto* z = (const float*)logits;
    if (top) return cap ? launch_scores<float, 4, true, true>(z, ld, rows, args, stream) : launch_scores<float, 4, false, true>(z, ld, rows, args, stream);
    return cap ? launch_scores<float, 4, true, false>(z, ld, rows, args, stream) : launch_scores<float, 4, false, false>(z, ld, rows, args, stream);
  }
  auto* z = (const bf16*)logits;
  if (top) return cap ? launch_scores<bf16, 2, true, true>(z, ld, rows, args, stream) : launch_scores<bf16, 2, false, true>(z, ld, rows, args, stream);
  return cap ? launch_scores<bf16, 2, true, false>(z, ld, rows, args, stream) : launch_scores<bf16, 2, false, false>(z, ld, rows, args, stream);
}

extern "C" int ob_join_scores(const float* parts, const float* target, long long stride, int n, const long long* ids, float* log_probs,
                              float* entropy, float* norm, long long rows, int V, int ignore_index, float softcap, double inv_temp,
                              cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (parts == nullptr || entropy == nullptr || (log_probs != nullptr && (ids == nullptr || target == nullptr)))
    OB_FAIL(-5, "scores of parts: missing tensor");
  if (n < 1 || stride < rows || rows > 32ll * INT_MAX) OB_FAIL(-3, "scores of parts: %lld rows in %d parts %lld apart", rows, n, stride);
  const ScoreArgs args{ids, log_probs, entropy, norm, 0, nullptr, nullptr, V, ignore_index, scaling(softcap, inv_temp)};
  join_scores_kernel<<<(unsigned)((rows + 31) / 32), 1024, 0, stream>>>((const float4*)parts, target, stride, n, rows, args);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int ob_token_log_probs_bwd(const void* logits, int dtype, long long ld, const long long* ids, const float* norm,
                                      const float* entropy, const float* g_log_probs, long long stride_lp,
                                      const float* g_entropy, long long stride_ent, void* dlogits, int dtype_d, long long ld_d,
                                      long long rows, int V, int ignore_index, float softcap, double inv_temp,
                                      cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("token_log_probs backward", logits, dtype, ld, rows, V)) return rc;
  if (norm == nullptr || dlogits == nullptr || (g_log_probs != nullptr && ids == nullptr) || (g_entropy != nullptr && entropy == nullptr))
    OB_FAIL(-5, "token_log_probs backward: missing tensor");
  const Scaling sc = scaling(softcap, inv_temp);
  const ScoreGradArgs args{ids, (const float2*)norm, entropy, g_log_probs, g_entropy, stride_lp, stride_ent, V, ignore_index, sc};
  return launch_gradient("token_log_probs backward", logits, dtype, ld, dlogits, dtype_d, ld_d, rows, V, stream,
                         [&](auto* z, auto* d, int parts, int per_block) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(z)>> T;
    typedef std::remove_pointer_t<decltype(d)> D;
    const unsigned blocks = (unsigned)(rows * parts);
    if (softcap > 0.f) token_log_probs_bwd_kernel<T, D, true><<<blocks, GRAD_THREADS, 0, stream>>>(z, ld, d, ld_d, parts, per_block, args);
    else token_log_probs_bwd_kernel<T, D, false><<<blocks, GRAD_THREADS, 0, stream>>>(z, ld, d, ld_d, parts, per_block, args);
  });
}

extern "C" int ob_distill_fwd(const void* logits, int dtype, long long ld, const void* teacher_ids, int ids_64,
                              const float* teacher_log_probs, long long ld_t, int k, int renormalize, float* row_loss,
                              float* row_stats, float* q, long long rows, int V, float softcap, double inv_temp,
                              cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("distillation", logits, dtype, ld, rows, V)) return rc;
  if (k < 1 || k > OB_TOP_K_MAX) OB_FAIL(-4, "distillation: %d teacher classes outside [1, %d]", k, OB_TOP_K_MAX);
  if (teacher_ids == nullptr || teacher_log_probs == nullptr || row_loss == nullptr || row_stats == nullptr || q == nullptr)
    OB_FAIL(-5, "distillation: missing tensor");
  const DistillArgs args{teacher_ids, teacher_log_probs, ids_64, k, renormalize, ld_t, row_loss, row_stats, q, V, inv_temp, scaling(softcap, inv_temp)};
  if (dtype == OB_F32)
    return softcap > 0.f ? launch_distill<float, 4, true>((const float*)logits, ld, rows, args, stream)
                         : launch_distill<float, 4, false>((const float*)logits, ld, rows, args, stream);
  return softcap > 0.f ? launch_distill<bf16, 2, true>((const bf16*)logits, ld, rows, args, stream)
                       : launch_distill<bf16, 2, false>((const bf16*)logits, ld, rows, args, stream);
}

extern "C" int ob_distill_bwd(const void* logits, int dtype, long long ld, const void* teacher_ids, int ids_64, long long ld_t,
                              int k, const float* row_stats, const float* q, const float* g, long long stride_g,
                              const float* inv_count, float scale, void* dlogits, int dtype_d, long long ld_d, long long rows,
                              int V, float softcap, double inv_temp, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("distillation backward", logits, dtype, ld, rows, V)) return rc;
  if (k < 1 || k > OB_TOP_K_MAX) OB_FAIL(-4, "distillation backward: %d teacher classes outside [1, %d]", k, OB_TOP_K_MAX);
  if (teacher_ids == nullptr || row_stats == nullptr || q == nullptr || dlogits == nullptr)
    OB_FAIL(-5, "distillation backward: missing tensor");
  const Scaling sc = scaling(softcap, inv_temp);
  const DistillGradArgs args{teacher_ids, ids_64, k, ld_t, row_stats, q, g, stride_g, inv_count, scale, V, sc};
  return launch_gradient("distillation backward", logits, dtype, ld, dlogits, dtype_d, ld_d, rows, V, stream,
                         [&](auto* z, auto* d, int parts, int per_block) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(z)>> T;
    typedef std::remove_pointer_t<decltype(d)> D;
    const unsigned blocks = (unsigned)(rows * parts);
    if (softcap > 0.f) distill_bwd_kernel<T, D, true><<<blocks, GRAD_THREADS, 0, stream>>>(z, ld, d, ld_d, parts, per_block, args);
    else distill_bwd_kernel<T, D, false><<<blocks, GRAD_THREADS, 0, stream>>>(z, ld, d, ld_d, parts, per_block, args);
  });
}

extern "C" int ob_distill_reduce(const float* row_loss, const float* row_stats, long long rows, int mean, float* loss,
                                 float* inv_count, cudaStream_t stream) {
  if (loss == nullptr || (rows > 0 && (row_loss == nullptr || row_stats == nullptr))) OB_FAIL(-5, "distillation sum: missing tensor");
  distill_reduce_kernel<<<1, 1024, 0, stream>>>(row_loss, row_stats, rows, mean, loss, inv_count);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int ob_distill_count(const void* teacher_ids, int ids_64, const float* teacher_log_probs, long long ld_t, int k,
                                int renormalize, long long rows, int V, float* inv_count, cudaStream_t stream) {
  if (inv_count == nullptr || (rows > 0 && (teacher_ids == nullptr || teacher_log_probs == nullptr)))
    OB_FAIL(-5, "distillation count: missing tensor");
  distill_count_kernel<<<1, 1024, 0, stream>>>(teacher_ids, ids_64, teacher_log_probs, ld_t, k, renormalize, rows, V, inv_count);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}
