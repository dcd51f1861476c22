// k3_objf.hip -- objectives and scores taken from the rows of a network's output: the log-probability of a given label with the row's entropy and best alternatives
// (k3_label_logprobs), its derivative (k3_label_logprobs_deriv), and distillation from a teacher's top logits with its derivative (k3_distill_objf_and_deriv).
// With a = log2(e) / temperature, M = max z, d_j = a (z_j - M), e_j = 2^d_j, s = sum e_j:  log q_j = ln 2 d_j - ln s,  q_j = e_j / s,  entropy = ln s - ln 2 sum e_j d_j / s
//   distillation, p = softmax of a row's teacher values:  objf = w T^2 sum_k p_k (log q_{i_k} - log p_k),  d objf / d z_j = w T (sum of p_k over i_k = j  -  q_j)
// Elements are held as they are stored and widened where they are used; statistics, sums and exponentials are float32.  The difference is taken before the product: a z_j alone would
// overflow at the lowest values of float32 and bfloat16, which masks are made of.
// Bound by memory, a row being read once (and its derivative written once): scores of float32 42752 x 6024 with 4 alternatives 165 us (6.2 TB/s), label derivative of bfloat16 2000 x 50001
// 78 us (5.1), distillation with derivative of float32 6400 x 6024 66 us (4.6) and of bfloat16 4096 x 128000 509 us (4.1: a row fills a compute unit's registers, and its
// vector instructions, 55 % of its cycles by counters, run under its own loads and stores only in part).
#include "k3_rowops.h"
#include <algorithm>
#include <type_traits>

namespace {
using namespace k3;

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff(), kMaxFloat = 3.402823466e38f;
constexpr int kMaxTop = 64;              // alternatives per row: one per lane of a wavefront
constexpr int kMaxTeacher = 1024;        // teacher entries per row: their probabilities lie in LDS
constexpr int kMaxSplits = 64;           // parts of a row: one per lane of the wavefront that joins them
constexpr int kCandidates = 512;         // places for the elements that may be among the best

struct Partial { float max, sum, weighted, unused; };      // of one part of a row: M, s, sum e_j d_j

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32: 1 ulp, results below 2^-126 are 0

// ---- order of (value, column): larger values first, equal ones by column
__device__ inline unsigned order_key(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v + 0.0f);      // -0 counts as 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ inline float key_value(unsigned k) { return __builtin_bit_cast(float, (k >> 31) ? k ^ 0x80000000u : ~k); }
__device__ inline unsigned long long pair_key(float v, int col) { return ((unsigned long long)order_key(v) << 32) | (unsigned)~col; }
constexpr unsigned kLowest = 0x007fffffu;      // order_key(-inf)

// the largest t found by descending its bits, from the first one in which the keys differ, such that at least k of 64 NW keys (NW of them in each lane of a wavefront) are >= t; stops as soon
// as exactly k are
template <int NW> __device__ inline unsigned kth_key(const unsigned (&key)[NW], int k) {
  float most = key_value(key[0]), least = most;
#pragma unroll
  for (int w = 1; w < NW; w++) { most = fmaxf(most, key_value(key[w])); least = fminf(least, key_value(key[w])); }
  const unsigned high = order_key(wave_max(most)), differ = high ^ order_key(-wave_max(-least));
  if (differ == 0) return high;
  const int top = 31 - __builtin_clz(differ);
  unsigned t = (high >> top >> 1) << top << 1;      // (the bits that all keys share)
  for (int bit = top; bit >= 0; bit--) {
    const unsigned u = t | (1u << bit);
    int n = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) n += __popcll(__ballot(key[w] >= u));
    if (n >= k) { t = u; if (n == k) break; }
  }
  return max(t, kLowest);
}
__device__ inline unsigned long long wave_max_u64(unsigned long long v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const unsigned hi = __shfl_xor((unsigned)(v >> 32), m), lo = __shfl_xor((unsigned)v, m);
    const unsigned long long o = ((unsigned long long)hi << 32) | lo;
    v = o > v ? o : v;
  }
  return v;
}

template <int NW> __device__ inline void row_barrier() {
  if constexpr (NW > 1) __syncthreads();
  else { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }
}

template <int NW> struct TopShared { unsigned long long cand[kCandidates + 8]; unsigned long long best[NW]; unsigned key[NW > 1 ? 64 * NW : 1], tau; int count; };

// The `top` largest of the E * N <= 64 (value, column) pairs of each of 64 NW threads, handed to emit(rank, value, column) with ranks 0 .. top - 1 (value -inf and column -1 where NaNs
// or a short row leave fewer).  value(i, j): the value a thread holds; pick(e): the same for e = i N + j; fetch(e, v, c): the same read from memory again, with its column (-1: none);
// column(e): its column alone; lane_max: the thread's largest value (-inf: none).
// Every lane's largest element bounds what can be among the best: with t = the top-th largest of the lanes' maxima, `top` elements are >= t, so only elements >= t (as a rule a few more
// than `top`) are gathered and ranked by counting.  Where more than fit are >= t (many equal values), the best are taken one after another instead,
// each with a read of the row (float32 42752 x 6024 of one value, 4 alternatives: 1215 us where random ones take 192).
template <int NW, int E, int N, typename V, typename P, typename C, typename G, typename F>
__device__ inline void emit_top(V value, P pick, C column, G fetch, float lane_max, int top, TopShared<NW> &sh, F emit) {
  constexpr int TPR = 64 * NW;
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  unsigned tau;
  if (t == 0) sh.count = 0;
  if constexpr (NW > 1) {      // (one wavefront looks for t; its bits are not worth the others' time)
    sh.key[t] = order_key(lane_max);
    __syncthreads();
    if (t < 64) {
      unsigned keys[NW];
#pragma unroll
      for (int w = 0; w < NW; w++) keys[w] = sh.key[w * 64 + t];
      tau = kth_key<NW>(keys, top);
      if (t == 0) sh.tau = tau;
    }
    __syncthreads();
    tau = sh.tau;
  } else {
    const unsigned keys[1] = {order_key(lane_max)};
    row_barrier<NW>();
    tau = kth_key<1>(keys, top);
  }
  const float bound = key_value(tau);
  unsigned long long mine = 0;      // which of the thread's elements are >= t
  if (lane_max >= bound)
#pragma unroll
    for (int i = 0; i < E; i++)
#pragma unroll
      for (int j = 0; j < N; j++) mine |= value(i, j) >= bound ? 1ull << (i * N + j) : 0;
  while (mine) {
    const int e = __builtin_ctzll(mine);
    mine &= mine - 1;
    const int c = column(e);
    if (c < 0) continue;
    const int slot = atomicAdd(&sh.count, 1);
    if (slot < kCandidates) sh.cand[slot] = pair_key(pick(e), c);
  }
  row_barrier<NW>();
  const int count = sh.count;
  if (count <= kCandidates) {
    for (int c = t; c < count; c += TPR) {
      const unsigned long long mine = sh.cand[c];
      int rank = 0;
      for (int o = 0; o < count; o += 8)      // (8 reads on their way together; what lies behind the last candidate does not count)
#pragma unroll
        for (int k = 0; k < 8; k++) rank += sh.cand[o + k] > mine && o + k < count ? 1 : 0;
      if (rank < top) emit(rank, key_value((unsigned)(mine >> 32)), (int)~(unsigned)mine);
    }
    for (int r = count + t; r < top; r += TPR) emit(r, -kInf, -1);
    return;
  }
  unsigned long long last = ~0ull;
  for (int r = 0; r < top; r++) {
    unsigned long long best = 0;
#pragma unroll 1
    for (int e = 0; e < E * N; e++) {
      float v;
      int c;
      fetch(e, v, c);
      const unsigned long long k = c >= 0 && v == v ? pair_key(v, c) : 0;
      if (k < last && k > best) best = k;
    }
    best = wave_max_u64(best);
    if constexpr (NW > 1) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) sh.best[threadIdx.x >> 6] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; w++) best = sh.best[w] > best ? sh.best[w] : best;
    }
    if (t == 0) { if (best) emit(r, key_value((unsigned)(best >> 32)), (int)~(unsigned)best); else emit(r, -kInf, -1); }
    last = best;
  }
}

struct ScoreArgs {
  const void *z; long long ld; int rows, cols;
  const int *labels;
  float a;                                             // log2(e) / temperature
  float *log_prob, *entropy, *stats, *alt_log_probs; int *alt_labels; int top;
  int splits, span;                                    // parts per row, columns per part
  Partial *partial; float *part_value; int *part_col;  // [rows][splits], [rows][splits][top]; partial null: one part per row, and the scores are written at once
};

// of one row, by one thread: its label's value (if it has a label) and its scores
__device__ inline bool label_of(const ScoreArgs &p, long long row, int &y) {
  y = p.labels ? p.labels[row] : -1;
  return y >= 0 && y < p.cols;
}
__device__ inline void write_scores(const ScoreArgs &p, long long row, float m, float s, float u, bool has_label, float label_value) {
  const float log_sum = logf(s);
  if (p.log_prob) p.log_prob[row] = !has_label ? 0.0f : m == -kInf && s == s ? -kInf : label_value - m - log_sum;
  if (p.entropy) p.entropy[row] = m == -kInf ? s : log_sum - kLn2 * (u / s);      // (of a row without any value: 0, which s is then; NaN where NaNs are all it has)
  if (p.stats) { p.stats[2 * row] = s == s ? m : s; p.stats[2 * row + 1] = m == -kInf ? s : log_sum; }
}
__device__ inline void write_alternative(const ScoreArgs &p, long long row, int rank, float value, int col, float m, float s, float log_sum) {
  const bool fine = s == s;
  if (p.alt_log_probs) p.alt_log_probs[row * p.top + rank] = !fine ? s : m == -kInf ? -kInf : value - m - log_sum;
  if (p.alt_labels) p.alt_labels[row * p.top + rank] = fine ? col : -1;
}

// Columns [begin, end) of a row in the registers of NW wavefronts: chunk t + 64 NW i of them is lane t's i-th.  Which of a lane's chunks are whole is the same for all lanes but for one chunk
// (number `whole`, the row's end lies in it), so whole chunks are loaded and stored without a branch of the lanes, from one base address.
template <typename T, int NW, int E> struct Part {
  static constexpr int N = Chunk<T>::N, SPAN = 64 * NW * N;      // columns of one chunk of every lane
  int begin, end, whole, t;
  __device__ inline Part(int begin, int end) : begin(begin), end(end), whole((end - begin) / SPAN), t(NW == 1 ? threadIdx.x & 63 : threadIdx.x) {}
  __device__ inline int column(int e) const { return begin + e / N * SPAN + t * N + e % N; }
  // -inf behind `end`
  __device__ inline void load(const T *row, Packed (&v)[E]) const {
    const Packed tail = load_packed<T>(row, begin + whole * SPAN + t * N, end - begin - whole * SPAN - t * N, (T)-kInf);
    const int fill = sizeof(T) == 4 ? (int)0xff800000 : std::is_same<T, bf16>::value ? (int)0xff80ff80 : (int)0xfc00fc00;
#pragma unroll
    for (int i = 0; i < E; i++) {
      if (i < whole) v[i] = __builtin_bit_cast(Packed, *reinterpret_cast<const typename Chunk<T>::type *>(row + begin + i * SPAN + (unsigned)(t * N)));
      else v[i] = i == whole ? tail : Packed{fill, fill, fill, fill};
    }
  }
  // value(packed chunk, j) rounded to the row's type
  template <typename F> __device__ inline void store(T *row, const Packed (&v)[E], F value) const {
    Packed last = v[0];
#pragma unroll
    for (int i = 0; i < E; i++) {
      if (i < whole) {
        typename Chunk<T>::type o;
#pragma unroll
        for (int j = 0; j < N; j++) o[j] = (T)value(v[i], i * N + j, j);
        *reinterpret_cast<typename Chunk<T>::type *>(row + begin + i * SPAN + (unsigned)(t * N)) = o;
      } else if (i == whole) last = v[i];
    }
    const int col = begin + whole * SPAN + t * N;
    if (col >= end) return;
    Packed one[1] = {last};
    keep_packed<T, 1>(one);
    last = one[0];
    typename Chunk<T>::type o;
#pragma unroll
    for (int j = 0; j < N; j++) o[j] = (T)value(last, whole * N + j, j);
    store_chunk(row, col, end - col, o);
  }
};
template <typename T, int E> __device__ inline float largest(const Packed (&v)[E]) {
  float m = -kInf;
#pragma unroll
  for (int i = 0; i < E; i++)
#pragma unroll
    for (int j = 0; j < Chunk<T>::N; j++) m = fmaxf(m, element<T>(v[i], j));
  return m;
}
// s of a row part whose largest value is -inf: 0, or NaN where there are NaNs beside it
template <typename T, int NW, int E> __device__ inline float empty_sum(const Packed (&v)[E], float *sh) {
  float bad = 0.0f;
#pragma unroll
  for (int i = 0; i < E; i++)
#pragma unroll
    for (int j = 0; j < Chunk<T>::N; j++) bad = element<T>(v[i], j) == element<T>(v[i], j) ? bad : 1.0f;
  return block_max<NW>(bad, sh) > 0.0f ? __builtin_nanf("") : 0.0f;
}

// One part of a row (with one part: the row) per NW wavefronts, in registers: it is read once.
template <typename T, int NW, int E> __global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k3_row_scores_kernel(ScoreArgs p) {
  constexpr int N = Chunk<T>::N, RPB = NW == 1 ? 4 : 1;
  __shared__ float sh[4 * NW];
  __shared__ TopShared<NW> top_sh[RPB];
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x, sub = NW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const long long item = block_number() * RPB + sub;
  if (item >= (long long)p.rows * p.splits) return;      // (NW = 1: a whole wavefront, and no barrier spans wavefronts)
  const long long row = item / p.splits;
  const int part = (int)(item - row * p.splits), begin = part * p.span, end = min(p.cols, begin + p.span);
  const T *z = (const T *)p.z + row * p.ld;
  int y;
  const bool has_label = !p.partial && label_of(p, row, y);
  const float label_value = has_label ? to_f32(z[y]) : 0.0f;
  Packed v[E];
  const Part<T, NW, E> columns(begin, end);
  columns.load(z, v);
  const float lane_max = largest<T, E>(v), m = block_max<NW>(lane_max, sh);
  keep_packed<T, E>(v);
  float s = 0.0f, u = 0.0f;
#pragma unroll
  for (int i = 0; i < E; i++)
#pragma unroll
    for (int j = 0; j < N; j++) {
      const float d = (element<T>(v[i], j) - m) * p.a, e = exp2_fast(d);
      s += e;
      u += e * fmaxf(d, -16384.0f);      // (e = 0 where d = -inf: the product is to be 0)
    }
  block_sum2<NW>(s, u, sh + NW);
  keep_packed<T, E>(v);
  if (m == -kInf) s = u = empty_sum<T, NW, E>(v, sh + 3 * NW);
  const auto value = [&](int i, int j) { return element<T>(v[i], j); };
  const auto column = [&](int e) { const int c = columns.column(e); return c < end ? c : -1; };
  const auto pick = [&](int e) {      // (a chain of selections: the elements' registers have no index)
    const int word = sizeof(T) == 4 ? e : e / 2;
    int w = v[0][0];
#pragma unroll
    for (int k = 1; k < E * 4; k++) w = word == k ? v[k / 4][k % 4] : w;
    return element<T>(Packed{w, w, w, w}, e & 1);
  };
  const auto fetch = [&](int e, float &f, int &c) {
    c = column(e);
    f = c >= 0 ? to_f32(z[c]) : -kInf;
  };
  if (t == 0) {
    if (p.partial) p.partial[item] = Partial{m, s, u, 0.0f};
    else write_scores(p, row, m, s, u, has_label, label_value);
  }
  if (p.top) {
    const float log_sum = logf(s);
    emit_top<NW, E, N>(value, pick, column, fetch, lane_max, p.top, top_sh[sub], [&](int rank, float value, int c) {
      if (p.partial) {
        p.part_value[item * p.top + rank] = value;
        p.part_col[item * p.top + rank] = c;
      } else write_alternative(p, row, rank, value, c, m, s, log_sum);
    });
  }
}

// the sums of a row from those of its parts (splits <= 64), the same in every lane of a wavefront
__device__ inline void join_parts(const Partial *part, int splits, float a, float &m, float &s, float &u) {
  const int lane = threadIdx.x & 63;
  Partial q = {-kInf, 0.0f, 0.0f, 0.0f};
  if (lane < splits) q = part[lane];
  m = wave_max(q.max);
  // (a part without values has s = u = 0, or NaN.  One of nothing but the type's lowest value is so far below the row's largest that d overflows: at -16384 its f is 0 all the same, and f d too)
  const float d = q.max == -kInf ? 0.0f : fmaxf((q.max - m) * a, -16384.0f), f = exp2_fast(d);
  s = wave_sum(q.sum * f);
  u = wave_sum(q.weighted * f + q.sum * f * d);
}

// scores of a row from its parts: one workgroup per row.  A part's best elements come in their order, `top` of them; at most 64 x 64 in all, 16 per thread
template <typename T> __global__ __launch_bounds__(256) void k3_row_scores_join_kernel(ScoreArgs p) {
  constexpr int E = kMaxSplits * kMaxTop / 256;
  __shared__ TopShared<4> top_sh;
  const long long row = block_number();
  if (row >= p.rows) return;
  int y;
  const bool has_label = label_of(p, row, y);
  const float label_value = has_label ? to_f32(((const T *)p.z)[row * p.ld + y]) : 0.0f;
  float v[E], lane_max = -kInf;
  const long long first = row * p.splits * p.top;
  const int n = p.splits * p.top;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int k = threadIdx.x + i * 256;
    v[i] = k < n ? p.part_value[first + k] : -kInf;
    lane_max = fmaxf(lane_max, v[i]);
  }
  float m, s, u;
  join_parts(p.partial + row * p.splits, p.splits, p.a, m, s, u);
  if (threadIdx.x == 0) write_scores(p, row, m, s, u, has_label, label_value);
  if (p.top) {
    const float log_sum = logf(s);
    const auto column = [&](int e) { const int k = threadIdx.x + e * 256; return k < n ? p.part_col[first + k] : -1; };
    const auto pick = [&](int e) { const int k = threadIdx.x + e * 256; return k < n ? p.part_value[first + k] : -kInf; };
    const auto fetch = [&](int e, float &f, int &c) {
      f = pick(e);
      c = column(e);
    };
    emit_top<4, E, 1>([&](int i, int) { return v[i]; }, pick, column, fetch, lane_max, p.top, top_sh,
                      [&](int rank, float value, int c) { write_alternative(p, row, rank, value, c, m, s, log_sum); });
  }
}

// d (g log q_y + h H) / d z_j = g [j = y] - q_j (g + h (log q_j + H)), one read and one write of every element: a wavefront takes 4 chunks per lane of a row
template <typename T> __global__ __launch_bounds__(256) void k3_label_deriv_kernel(const T *z, long long ld, const int *labels, const float *stats, const float *entropy,
    const float *log_prob_deriv, const float *entropy_deriv, T *dz, long long ldd, int cols, int segments, long long items) {
  constexpr int N = Chunk<T>::N, E = 4;
  const long long item = block_number() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= items) return;
  const long long row = item / segments;
  const int begin = (int)(item - row * segments) * (64 * E * N), end = min(cols, begin + 64 * E * N);
  const Part<T, 1, E> columns(begin, end);
  Packed v[E];
  columns.load(z + row * ld, v);
  const float m = stats[2 * row], log_sum = stats[2 * row + 1], h = entropy_deriv ? entropy_deriv[row] : 0.0f;
  int y = labels ? labels[row] : -1;
  if (y < 0 || y >= cols) y = -1;
  const float g = y >= 0 && log_prob_deriv ? log_prob_deriv[row] : 0.0f, b = -h, c = -g - (h != 0.0f ? h * entropy[row] : 0.0f);
  const bool empty = m == -kInf || (g == 0.0f && h == 0.0f);      // (nothing to pass on: zeros, whatever the row holds)
  columns.store(dz + row * ldd, v, [&](Packed w, int e, int j) {
    const float lq = element<T>(w, j) - m - log_sum, q = exp2_fast(lq * kLog2e), d = q * __builtin_fmaf(b, fmaxf(lq, -16384.0f), c);      // (q = 0 where lq = -inf)
    return empty ? 0.0f : columns.column(e) == y ? d + g : d;
  });
}

struct DistillArgs {
  const void *z; long long ld; int rows, cols;
  const void *values; long long ld_values; const int *indexes; long long ld_indexes; int top;
  const float *weights;
  float temperature, a;
  float *objf; void *dz; long long ldd;
  int splits; const Partial *partial; float4 *coef; float *prob;      // of the rows that are too wide for one workgroup
};
// a row's teacher entries in LDS: column (-1: not used), the teacher's e and value below its largest, and the student's value there
struct Entry { int col; float e, d, z; };
struct Teacher { float sum; bool live; };      // sum of the e; whether the row counts (an entry that is not -inf, and a weight that is not 0)

// the first step reads the entries, the second has their softmax and the student's values; `sh` holds 3 NW floats
template <typename T> __device__ inline float read_teacher(const DistillArgs &p, long long row, Entry *entry, int t, int threads) {
  float m = -kInf;
  for (int k = t; k < p.top; k += threads) {
    const int c = p.indexes[row * p.ld_indexes + k];
    const bool used = c >= 0 && c < p.cols;
    const float v = used ? to_f32(((const T *)p.values)[row * p.ld_values + k]) : -kInf;
    entry[k].col = used ? c : -1;
    entry[k].d = v;
    m = fmaxf(m, v == v ? v : 0.0f);      // (a NaN makes the row count, and shows in the sum)
  }
  return m;
}
template <typename T, int NW> __device__ inline Teacher teacher_softmax(const DistillArgs &p, long long row, Entry *entry, float lane_max, int t, float *sh) {
  const float m = block_max<NW>(lane_max, sh);
  float s = 0.0f;
  for (int k = t; k < p.top; k += 64 * NW) {
    const int c = entry[k].col;
    const float v = entry[k].d, d = v == -kInf ? -kInf : v - m, e = exp2_fast(d * p.a);
    entry[k].z = c >= 0 ? to_f32(((const T *)p.z)[row * p.ld + c]) : 0.0f;
    entry[k].d = d;
    entry[k].e = e;
    s += e;
  }
  return Teacher{block_sum<NW>(s, sh + NW), m != -kInf && !(p.weights && p.weights[row] == 0.0f)};
}
// sum_k e_k ((z_k - M) - (v_k - max v)) / 4096, in every thread.  The differences stay in the logits' units, and 1024 of them are added up well within float32's range: in the units of the
// exponentials, or as they are, those that have a lowest value in them would overflow, which the objective does not
constexpr float kShrink = 1.0f / (4 * kMaxTeacher);
template <int NW> __device__ inline float teacher_differences(const DistillArgs &p, const Entry *entry, float m, int t, float *sh) {
  float f = 0.0f;
  for (int k = t; k < p.top; k += 64 * NW)
    if (!(entry[k].e == 0.0f)) f += entry[k].e * (kShrink * (entry[k].z - m - entry[k].d));
  return block_sum<NW>(f, sh);
}
// w T^2 sum_k p_k (log q_k - log p_k) from them and the student's M and s, with wt = w T; by one thread
__device__ inline float teacher_objf(const DistillArgs &p, Teacher w, float wt, float m, float s, float f) {
  if (!w.live) return 0.0f;
  return m == -kInf && s == s ? wt * -kInf : wt / kShrink * (f / w.sum + kShrink * p.temperature * kLn2 * (log2f(w.sum) - log2f(s)));
}

// One row per NW wavefronts, held in registers from the sums to the derivative: read once, written once.  The teacher's columns are corrected behind the row's own store (by the same
// workgroup, after a barrier).
template <typename T, int NW, int E> __global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW, NW >= 8 ? 4 : 1) void k3_distill_kernel(DistillArgs p) {
  constexpr int N = Chunk<T>::N, RPB = NW == 1 ? 4 : 1;
  __shared__ float sh[6 * NW];
  extern __shared__ Entry entries[];
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x, sub = NW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const long long row = block_number() * RPB + sub;
  if (row >= p.rows) return;      // (NW = 1: a whole wavefront, and no barrier spans wavefronts)
  Entry *entry = entries + sub * p.top;
  const float teacher_max = read_teacher<T>(p, row, entry, t, 64 * NW);
  Packed v[E];
  const Part<T, NW, E> columns(0, p.cols);
  columns.load((const T *)p.z + row * p.ld, v);
  // each lane's sum against its own largest value so far, so that chunks are worked on while later ones are still on their way
  float lm = -kMaxFloat, s = 0.0f;
#pragma unroll
  for (int i = 0; i < E; i++) {
    float c = element<T>(v[i], 0);
#pragma unroll
    for (int j = 1; j < N; j++) c = fmaxf(c, element<T>(v[i], j));
    c = fmaxf(c, lm);
    s *= exp2_fast((lm - c) * p.a);
    lm = c;
#pragma unroll
    for (int j = 0; j < N; j++) s += exp2_fast((element<T>(v[i], j) - c) * p.a);
  }
  const Teacher teacher = teacher_softmax<T, NW>(p, row, entry, teacher_max, t, sh);
  float m = block_max<NW>(lm, sh + 2 * NW);
  s = block_sum<NW>(s * exp2_fast((lm - m) * p.a), sh + 3 * NW);
  const bool empty = s == 0.0f;      // (the row's largest value adds 1: nothing but -inf)
  if (empty) m = -kInf;
  const float w = (p.weights ? p.weights[row] : 1.0f) * p.temperature;
  const float f = teacher_differences<NW>(p, entry, m, t, sh + 4 * NW);
  if (t == 0) p.objf[row] = teacher_objf(p, teacher, w, m, s, f);
  if (!p.dz) return;
  T *dz = (T *)p.dz + row * p.ldd;
  if (!teacher.live || empty) {
    for (int c = t; c < p.cols; c += 64 * NW) dz[c] = (T)0.0f;
    return;
  }
  keep_packed<T, E>(v);
  const float g = -w / s;
  columns.store(dz, v, [&](Packed w, int, int j) { return g * exp2_fast((element<T>(w, j) - m) * p.a); });
  row_barrier<NW>();
  for (int k = t; k < p.top; k += 64 * NW) {
    const int c = entry[k].col;
    if (c < 0) continue;
    float e = 0.0f;
    for (int o = 0; o < p.top; o++) e += entry[o].col == c ? entry[o].e : 0.0f;      // an index that comes twice: both write the same sum
    dz[c] = (T)(w * (e / teacher.sum - exp2_fast((entry[k].z - m) * p.a) / s));
  }
}

// rows in parts: the objective, and what the derivative needs of a row: coef = {M, -w T / s, w T, whether it is not zero}, prob = its teacher's probabilities
template <typename T> __global__ __launch_bounds__(64) void k3_distill_join_kernel(DistillArgs p) {
  extern __shared__ Entry entries[];
  const long long row = block_number();
  if (row >= p.rows) return;
  const int t = threadIdx.x;
  const float teacher_max = read_teacher<T>(p, row, entries, t, 64);
  const Teacher teacher = teacher_softmax<T, 1>(p, row, entries, teacher_max, t, nullptr);
  float m, s, u;
  join_parts(p.partial + row * p.splits, p.splits, p.a, m, s, u);
  const float w = (p.weights ? p.weights[row] : 1.0f) * p.temperature, f = teacher_differences<1>(p, entries, m, t, nullptr);
  if (t == 0) {
    p.objf[row] = teacher_objf(p, teacher, w, m, s, f);
    if (p.dz) p.coef[row] = make_float4(m, -w / s, w, teacher.live && !(m == -kInf && s == s) ? 1.0f : 0.0f);
  }
  if (p.dz)
    for (int k = t; k < p.top; k += 64) p.prob[row * p.top + k] = entries[k].e / teacher.sum;
}
template <typename T> __global__ __launch_bounds__(256) void k3_distill_deriv_kernel(DistillArgs p, int segments) {
  constexpr int N = Chunk<T>::N, E = 4, SEG = 256 * E * N;
  const long long row = block_number() / segments;
  if (row >= p.rows) return;
  const int begin = (int)(block_number() - row * segments) * SEG, end = min(p.cols, begin + SEG), t = threadIdx.x;
  const T *z = (const T *)p.z + row * p.ld;
  T *dz = (T *)p.dz + row * p.ldd;
  const int *index = p.indexes + row * p.ld_indexes;
  const float *prob = p.prob + row * p.top;
  Packed v[E];
  const Part<T, 4, E> columns(begin, end);
  columns.load(z, v);
  const float4 c = p.coef[row];
  constexpr int K = kMaxTeacher / 256;
  float zk[K];      // read before anything of this part is written: dz may be z
#pragma unroll
  for (int i = 0; i < K; i++) {
    const int k = t + i * 256, j = k < p.top ? index[k] : -1;
    zk[i] = j >= begin && j < end ? to_f32(z[j]) : 0.0f;
  }
  __syncthreads();
  columns.store(dz, v, [&](Packed w, int, int j) { return c.w == 0.0f ? 0.0f : c.y * exp2_fast((element<T>(w, j) - c.x) * p.a); });
  if (c.w == 0.0f) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < K; i++) {
    const int k = t + i * 256, j = k < p.top ? index[k] : -1;
    if (j < begin || j >= end) continue;
    float q = 0.0f;
    for (int o = 0; o < p.top; o++) q += index[o] == j ? prob[o] : 0.0f;
    dz[j] = (T)(c.z * q + c.y * exp2_fast((zk[i] - c.x) * p.a));
  }
}

// ---- shapes

// wavefronts and chunks per thread that hold `cols` columns: one wavefront up to 8 chunks per lane, then 4 up to 8, 8 up to 16 (two such workgroups, with 64 of their 128 registers full of
// row, fill a compute unit) and 16 up to 16; e = 0: too wide
struct Shape { int nw, e; };
template <typename T> Shape shape_of(int cols, int least_waves, int most_waves) {
  const int chunks = (cols + Chunk<T>::N - 1) / Chunk<T>::N;
  for (const Shape hold : {Shape{1, 8}, Shape{4, 8}, Shape{8, 16}, Shape{16, 16}}) {
    const int e = (chunks + 64 * hold.nw - 1) / (64 * hold.nw);
    if (hold.nw >= least_waves && hold.nw <= most_waves && e <= hold.e) return {hold.nw, e <= 4 ? e : e <= 6 ? 6 : e <= 8 ? 8 : e <= 12 ? 12 : 16};
  }
  return {0, 0};
}
// f(NW, E) as integral constants
template <int NW, typename F> void with_chunks(int e, F f) {
#define K3_E(v) case v: f(std::integral_constant<int, NW>(), std::integral_constant<int, v>()); return
  if constexpr (NW <= 4) {
    switch (e) { K3_E(1); K3_E(2); K3_E(3); K3_E(4); K3_E(6); K3_E(8); default: return; }
  } else if constexpr (NW == 8) {
    switch (e) { K3_E(6); K3_E(8); K3_E(12); K3_E(16); default: return; }
  } else {
    switch (e) { K3_E(12); K3_E(16); default: return; }
  }
#undef K3_E
}

// the parts of a row: one where a workgroup of four wavefronts holds the row and the rows alone fill the chip; parts of 2048 columns at least where there are few rows
template <typename T> void split_rows(int rows, int cols, int &splits, int &span) {
  const int hold = 4 * 64 * 8 * Chunk<T>::N;
  int n = (cols + hold - 1) / hold;
  if ((long long)rows * n < 512) n = std::max(n, std::min({(512 + rows - 1) / rows, (cols + 2047) / 2048, kMaxSplits}));
  span = ((cols + n - 1) / n + 63) / 64 * 64;
  splits = (cols + span - 1) / span;
}
template <typename T> int launch_scores(ScoreArgs p, hipStream_t st) {
  const Shape s = shape_of<T>(std::min(p.cols, p.span), 1, 4);
  const long long items = (long long)p.rows * p.splits, blocks = s.nw == 1 ? (items + 3) / 4 : items;
  K3_REQUIRE(s.e && blocks <= kMostGroups, "k3_objf: matrix too large");
  const auto launch = [&](auto nw, auto e) {
    constexpr int NW = decltype(nw)::value, E = decltype(e)::value;
    hipLaunchKernelGGL((k3_row_scores_kernel<T, NW, E>), grid_of(blocks, 256), dim3(NW == 1 ? 256 : 64 * NW), 0, st, p);
  };
  if (s.nw == 1) with_chunks<1>(s.e, launch);
  else with_chunks<4>(s.e, launch);
  K3_HIP_CHECK(hipGetLastError());
  return K3_OK;
}
constexpr int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
template <typename T> int64_t scores_workspace(int rows, int cols, int top) {
  int splits, span;
  split_rows<T>(rows, cols, splits, span);
  return splits == 1 ? 0 : up16((int64_t)rows * splits * sizeof(Partial)) + 2 * up16((int64_t)rows * splits * top * 4);
}
template <typename T> int label_logprobs(ScoreArgs p, void *workspace, hipStream_t st) {
  split_rows<T>(p.rows, p.cols, p.splits, p.span);
  if (p.splits == 1) return launch_scores<T>(p, st);
  char *w = (char *)workspace;
  p.partial = (Partial *)w;
  w += up16((int64_t)p.rows * p.splits * sizeof(Partial));
  p.part_value = (float *)w;
  w += up16((int64_t)p.rows * p.splits * p.top * 4);
  p.part_col = (int *)w;
  const int rc = launch_scores<T>(p, st);
  if (rc) return rc;
  hipLaunchKernelGGL((k3_row_scores_join_kernel<T>), grid_of(p.rows, 256), dim3(256), 0, st, p);
  K3_HIP_CHECK(hipGetLastError());
  return K3_OK;
}

// whether a distillation row goes through one workgroup: up to 4 wavefronts without a derivative (wider rows are read by several workgroups), up to 16 with it
template <typename T> Shape distill_shape(int cols, int top, bool deriv) { return shape_of<T>(cols, top > 256 ? 4 : 1, deriv ? 16 : 4); }
template <typename T> int64_t distill_workspace(int rows, int cols, int top, bool deriv) {
  if (distill_shape<T>(cols, top, deriv).e) return 0;
  int splits, span;
  split_rows<T>(rows, cols, splits, span);
  return up16((int64_t)rows * splits * sizeof(Partial)) + (deriv ? (int64_t)rows * 16 + up16((int64_t)rows * top * 4) : 0);
}
template <typename T> int distill(DistillArgs p, void *workspace, hipStream_t st) {
  const Shape s = distill_shape<T>(p.cols, p.top, p.dz != nullptr);
  if (s.e) {
    const auto launch = [&](auto nw, auto e) {
      constexpr int NW = decltype(nw)::value, E = decltype(e)::value, RPB = NW == 1 ? 4 : 1;
      hipLaunchKernelGGL((k3_distill_kernel<T, NW, E>), grid_of((p.rows - 1) / RPB + 1, NW == 1 ? 256 : 64 * NW), dim3(NW == 1 ? 256 : 64 * NW), sizeof(Entry) * RPB * p.top, st, p);
    };
    if (s.nw == 1) with_chunks<1>(s.e, launch);
    else if (s.nw == 4) with_chunks<4>(s.e, launch);
    else if (s.nw == 8) with_chunks<8>(s.e, launch);
    else with_chunks<16>(s.e, launch);
    K3_HIP_CHECK(hipGetLastError());
    return K3_OK;
  }
  ScoreArgs sc{};
  sc.z = p.z; sc.ld = p.ld; sc.rows = p.rows; sc.cols = p.cols; sc.a = p.a;
  split_rows<T>(p.rows, p.cols, sc.splits, sc.span);
  char *w = (char *)workspace;
  sc.partial = (Partial *)w;
  p.partial = sc.partial;
  p.splits = sc.splits;
  w += up16((int64_t)p.rows * sc.splits * sizeof(Partial));
  p.coef = (float4 *)w;
  p.prob = (float *)(w + (int64_t)p.rows * 16);
  const int segments = (p.cols + 256 * 4 * Chunk<T>::N - 1) / (256 * 4 * Chunk<T>::N);
  K3_REQUIRE((long long)p.rows * segments <= kMostGroups, "k3_distill_objf_and_deriv: matrix too large");
  const int rc = launch_scores<T>(sc, st);
  if (rc) return rc;
  hipLaunchKernelGGL((k3_distill_join_kernel<T>), grid_of(p.rows, 64), dim3(64), sizeof(Entry) * p.top, st, p);
  K3_HIP_CHECK(hipGetLastError());
  if (p.dz) {
    hipLaunchKernelGGL((k3_distill_deriv_kernel<T>), grid_of((long long)p.rows * segments, 256), dim3(256), 0, st, p, segments);
    K3_HIP_CHECK(hipGetLastError());
  }
  return K3_OK;
}

const int kMaxCols = kMaxSplits * 4 * 64 * 8 * 4;      // 64 parts of what a workgroup of four wavefronts holds of float32 columns: 2^19
const int kMaxDerivCols = 0x7fffffff - 4095;                // column numbers of k3_label_deriv_kernel's threads that run ahead of a row's end still fit 32 bits

}  // namespace

extern "C" int64_t k3_label_logprobs_workspace(int32_t dtype, int32_t rows, int32_t cols, int32_t num_alternatives) {
  if (!dtype_ok(dtype) || rows <= 0 || cols <= 0 || num_alternatives < 0) return 0;
  return dtype == K3_F32 ? scores_workspace<float>(rows, cols, num_alternatives) : scores_workspace<f16>(rows, cols, num_alternatives);
}

extern "C" int k3_label_logprobs(int32_t dtype, const void *d_z, int64_t ld, const int32_t *d_labels, float *d_log_prob, float *d_entropy, float *d_stats, int32_t num_alternatives,
                                 float *d_alt_log_probs, int32_t *d_alt_labels, void *d_workspace, int64_t workspace_bytes, int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_label_logprobs: unknown type");
  K3_REQUIRE(rows >= 0 && cols >= 1 && ld >= cols && num_alternatives >= 0, "k3_label_logprobs: bad argument");
  if (cols > kMaxCols || num_alternatives > kMaxTop) { set_error("k3_label_logprobs: at most %d columns and %d alternatives", kMaxCols, kMaxTop); return K3_ERR_UNSUPPORTED; }
  K3_REQUIRE(num_alternatives <= cols, "k3_label_logprobs: more alternatives than columns");
  K3_REQUIRE((num_alternatives > 0) == (d_alt_log_probs || d_alt_labels), "k3_label_logprobs: alternatives and their number do not go together");
  if (rows == 0) return K3_OK;
  K3_REQUIRE(d_z && (d_labels || !d_log_prob), "k3_label_logprobs: null input");
  const int64_t need = k3_label_logprobs_workspace(dtype, rows, cols, num_alternatives);
  K3_REQUIRE(need == 0 || (d_workspace && workspace_bytes >= need && ((uintptr_t)d_workspace & 15) == 0), "k3_label_logprobs: workspace too small or not aligned");
  const Span z = matrix_span(d_z, ld, rows, cols, dtype_size(dtype)), y = vector_span(d_labels, rows);
  for (const Span &out : {vector_span(d_log_prob, rows), vector_span(d_entropy, rows), vector_span(d_stats, 2 * (int64_t)rows), vector_span(d_alt_log_probs, (int64_t)rows * num_alternatives),
                          vector_span(d_alt_labels, (int64_t)rows * num_alternatives)})
    K3_REQUIRE(!on_any(out, {z, y}), "k3_label_logprobs: an output lies on an input");
  ScoreArgs p{};
  p.z = d_z; p.ld = ld; p.rows = rows; p.cols = cols; p.labels = d_labels; p.a = kLog2e;
  p.log_prob = d_log_prob; p.entropy = d_entropy; p.stats = d_stats; p.alt_log_probs = d_alt_log_probs; p.alt_labels = d_alt_labels; p.top = num_alternatives;
  int rc = K3_OK;
#define K3_LABELS(T) rc = label_logprobs<T>(p, d_workspace, (hipStream_t)stream)
  K3_FOR_DTYPE(dtype, K3_LABELS);
  return rc;
}

extern "C" int k3_label_logprobs_deriv(int32_t dtype, const void *d_z, int64_t ld, const int32_t *d_labels, const float *d_stats, const float *d_entropy, const float *d_log_prob_deriv,
                                       const float *d_entropy_deriv, void *d_dz, int64_t ldd, int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_label_logprobs_deriv: unknown type");
  K3_REQUIRE(rows >= 0 && cols >= 1 && ld >= cols && ldd >= cols, "k3_label_logprobs_deriv: bad argument");
  if (cols > kMaxDerivCols) { set_error("k3_label_logprobs_deriv: at most %d columns", kMaxDerivCols); return K3_ERR_UNSUPPORTED; }
  if (rows == 0) return K3_OK;
  K3_REQUIRE(d_z && d_dz && d_stats && (d_labels || !d_log_prob_deriv) && (d_entropy || !d_entropy_deriv), "k3_label_logprobs_deriv: null input");
  const Span z = matrix_span(d_z, ld, rows, cols, dtype_size(dtype)), dz = matrix_span(d_dz, ldd, rows, cols, dtype_size(dtype));
  K3_REQUIRE((same(z, dz) || !overlap(z, dz)) && !on_any(dz, {vector_span(d_labels, rows), vector_span(d_stats, 2 * (int64_t)rows), vector_span(d_entropy, rows), vector_span(d_log_prob_deriv, rows),
                                                              vector_span(d_entropy_deriv, rows)}), "k3_label_logprobs_deriv: the output lies on another operand");
#define K3_LABEL_DERIV(T)                                                                                                                            \
  const int segments = (cols + 256 * Chunk<T>::N - 1) / (256 * Chunk<T>::N);                                                                         \
  const long long items = (long long)rows * segments, blocks = (items + 3) / 4;                                                                      \
  K3_REQUIRE(blocks <= kMostGroups, "k3_label_logprobs_deriv: matrix too large");                                                                    \
  hipLaunchKernelGGL((k3_label_deriv_kernel<T>), grid_of(blocks, 256), dim3(256), 0, (hipStream_t)stream, (const T *)d_z, (long long)ld, d_labels,   \
                    d_stats, d_entropy, d_log_prob_deriv, d_entropy_deriv, (T *)d_dz, (long long)ldd, cols, segments, items)
  K3_FOR_DTYPE(dtype, K3_LABEL_DERIV);
  K3_HIP_CHECK(hipGetLastError());
  return K3_OK;
}

extern "C" int64_t k3_distill_workspace(int32_t dtype, int32_t rows, int32_t cols, int32_t num_entries, int32_t with_deriv) {
  if (!dtype_ok(dtype) || rows <= 0 || cols <= 0 || num_entries <= 0) return 0;
  return dtype == K3_F32 ? distill_workspace<float>(rows, cols, num_entries, with_deriv) : distill_workspace<f16>(rows, cols, num_entries, with_deriv);
}

extern "C" int k3_distill_objf_and_deriv(int32_t dtype, float temperature, const void *d_z, int64_t ld, const void *d_teacher_values, int64_t ld_values, const int32_t *d_teacher_indexes,
                                         int64_t ld_indexes, int32_t num_entries, const float *d_weights, float *d_objf, void *d_dz, int64_t ldd, void *d_workspace,
                                         int64_t workspace_bytes, int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_distill_objf_and_deriv: unknown type");
  K3_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, "k3_distill_objf_and_deriv: the temperature is to be within 1e-3 .. 1e3");
  K3_REQUIRE(rows >= 0 && cols >= 1 && num_entries >= 1 && ld >= cols && ld_values >= num_entries && ld_indexes >= num_entries && (!d_dz || ldd >= cols),
             "k3_distill_objf_and_deriv: bad argument");
  if (cols > kMaxCols || num_entries > kMaxTeacher) { set_error("k3_distill_objf_and_deriv: at most %d columns and %d entries per row", kMaxCols, kMaxTeacher); return K3_ERR_UNSUPPORTED; }
  if (rows == 0) return K3_OK;
  K3_REQUIRE(d_z && d_teacher_values && d_teacher_indexes && d_objf, "k3_distill_objf_and_deriv: null input");
  const int64_t need = k3_distill_workspace(dtype, rows, cols, num_entries, d_dz != nullptr);
  K3_REQUIRE(need == 0 || (d_workspace && workspace_bytes >= need && ((uintptr_t)d_workspace & 15) == 0), "k3_distill_objf_and_deriv: workspace too small or not aligned");
  const size_t size = dtype_size(dtype);
  const Span z = matrix_span(d_z, ld, rows, cols, size), v = matrix_span(d_teacher_values, ld_values, rows, num_entries, size), i = matrix_span(d_teacher_indexes, ld_indexes, rows, num_entries, 4),
             w = vector_span(d_weights, rows), f = vector_span(d_objf, rows), dz = matrix_span(d_dz, ldd, rows, cols, size);
  K3_REQUIRE((same(z, dz) || !overlap(z, dz)) && !on_any(dz, {v, i, w, f}) && !on_any(f, {z, v, i, w}), "k3_distill_objf_and_deriv: an output lies on another operand");
  DistillArgs p{};
  p.z = d_z; p.ld = ld; p.rows = rows; p.cols = cols; p.values = d_teacher_values; p.ld_values = ld_values; p.indexes = d_teacher_indexes; p.ld_indexes = ld_indexes;
  p.top = num_entries; p.weights = d_weights; p.temperature = temperature; p.a = kLog2e / temperature; p.objf = d_objf; p.dz = d_dz; p.ldd = ldd;
  int rc = K3_OK;
#define K3_DISTILL(T) rc = distill<T>(p, d_workspace, (hipStream_t)stream)
  K3_FOR_DTYPE(dtype, K3_DISTILL);
  return rc;
}
