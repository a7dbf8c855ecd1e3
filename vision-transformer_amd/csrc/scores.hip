// Operators on class scores (logits): log probabilities of given classes with entropy and top alternatives, and
// distillation from a teacher's top log probabilities, each with its gradient.
//
//   log_probs       x = z / T, m = max x, s = sum e^(x - m): lse = m + ln s, log p_v = x_v - lse,
//                   H = ln s - sum e^(x - m) (x - m) / s, and the K largest x in order
//   log_probs_bwd   dz_v = p_v / T * (g_lse - sum g_entries - g_H (log p_v + H)) + sum of the entries at v / T
//   distill         q from the teacher's list, p = softmax(z / T):
//                   (1 - a) T^2 [sum q_k (ln q_k - ln p(c_k)) + q_r (ln q_r - ln p_r)] + a CE(z, y), and d/dz
//
// All of them are bound by HBM: one multiply-add, one exponential and a few adds per class against 2 or 4 bytes.  A row belongs
// to one wave or workgroup (plan_rows) that walks over it in 16-byte granules with running maxima and sums (6.0 TB/s of reads at
// 4096 x 65537 bf16 with entropies, call after call, 5.6 under the profiler, where a copy of 2 GiB reaches 4.9 TB/s of reads and
// writes); what belongs to the row besides, the given classes, the top list, the teacher's list, hides behind other rows' walks.
// Loss and gradient in one call keep the row in registers between the two where that is faster (plan_distill_fused).  Classes that pass once bypass the caches
// (nontemporal): 81 us against 95 us for the bare walk over 512 MiB.
// A granule is 16 aligned bytes of memory, whatever the alignment of the row: the granules a row covers only in part are read and
// written class by class, so that nothing outside the row is touched and odd row lengths keep 16-byte accesses.
//
// Sums and maxima are fp32, combined in a fixed order (logarithms and their differences, and the total of a distillation's
// rows: 64 bits); no floating-point atomics, so equal calls give equal bits.  Outputs of 16 bits are rounded once, from fp32.
#include "common.h"

typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

namespace {

constexpr int kMaxTop = 128;          // length of a top list, of a teacher's list and of a target list
constexpr int kMaxClasses = 500000;   // what the LDS of a workgroup has room for: 32 cells a thread, a byte a granule
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
#define NINF (-__builtin_inff())

// ---- rows and granules -------------------------------------------------------------------------------------------
template <typename T> struct Gran;
template <> struct Gran<bf16_t> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float at(u32x4_t d, int e) {
    const unsigned w = d[e >> 1];
    return __builtin_bit_cast(float, (e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ u32x4_t pack(const float* x) {
    u32x4_t d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = pack_bf2(x[2 * i], x[2 * i + 1]);
    return d;
  }
  static __device__ __forceinline__ float get(const bf16_t* p) { return bf2f(*p); }
  static __device__ __forceinline__ void put(bf16_t* p, float v) { *p = f2bf(v); }
  static __device__ __forceinline__ unsigned ninf() { return 0xff80ff80u; }
  static __device__ __forceinline__ u32x4_t next(u32x4_t d) {   // its classes move down by one
    return u32x4_t{d[0] >> 16 | d[1] << 16, d[1] >> 16 | d[2] << 16, d[2] >> 16 | d[3] << 16, d[3] >> 16};
  }
};
template <> struct Gran<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float at(u32x4_t d, int e) {
    const unsigned w = d[e];   // by value: a bit cast of the vector's element itself reads element 0
    return __builtin_bit_cast(float, w);
  }
  static __device__ __forceinline__ u32x4_t pack(const float* x) {
    u32x4_t d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = __builtin_bit_cast(unsigned, x[i]);
    return d;
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ unsigned ninf() { return 0xff800000u; }
  static __device__ __forceinline__ u32x4_t next(u32x4_t d) { return u32x4_t{d[1], d[2], d[3], 0u}; }
};

// Where the rows of a call are: row r starts at base + (r / inner) * ld_outer + (r % inner) * ld elements.
struct RowsAt {
  int64_t ld_outer, ld;
  int inner;
  __host__ __device__ int64_t offset(int r) const { return (int64_t)(r / inner) * ld_outer + (int64_t)(r % inner) * ld; }
};

template <typename T> struct Row {
  const T* p;
  const char* g0;   // the granule that holds the first class
  int a;            // classes' worth of it in front of the row
  int V, nq;        // classes, granules touched
  int qf, ql;       // first and last granule that lie in the row entirely (ql < qf: none)
  __device__ __forceinline__ Row(const T* base, const RowsAt& at, int r, int V_) {
    constexpr int E = Gran<T>::E;
    p = base + at.offset(r);
    a = (int)(((uintptr_t)p & 15) / sizeof(T));
    g0 = (const char*)p - a * sizeof(T);
    V = V_;
    nq = (V + a + E - 1) / E;
    qf = a > 0 ? 1 : 0;
    ql = (V + a) / E - 1;
  }
  __device__ __forceinline__ bool head_partial() const { return a > 0 || V < Gran<T>::E; }
  __device__ __forceinline__ bool tail_partial() const { return (V + a) % Gran<T>::E != 0 && (nq > 1 || !head_partial()); }
  __device__ __forceinline__ int first_class(int q) const { return q * Gran<T>::E - a; }
};

// A segment [qa, qb) of a row's granules (the whole row, or the part that a workgroup maps) is walked in three parts: whole chunks
// of NV granules a thread, without a condition; the rest of the granules that lie in the row entirely; and the row's first and last
// granule where they do not ("edges", one thread each).  The index of what a thread holds: granule q0 + j * G + tid, or
// edge_granule().
template <typename T> struct Segment {
  int lo, hi;         // granules of the segment that lie in the row entirely
  bool head, tail;    // the segment holds the partial first / last granule
  __device__ __forceinline__ Segment(const Row<T>& row, int qa, int qb) {
    lo = max(qa, row.qf);
    hi = max(lo, min(qb, row.ql + 1));
    head = row.head_partial() && qa == 0;
    tail = row.tail_partial() && qa < row.nq && qb >= row.nq;
  }
  __device__ __forceinline__ bool edges() const { return head || tail; }
};
template <typename T> __device__ __forceinline__ int edge_granule(const Row<T>& row, const Segment<T>& sg, int tid) {
  return tid == 0 && sg.head ? 0 : tid == 1 && sg.tail ? row.nq - 1 : -1;
}
template <typename T> __device__ __forceinline__ u32x4_t no_class() {
  const unsigned ni = Gran<T>::ninf();
  return u32x4_t{ni, ni, ni, ni};
}
template <typename T> __device__ __forceinline__ const u32x4_t* granule(const Row<T>& row, int q) {
  return (const u32x4_t*)(row.g0 + (int64_t)q * 16);
}
template <typename T, int G, int NV, bool ONCE>
__device__ __forceinline__ void load_whole(const Row<T>& row, int q0, int tid, u32x4_t (&d)[NV]) {
  const u32x4_t* p = granule(row, q0 + tid);
#pragma unroll
  for (int j = 0; j < NV; ++j) d[j] = ONCE ? __builtin_nontemporal_load(p + j * G) : p[j * G];
}
template <typename T, int G, int NV>
__device__ __forceinline__ void load_rest(const Row<T>& row, int q0, int hi, int tid, u32x4_t (&d)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int q = q0 + j * G + tid;
    d[j] = no_class<T>();
    if (q < hi) d[j] = *granule(row, q);
  }
}
// an edge granule, classes outside the row as -inf
template <typename T> __device__ __forceinline__ u32x4_t load_edge(const Row<T>& row, int q) {
  constexpr int E = Gran<T>::E;
  float x[E];
  const int c0 = row.first_class(q);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = NINF;
    if (c0 + e >= 0 && c0 + e < row.V) x[e] = Gran<T>::get(row.p + c0 + e);
  }
  return Gran<T>::pack(x);
}

// out[row][c] for the classes of granule q, 16 bytes at a time where the output row lies on granules as the input row does
template <typename T>
__device__ __forceinline__ void store_granule(const Row<T>& row, T* out, bool same, int q, const float* x) {
  constexpr int E = Gran<T>::E;
  const int c0 = row.first_class(q);
  if (same && q >= row.qf && q <= row.ql) {
    *(u32x4_t*)(out + c0) = Gran<T>::pack(x);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c0 + e >= 0 && c0 + e < row.V) Gran<T>::put(out + c0 + e, x[e]);
  }
}
template <typename T> __device__ __forceinline__ bool same_granules(const T* in, const T* out) {
  return (((uintptr_t)in ^ (uintptr_t)out) & 15) == 0;
}

// out = f(score) for the classes of a segment
template <typename T, int G, int NV, class F>
__device__ __forceinline__ void map_segment(const Row<T>& row, const Segment<T>& sg, T* out, F f) {
  constexpr int E = Gran<T>::E;
  const int tid = threadIdx.x;
  const bool same = same_granules(row.p, (const T*)out);
  auto one = [&](u32x4_t d, int q) {
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = f(Gran<T>::at(d, e));
    store_granule(row, out, same, q, x);
  };
  int q0 = sg.lo;
  if (same) {
    char* o0 = (char*)(out + row.first_class(0));   // the granules of the output row
    for (; q0 + G * NV <= sg.hi; q0 += G * NV) {
      u32x4_t d[NV];
      load_whole<T, G, NV, true>(row, q0, tid, d);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = f(Gran<T>::at(d[j], e));
        __builtin_nontemporal_store(Gran<T>::pack(x), (u32x4_t*)(o0 + (int64_t)(q0 + j * G + tid) * 16));
      }
    }
  }
  for (int q = q0 + tid; q < sg.hi; q += G) one(*granule(row, q), q);
  const int q = edge_granule(row, sg, tid);
  if (q >= 0) one(load_edge(row, q), q);
}

// A barrier alone orders what waves write to LDS: their stores to memory may still be on their way, and another wave's store to the
// same place would race with them.
__device__ __forceinline__ void barrier_after_stores() {
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
  __syncthreads();
}

// What lanes of this wave wrote to LDS before is seen by its other lanes behind it.  LDS serves a wave's accesses in order, so this
// costs no instruction; without it nothing keeps the compiler from moving a read in front of the write.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- reductions over a workgroup of G threads --------------------------------------------------------------------
// Within a wave by lane permutations of the VALU (DPP): a shuffle through LDS takes tens of cycles of a pipe that all waves of a
// CU share, and the short rows of a classifier are mostly such reductions.  All lanes have to be active.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
struct Halves {
  float lo, hi;
};
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
  const Halves h = __builtin_bit_cast(Halves, v);
  return __builtin_bit_cast(double, Halves{dpp<CTRL>(h.lo), dpp<CTRL>(h.hi)});
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  const Halves h = __builtin_bit_cast(Halves, v);
  return __builtin_bit_cast(double, Halves{lane_value(h.lo, lane), lane_value(h.hi, lane)});
}
// op over groups of N neighbouring lanes, the same result in all of them
template <int N, class F, class Op> __device__ __forceinline__ F lane_reduce(F v, Op op) {
  static_assert(N == 4 || N == 8 || N == 16 || N == 64, "groups of a quad, half a row, a row or the wave");
  v = op(v, dpp<0xB1>(v));                      // quad_perm 1 0 3 2
  v = op(v, dpp<0x4E>(v));                      // quad_perm 2 3 0 1
  if constexpr (N >= 8) v = op(v, dpp<0x141>(v));    // row_half_mirror
  if constexpr (N >= 16) v = op(v, dpp<0x140>(v));   // row_mirror
  if constexpr (N == 64) v = op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
  return v;
}
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
  template <class F> __device__ __forceinline__ F operator()(F a, F b) const { return a + b; }
};
__device__ __forceinline__ float wave_max(float v) { return lane_reduce<64>(v, Max()); }
template <class F> __device__ __forceinline__ F wave_add(F v) { return lane_reduce<64>(v, Add()); }
template <int G> __device__ __forceinline__ float block_max(float v, float* sh) {
  v = wave_max(v);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < G / 64; ++w) v = fmaxf(v, sh[w]);
    __syncthreads();
  }
  return v;
}
template <int G> __device__ __forceinline__ int block_total(int wave_uniform, int* sh) {   // sum of one number per wave
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = wave_uniform;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) t += sh[w];
    __syncthreads();
    return t;
  }
  return wave_uniform;
}

// Partial softmax sums with respect to the maximum m: s = sum 2^(c (x - m)), s1 the same with c1, u = sum 2^t t for
// t = c (x - m).  m = -inf stands for "no class yet" (s = 0); a NaN or +inf among the scores makes s NaN, and keeps it so.
struct Sums {
  float m, s, s1, u;
};
// ln x by the hardware's base-2 function: off by a unit or two of fp32 where it is used (arguments of 1 or more)
__device__ __forceinline__ float ln_of(float x) { return kLn2 * __builtin_amdgcn_logf(x); }
// ln x to 4e-8 whatever its size: the exponent's part in 64 bits, the hardware's logarithm for the mantissa in [0.5, 1)
__device__ __forceinline__ double wide_ln_of(float x) {
  return fma((double)__builtin_amdgcn_frexp_expf(x), 0.6931471805599453, (double)ln_of(__builtin_amdgcn_frexp_mantf(x)));
}
__device__ __forceinline__ float rebase(float m, float M, float c) { return m == NINF ? 0.f : __builtin_amdgcn_exp2f((m - M) * c); }
__device__ __forceinline__ void rebase_to(Sums& a, float M, float c, float c1) {
  const float w = rebase(a.m, M, c), t = a.m == NINF ? 0.f : (a.m - M) * c;
  a.u = w * fmaf(t, a.s, a.u);   // w = 0 leaves 0; t is finite wherever w is not 0
  if (w == 0.f && a.u != a.u) a.u = 0.f;
  a.s *= w;
  a.s1 *= rebase(a.m, M, c1);
  a.m = M;
}
template <bool TWO, bool ENT>
__device__ __forceinline__ Sums merge(Sums a, Sums b, float c, float c1) {
  const float M = fmaxf(a.m, b.m);
  rebase_to(a, M, c, c1);
  rebase_to(b, M, c, c1);
  a.s += b.s;
  if (TWO) a.s1 += b.s1;
  if (ENT) a.u += b.u;
  return a;
}

// a chunk joins this thread's running sums; returns the chunk's maximum
template <typename T, int NV, bool TWO, bool ENT>
__device__ __forceinline__ float add_chunk(Sums& r, const u32x4_t (&d)[NV], float c, float c1) {
  constexpr int E = Gran<T>::E;
  float top = NINF;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, Gran<T>::at(d[j], e));
  const float m = fmaxf(r.m, top);
  rebase_to(r, m, c, c1);
  const float b = m == NINF ? 0.f : m;
  float s[2] = {0.f, 0.f}, s1[2] = {0.f, 0.f}, u[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = Gran<T>::at(d[j], e) - b, t = x * c, w = __builtin_amdgcn_exp2f(t);
      s[e & 1] += w;
      if (TWO) s1[e & 1] += __builtin_amdgcn_exp2f(x * c1);
      if (ENT) u[e & 1] = fmaf(w, fmaxf(t, -1e30f), u[e & 1]);   // 0 for a masked class
    }
  r.s += s[0] + s[1];
  if (TWO) r.s1 += s1[0] + s1[1];
  if (ENT) r.u += u[0] + u[1];
  return top;
}
// each thread's part of the sums of a row.  take(d, q): what to make of granule q before it counts (the tail form takes the
// listed classes out); seen(i, m): the maximum of the thread's i-th chunk, the edges' last.
struct AsItIs {
  __device__ __forceinline__ u32x4_t operator()(u32x4_t d, int) const { return d; }
};
struct NoMaxima {
  __device__ __forceinline__ void operator()(int, float) const {}
};
template <typename T, int G, int NV, bool TWO, bool ENT, bool ONCE, class Take = AsItIs, class Seen = NoMaxima>
__device__ __forceinline__ Sums row_sums(const Row<T>& row, const Segment<T>& sg, float c, float c1, Take take = Take(), Seen seen = Seen()) {
  const int tid = threadIdx.x % G;   // (a workgroup may hold several rows of one wave each)
  Sums r = {NINF, 0.f, 0.f, 0.f};
  int q0 = sg.lo, i = 0;
  for (; q0 + G * NV <= sg.hi; q0 += G * NV, ++i) {
    u32x4_t d[NV];
    load_whole<T, G, NV, ONCE>(row, q0, tid, d);
#pragma unroll
    for (int j = 0; j < NV; ++j) d[j] = take(d[j], q0 + j * G + tid);
    seen(i, add_chunk<T, NV, TWO, ENT>(r, d, c, c1));
  }
  if (q0 < sg.hi) {
    u32x4_t d[NV];
    load_rest<T, G, NV>(row, q0, sg.hi, tid, d);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (q0 + j * G + tid < sg.hi) d[j] = take(d[j], q0 + j * G + tid);
    seen(i++, add_chunk<T, NV, TWO, ENT>(r, d, c, c1));
  }
  if (sg.edges()) {
    u32x4_t d[1] = {no_class<T>()};
    const int q = edge_granule(row, sg, tid);
    if (q >= 0) d[0] = take(load_edge(row, q), q);
    seen(i, add_chunk<T, 1, TWO, ENT>(r, d, c, c1));
  }
  return r;
}
// the sums of N neighbouring lanes, the same in all of them
template <int N, bool TWO, bool ENT> __device__ __forceinline__ Sums lane_sums(Sums r, float c, float c1) {
  rebase_to(r, lane_reduce<N>(r.m, Max()), c, c1);
  r.s = lane_reduce<N>(r.s, Add());
  if (TWO) r.s1 = lane_reduce<N>(r.s1, Add());
  if (ENT) r.u = lane_reduce<N>(r.u, Add());
  return r;
}
// every thread's sums -> the workgroup's, the same in all threads
template <int G, bool TWO, bool ENT> __device__ __forceinline__ Sums block_sums(Sums r, float c, float c1, float* sh) {
  r = lane_sums<(G < 64 ? G : 64), TWO, ENT>(r, c, c1);   // G < 64: of the G lanes that share a row
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    if ((threadIdx.x & 63) == 0) *(Sums*)(sh + 4 * (threadIdx.x >> 6)) = r;
    __syncthreads();
    r = lane_sums<W, TWO, ENT>(*(const Sums*)(sh + 4 * (threadIdx.x % W)), c, c1);
    __syncthreads();
  }
  return r;
}

// ---- the K largest of a row, in order -------------------------------------------------------------------------------
// A value and its class are one 64-bit key, the larger the earlier in the list: the value's bits in an order of unsigned numbers,
// then the class, the lower first.  (-0 counts as 0.)
typedef unsigned long long key64;
__device__ __forceinline__ unsigned float_key(float f) {
  const unsigned b = __builtin_bit_cast(unsigned, f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_float(unsigned k) {
  return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ key64 key_of(float v, int i) { return (key64)float_key(v + 0.f) << 32 | (unsigned)~i; }
__device__ __forceinline__ float value_of(key64 k) { return key_float((unsigned)(k >> 32)); }
__device__ __forceinline__ int class_of(key64 k) { return (int)~(unsigned)k; }

constexpr int kCand = 512;
struct __align__(16) TopScratch {
  key64 key[kCand];     // candidates, in any order
  float group[256];     // maxima of groups of threads
  int n, cells;         // how many there are, which may exceed the room
  int cnt[16];
  float red[16];
};
struct TopList {
  key64 key[2][kMaxTop];   // in order, in key[cur]; before the first values come, as if below everything
  float thr;               // the K-th value
  int cur;
};
template <int G> __device__ __forceinline__ void clear_list(int K, TopScratch& sc, TopList& L) {
  for (int k = threadIdx.x; k < K; k += G) L.key[0][k] = 0;
  if (threadIdx.x == 0) {
    L.cur = 0;
    L.thr = NINF;
    sc.n = sc.cells = 0;
  }
  __syncthreads();
}
// the first n candidates join the list: each finds its rank by counting those before it
template <int G> __device__ __forceinline__ void merge_list(int K, int n, TopScratch& sc, TopList& L) {
  const int tid = threadIdx.x, cur = L.cur;
  const bool fresh = L.key[cur][0] == 0;
  const int listed = fresh && n >= K ? 0 : K;   // of the list: none where the candidates fill it
  for (int k = tid; k < n + listed; k += G) {
    const key64 mine = k < n ? sc.key[k] : L.key[cur][k - n];
    int rank = k < n ? 0 : k - n;   // the list is in order
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += sc.key[j] > mine ? 1 : 0;
    if (k < n && !fresh)
#pragma unroll 8
      for (int j = 0; j < K; ++j) rank += L.key[cur][j] > mine ? 1 : 0;
    if (rank < K) L.key[cur ^ 1][rank] = mine;
  }
  __syncthreads();
  if (tid == 0) {
    const key64 last = L.key[cur ^ 1][K - 1];
    L.cur = cur ^ 1;
    L.thr = last == 0 ? NINF : value_of(last);
    sc.n = 0;
  }
  __syncthreads();
}

// A lower bound of the K-th largest class from the maxima of min(G, 256) groups of threads: at least K of them reach it, hence
// K classes, and hardly more than 5 K / 4 unless many are equal.  Every wave finds it for itself, by bisection over the bits:
// a few ballots a step, where counting for every maximum how many reach it costs 64 LDS reads a thread.
template <int G> __device__ __forceinline__ float bound_of_groups(int K, const TopScratch& sc) {
  constexpr int NG = G < 256 ? G : 256, N = NG / 64;
  if (K > NG) return NINF;
  float g[N], hi = NINF, lo = __builtin_inff();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    g[i] = sc.group[(threadIdx.x & 63) + 64 * i];
    hi = fmaxf(hi, g[i]);
    lo = fminf(lo, g[i]);
  }
  unsigned a = float_key(-wave_max(-lo)), b = float_key(wave_max(hi)) + 1;
  int reach = NG;   // groups that reach a; fewer than K reach b
  while (b - a > 1 && reach > K + K / 4 + 4) {
    const unsigned mid = a + (b - a) / 2;
    const float f = key_float(mid);
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += __popcll(__ballot(g[i] >= f));
    if (c >= K) {
      a = mid;
      reach = c;
    } else {
      b = mid;
    }
  }
  return key_float(a);
}

// The values of the wave that are above thr (AT: or equal to it; TIES: equal to it with a class below `below`, and any class has
// to be in [0, V)) become candidates.  One LDS atomic a wave.
template <int NE, bool AT, bool TIES, class Val, class Idx>
__device__ __forceinline__ void append(TopScratch& sc, float thr, int below, int V, Val val, Idx idx) {
  auto in = [&](int e, float t) {
    if (TIES) return val(e) >= t && (unsigned)idx(e) < (unsigned)(val(e) == t ? below : V);
    return AT ? val(e) >= t : val(e) > t;
  };
  int c = 0;
#pragma unroll
  for (int e = 0; e < NE; ++e) c += in(e, thr) ? 1 : 0;
  if (__ballot(c != 0) == 0) return;
  const int lane = threadIdx.x & 63;
  int end = c;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(end, o, 64);
    if (lane >= o) end += t;
  }
  int base = 0;
  if (lane == 63) base = atomicAdd(&sc.n, end);
  int pos = __shfl(base, 63, 64) + end - c;
  float again = thr;
  asm volatile("" : "+v"(again));   // compared anew: NE masks kept from above would not fit the scalar registers
#pragma unroll
  for (int e = 0; e < NE; ++e)
    if (in(e, again)) {
      if (pos < kCand) sc.key[pos] = key_of(val(e), idx(e));
      ++pos;
    }
}
// The K largest of the values a workgroup holds in registers: val(e) for e in [0, NE), idx(e) their classes, of which only those
// in [0, V) exist (the others' values are -inf); `exist`: how many values the workgroup holds.  Leaves at most kCand candidates
// among which they are (or all, if there are fewer), and returns their number.  Where more reach the bound than there is room
// for (many equal values, or an order that defeats the groups), it is raised by bisection over the bits, and among equal values
// by bisection over the classes.
template <int G, int NE, class Val, class Idx>
__device__ __forceinline__ int select_top(int K, int V, int exist, TopScratch& sc, Val val, Idx idx) {
  const int tid = threadIdx.x;
  constexpr int NG = G < 256 ? G : 256, PER = G / NG;
  float mine = NINF;
#pragma unroll
  for (int e = 0; e < NE; ++e) mine = fmaxf(mine, val(e));
  const float top = block_max<G>(mine, sc.red);
#pragma unroll
  for (int o = 1; o < PER; o <<= 1) mine = fmaxf(mine, __shfl_xor(mine, o, 64));
  if (tid % PER == 0) sc.group[tid / PER] = mine;
  if (tid == 0) sc.n = 0;
  __syncthreads();
  float thr = bound_of_groups<G>(K, sc);
  auto count_from = [&](float f) {   // values >= f > -inf
    int c = 0;
#pragma unroll
    for (int e = 0; e < NE; ++e) c += __popcll(__ballot(val(e) >= f));
    return block_total<G>(c, sc.cnt);
  };
  int below = V;   // of the values equal to thr, those with a class below this belong to the list
  if ((thr == NINF ? exist : count_from(thr)) > kCand) {
    unsigned lo = float_key(thr), hi = float_key(top) + 1;
    bool done = false;
    while (hi - lo > 1 && !done) {
      const unsigned mid = lo + (hi - lo) / 2;
      const int c = count_from(key_float(mid));
      if (c < K) {
        hi = mid;
      } else {
        lo = mid;
        done = c <= kCand;
      }
    }
    thr = key_float(lo);
    if (!done) {   // more than there is room for are equal to thr, fewer than K above it
      int c = 0;
#pragma unroll
      for (int e = 0; e < NE; ++e) c += __popcll(__ballot(val(e) > thr));
      const int need = K - block_total<G>(c, sc.cnt);
      int from = 0;   // fewer than `need` of them below `from`, at least `need` below `below`
      while (below - from > 1) {
        const int mid = from + (below - from) / 2;
        c = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) c += __popcll(__ballot(val(e) == thr && (unsigned)idx(e) < (unsigned)mid));
        if (block_total<G>(c, sc.cnt) >= need) below = mid;
        else from = mid;
      }
    }
  }
  if (thr != NINF && below == V) append<NE, true, false>(sc, thr, V, V, val, idx);
  else append<NE, true, true>(sc, thr, below, V, val, idx);   // -inf also stands where no class is; ties have to be told apart
  __syncthreads();
  return min(sc.n, kCand);
}
// the values above the list's K-th become candidates; returns the number of those there are, which may exceed the room
template <int NE, class Val, class Idx>
__device__ __forceinline__ int offer(TopScratch& sc, const TopList& L, Val val, Idx idx) {
  append<NE, false, false>(sc, L.thr, 0, 0, val, idx);
  __syncthreads();
  const int n = sc.n;
  __syncthreads();
  return n;
}

// ---- log probabilities --------------------------------------------------------------------------------------------
struct LogProbsArgs {
  const void* logits;
  RowsAt at;
  int R, V;
  float inv_t;
  const int64_t* targets;
  int G;                 // targets a row
  int64_t ignore;
  int K;
  float *logprobs, *lse, *entropy, *top_lp;
  int64_t* top_idx;
  float* stats;          // [R][2]: m (unscaled), s: what the gradient needs
};

// a given class of a row and its score: fetched before the walk over the row, so that nothing waits for it behind
struct Given {
  int64_t y;
  float z;
};
template <typename T> __device__ __forceinline__ Given fetch_given(const LogProbsArgs& A, const T* p, int r, int g) {
  Given v = {A.ignore, 0.f};
  if (g < A.G) {
    v.y = A.targets[(int64_t)r * A.G + g];
    if (v.y >= 0 && v.y < A.V) v.z = Gran<T>::get(p + v.y);
  }
  return v;
}
// x - lse for a score z: the difference is 64 bits and rounded once
__device__ __forceinline__ float log_prob(float z, float m, float inv_t, double ln_s) {
  return (float)fma((double)z - (double)m, (double)inv_t, -ln_s);
}
// everything of a row that follows from its sums, by `n` threads, each of which holds the given class of its own number
template <typename T>
__device__ __forceinline__ void row_answers(const LogProbsArgs& A, const T* p, int r, Sums t, Given v, int tid, int n) {
  float inv_t = A.inv_t;
  asm volatile("" : "+v"(inv_t), "+v"(v.z));   // widened here: in front of the walk the 64 bits would cost it registers
  const double ln_s = wide_ln_of(t.s);
  const bool none = t.m == NINF && t.s == 0.f;      // no class has a finite score
  if (tid == 0) {
    if (A.lse) A.lse[r] = none ? NINF : (float)fma((double)t.m, (double)inv_t, ln_s);
    if (A.entropy) A.entropy[r] = none ? 0.f : (float)(ln_s - (double)(kLn2 * (t.u / t.s)));
    if (A.stats) {
      A.stats[2 * (int64_t)r] = t.m;
      A.stats[2 * (int64_t)r + 1] = t.s;
    }
  }
  for (int g = tid; g < A.G; g += n) {
    if (g != tid) v = fetch_given<T>(A, p, r, g);
    float lp = 0.f;
    if (v.y != A.ignore) {
      if (v.y < 0 || v.y >= A.V) lp = __builtin_nanf("");
      else lp = none ? NINF : log_prob(v.z, t.m, inv_t, ln_s);
    }
    A.logprobs[(int64_t)r * A.G + g] = lp;
  }
}
__device__ __forceinline__ void put_list(const LogProbsArgs& A, int r, Sums t, const TopList& L, int tid, int n) {
  const double ln_s = wide_ln_of(t.s);
  const bool nan = t.s != t.s;
  for (int k = tid; k < A.K; k += n) {
    const int64_t at = (int64_t)r * A.K + k;
    const key64 v = L.key[L.cur][k];
    A.top_lp[at] = nan ? t.s : t.m == NINF ? NINF : log_prob(value_of(v), t.m, A.inv_t, ln_s);
    A.top_idx[at] = nan ? -1 : (int64_t)class_of(v);
  }
}

// Short rows share a workgroup of 256 threads, the shortest a wave: 4 lanes a row of up to 4 granules, 16 up to 16.  A million
// rows of 10 bf16 classes with a target each take 440 us with a wave each, bound by instructions, 36 us so.
constexpr int rows_of_group(int G) { return G <= 64 ? 256 / G : 1; }
template <typename T, int G, int NV>
__global__ __launch_bounds__(G * rows_of_group(G)) void log_probs_kernel(LogProbsArgs A) {
  __shared__ __align__(16) float sh[G > 64 ? 4 * (G / 64) : 4];
  const int r = blockIdx.x * rows_of_group(G) + threadIdx.x / G, tid = threadIdx.x % G;
  if (r >= A.R) return;   // all the lanes of a row, and of a long row's workgroup
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  const Segment<T> sg(row, 0, row.nq);
  const float c = A.inv_t * kLog2e;
  const Given given = fetch_given<T>(A, row.p, r, tid);
  Sums t = A.entropy ? row_sums<T, G, NV, false, true, true>(row, sg, c, 0.f) : row_sums<T, G, NV, false, false, true>(row, sg, c, 0.f);
  t = block_sums<G, false, true>(t, c, 0.f, sh);
  row_answers<T>(A, row.p, r, t, given, tid, G);
}

// with a top list, one wave a row, all of the row in its registers
template <typename T, int NV>
__global__ __launch_bounds__(64) void log_probs_wave_top_kernel(LogProbsArgs A) {
  constexpr int E = Gran<T>::E;
  __shared__ TopScratch sc;
  __shared__ TopList L;
  const int tid = threadIdx.x, r = blockIdx.x;
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  const Segment<T> sg(row, 0, row.nq);
  const float c = A.inv_t * kLog2e;
  u32x4_t d[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int q = j * 64 + tid;
    d[j] = no_class<T>();
    if (q >= sg.lo && q < sg.hi) d[j] = __builtin_nontemporal_load(granule(row, q));
    else if ((sg.head && q == 0) || (sg.tail && q == row.nq - 1)) d[j] = load_edge(row, q);
  }
  const Given given = fetch_given<T>(A, row.p, r, tid);
  clear_list<64>(A.K, sc, L);
  Sums t = {NINF, 0.f, 0.f, 0.f};
  if (A.entropy) add_chunk<T, NV, false, true>(t, d, c, 0.f);
  else add_chunk<T, NV, false, false>(t, d, c, 0.f);
  t = block_sums<64, false, true>(t, c, 0.f, nullptr);
  row_answers<T>(A, row.p, r, t, given, tid, 64);
  const int n = select_top<64, NV * E>(A.K, row.V, row.V, sc, [&](int e) { return Gran<T>::at(d[e / E], e % E); },
                                       [&](int e) { return row.first_class((e / E) * 64 + tid) + e % E; });
  merge_list<64>(A.K, n, sc, L);
  put_list(A, r, t, L, tid, 64);
}

// With a top list, G threads a row.  The walk over the classes is that of log_probs_kernel; all it leaves for the list is the
// maximum of every cell, the classes of one thread in one chunk (LDS, a float a cell).  The K-th largest of the maxima of 256
// groups of threads bounds the K-th largest class from below, so only cells that reach it can hold classes of the list: about
// K of them, whose few granules are read again.  Where more do than there is room for (a great many equal classes, few unmasked
// ones) the row is read once more in order, a granule a thread, against the K-th of the list so far.
constexpr int kTopChunks = 32;   // most chunks of a row: 32 cells a thread
template <typename T, int G, int NV>
__global__ __launch_bounds__(G) void log_probs_top_kernel(LogProbsArgs A) {
  constexpr int E = Gran<T>::E, PER = G / 256;
  __shared__ __align__(16) float sh[4 * (G / 64)];
  __shared__ TopScratch sc;
  __shared__ TopList L;
  __shared__ int cells[kCand];      // chunk * G + thread of those that reach the bound, in any order
  extern __shared__ float cell[];   // [chunk][thread]
  const int tid = threadIdx.x, r = blockIdx.x;
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  const Segment<T> sg(row, 0, row.nq);
  const float c = A.inv_t * kLog2e;
  const int chunks = (sg.hi - sg.lo + G * NV - 1) / (G * NV);
  const Given given = fetch_given<T>(A, row.p, r, tid);
  clear_list<G>(A.K, sc, L);
  float mine = NINF;
  auto seen = [&](int i, float m) {
    mine = fmaxf(mine, m);
    if (i < chunks) cell[i * G + tid] = m;
  };
  Sums t = A.entropy ? row_sums<T, G, NV, false, true, true>(row, sg, c, 0.f, AsItIs(), seen)
                     : row_sums<T, G, NV, false, false, true>(row, sg, c, 0.f, AsItIs(), seen);
  t = block_sums<G, false, true>(t, c, 0.f, sh);
  row_answers<T>(A, row.p, r, t, given, tid, G);

#pragma unroll
  for (int o = 1; o < PER; o <<= 1) mine = fmaxf(mine, __shfl_xor(mine, o, 64));
  if (tid % PER == 0) sc.group[tid / PER] = mine;
  __syncthreads();
  const float thr = bound_of_groups<G>(A.K, sc);
  int some = 0;
  for (int i = 0; i < chunks; ++i) some += cell[i * G + tid] >= thr ? 1 : 0;
  if (some > 0) {
    int pos = atomicAdd(&sc.cells, some);
    for (int i = 0; i < chunks; ++i)
      if (cell[i * G + tid] >= thr) {
        if (pos < kCand) cells[pos] = i * G + tid;
        ++pos;
      }
  }
  __syncthreads();
  bool whole = sc.cells > kCand;
  if (!whole) {
    auto take = [&](u32x4_t d, int q) {
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const float v = Gran<T>::at(d, 0);
        const int i = row.first_class(q) + e;
        if (v >= thr && (unsigned)i < (unsigned)row.V) {
          const int pos = atomicAdd(&sc.n, 1);
          if (pos < kCand) sc.key[pos] = key_of(v, i);
        }
        d = Gran<T>::next(d);
      }
    };
    for (int k = tid; k < sc.cells * NV; k += G) {
      const int id = cells[k / NV], q = sg.lo + (id / G) * G * NV + (k % NV) * G + id % G;
      if (q < sg.hi) take(*granule(row, q), q);
    }
    const int eq = edge_granule(row, sg, tid);
    if (eq >= 0) take(load_edge(row, eq), eq);
    __syncthreads();
    const int n = sc.n;
    __syncthreads();
    if (n <= kCand) {
      merge_list<G>(A.K, n, sc, L);
    } else {
      whole = true;
      if (tid == 0) sc.n = 0;
      __syncthreads();
    }
  }
  if (whole) {
    int waiting = 0;
    for (int q0 = 0; q0 < row.nq; q0 += G) {   // in the order of the classes, edges included
      const int q = q0 + tid;
      u32x4_t d = no_class<T>();
      if (q >= sg.lo && q < sg.hi) d = *granule(row, q);
      else if ((sg.head && q == 0) || (sg.tail && q == row.nq - 1)) d = load_edge(row, q);
      auto val = [&](int e) { return Gran<T>::at(d, e); };
      auto idx = [&](int e) { return q < row.nq ? row.first_class(q) + e : row.V; };
      for (int attempt = q0 == 0 ? 2 : 0;;) {
        const int n = attempt < 2 ? offer<E>(sc, L, val, idx)
                                  : select_top<G, E>(A.K, row.V, min(row.nq - q0, G) * E, sc, val, idx);
        if (attempt < 2 && n < 64) {
          waiting = n;
          break;
        }
        const bool room = attempt == 2 || n <= kCand, again = attempt == 0 && waiting > 0;
        merge_list<G>(A.K, room ? n : waiting, sc, L);
        waiting = 0;
        if (room) break;
        attempt = again ? 1 : 2;
      }
    }
    if (waiting > 0) merge_list<G>(A.K, waiting, sc, L);
  }
  put_list(A, r, t, L, tid, G);
}

struct LogProbsBwdArgs {
  const void* logits;
  RowsAt at;
  int R, V, nseg, per;       // segments a row, granules a segment
  float inv_t;
  const int64_t* targets;
  int G;
  int64_t ignore;
  const int64_t* top_idx;
  int K;
  const float *stats, *entropy;
  const float *g_logprobs, *g_lse, *g_entropy, *g_top;   // each nullable
  void* dlogits;
  RowsAt out_at;
};
// One read and one write of HBM: 51 us at 2048 x 32001 bf16, 5.1 TB/s.  The entries (targets and top classes, a class may occur
// several times) are written over the dense part by one thread per different class, which adds them in the order of the list.
template <typename T, int G, int NV>
__global__ __launch_bounds__(G) void log_probs_bwd_kernel(LogProbsBwdArgs A) {
  __shared__ int s_idx[2 * kMaxTop];
  __shared__ float s_g[2 * kMaxTop];
  __shared__ float s_sum;
  const int tid = threadIdx.x;
  const int r = blockIdx.x / A.nseg, seg = blockIdx.x - r * A.nseg;
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  T* out = (T*)A.dlogits + A.out_at.offset(r);
  const int qa = seg * A.per, qb = min(qa + A.per, row.nq);
  if (qa >= qb) return;
  const int ng = A.g_logprobs ? A.G : 0, n = ng + (A.g_top ? A.K : 0);
  for (int k = tid; k < n; k += G) {
    const bool tgt = k < ng;
    const int64_t i = tgt ? A.targets[(int64_t)r * A.G + k] : A.top_idx[(int64_t)r * A.K + k - ng];
    const float g = tgt ? A.g_logprobs[(int64_t)r * A.G + k] : A.g_top[(int64_t)r * A.K + k - ng];
    const bool ok = i >= 0 && i < A.V && !(tgt && i == A.ignore);
    s_idx[k] = ok ? (int)i : -1;
    s_g[k] = ok ? g : 0.f;
  }
  __syncthreads();
  if (tid < 64) {
    float s = 0.f;
    for (int k = tid; k < n; k += 64) s += s_g[k];
    s = wave_add(s);
    if (tid == 0) s_sum = s;
  }
  __syncthreads();
  const float m = A.stats[2 * (int64_t)r], s = A.stats[2 * (int64_t)r + 1];
  const bool none = m == NINF && s == 0.f;
  const float c = A.inv_t * kLog2e, gh = A.g_entropy ? A.g_entropy[r] : 0.f;
  const float lead = (A.g_lse ? A.g_lse[r] : 0.f) - s_sum;
  // dz = w (k0 - k1 t) with w = 2^t, t = c (z - m): log p + H = ln2 t - ln s + H
  const float scale = none ? 0.f : A.inv_t / s;
  const float k1 = gh * kLn2, k0 = lead - (A.g_entropy ? gh * (float)((double)A.entropy[r] - wide_ln_of(s)) : 0.f);
  auto dense = [&](float z) {
    const float t = (z - m) * c, w = __builtin_amdgcn_exp2f(t) * scale;
    return none || w == 0.f ? 0.f : w * fmaf(-k1, t, k0);
  };
  map_segment<T, G, NV>(row, Segment<T>(row, qa, qb), out, dense);
  if (n == 0 || none) return;
  barrier_after_stores();   // the entries are written over the dense values
  const int c0 = row.first_class(qa), c1 = row.first_class(qb);
  for (int k = tid; k < n; k += G) {
    const int i = s_idx[k];
    if (i < 0 || i < c0 || i >= c1) continue;
    float g = 0.f;
    bool first = true;
    for (int j = 0; j < n; ++j)
      if (s_idx[j] == i) {
        if (j < k) first = false;
        g += s_g[j];
      }
    if (first) Gran<T>::put(out + i, fmaf(g, A.inv_t, dense(Gran<T>::get(row.p + i))));
  }
}

// ---- distillation -------------------------------------------------------------------------------------------------
// What the gradient of a row needs (kState floats a row): dz_v = wT 2^(cT (z - md)) + w1 2^(c1 (z - md)) for a class that is
// neither in the teacher's list nor the label; classes of the list go by the totals m, aT, a1 instead (put_entries).
// In the tail form wT is the difference of the softmax's and the tail's weight, taken with respect to the maximum md of the
// classes outside the list, so that neither a tail of tiny mass nor a list that holds nearly everything loses its digits.
constexpr int kState = 8;
struct RowState {
  float md, wT, w1, m, aT, a1, cq, ok;   // ok: 0 = no gradient (ignored row, refused index, no class left)
};
struct DistillArgs {
  const void* logits;
  RowsAt at;
  int R, V, nseg, per;         // segments a row, granules a segment (gradient alone)
  float temperature, label_weight;
  int tail;
  int apart;                   // the listed classes are taken out of the sums over the row (keeps_apart)
  const float* teacher;        // [R][K] log probabilities
  const int64_t* indices;      // [R][K], -1: absent
  int K;
  const int64_t* labels;       // [R] or null
  int64_t ignore;
  float* row_loss;
  float* state;                // [R][kState] or null
  const float* inv_count;      // 1 / (counted rows) on the device, or null: host_scale
  int count_here;              // every workgroup counts the labels itself
  float host_scale;
  const float* upstream;       // null: 1; else one float, or one a row
  int upstream_rows;
  void* dlogits;
  RowsAt out_at;
};
struct __align__(16) ListScratch {
  int idx[kMaxTop];            // -1: absent
  float l[kMaxTop], q[kMaxTop], z[kMaxTop];   // the teacher's log probabilities, its probabilities e^(l - norm), the student's scores
  double norm;
  float q_rest, Q;             // tail mass of the teacher, mass of its list
  int bad;                     // an index outside the classes
  int64_t y;                   // the label and its score
  float zy;
  RowState st;
  Sums dn, tot;                // over the classes that the walk summed, and over all
  bool others;                 // the walk saw classes
  float fixed_loss;            // of a row without a gradient
  float scale;
};
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
// f(j) for the entries j of the list that name class i
template <class F> __device__ __forceinline__ void for_entries(const ListScratch& L, int K, int i, F f) {
#pragma unroll 4
  for (int j = 0; j < K; j += 4) {
    const i32x4_t v = *(const i32x4_t*)(L.idx + j);   // entries from K on are absent
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] == i) f(j + e);
  }
}
// wave 0: the teacher's list of a row and what belongs to it, two entries a lane
template <typename T> __device__ __forceinline__ void read_list(const DistillArgs& A, const T* p, int r, ListScratch& L) {
  const int lane = threadIdx.x & 63;
  const int64_t y = A.labels ? A.labels[r] : A.ignore;
  bool bad = false;
  int ix[2];
  float l[2], z[2], q[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = lane + 64 * h;
    ix[h] = -1;
    l[h] = z[h] = NINF;
    if (k < A.K) {
      const int64_t i = A.indices[(int64_t)r * A.K + k];
      const float t = A.teacher[(int64_t)r * A.K + k];
      if (i >= 0 && i < A.V) {
        ix[h] = (int)i;
        l[h] = t;
        z[h] = Gran<T>::get(p + i);
      } else if (i != -1) {
        bad = true;
      }
    }
  }
  const float zy = y >= 0 && y < A.V ? Gran<T>::get(p + y) : 0.f;
  double norm = 0.;
  if (!A.tail) {   // renormalised over the list
    float mx = wave_max(fmaxf(l[0], l[1]));
    mx = mx == NINF ? 0.f : mx;
    norm = mx + wide_ln_of(wave_add(expf(l[0] - mx) + (A.K > 64 ? expf(l[1] - mx) : 0.f)));
    if (norm == NINF) norm = 0.;   // nothing in the list
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    q[h] = A.K > 64 * h ? expf((float)(l[h] - norm)) : 0.f;
    L.idx[lane + 64 * h] = ix[h];
    L.l[lane + 64 * h] = l[h];
    L.q[lane + 64 * h] = q[h];
    L.z[lane + 64 * h] = z[h];
  }
  const float Q = wave_add(q[0] + q[1]);
  const bool any_bad = __ballot(bad) != 0;
  if (lane == 0) {
    L.Q = Q;
    L.norm = norm;
    L.q_rest = A.tail ? fmaxf(1.f - Q, 0.f) : 0.f;
    L.bad = any_bad;
    L.y = y;
    L.zy = zy;
  }
}

// x - 1 + e^-x for |x| < 1: the series, without the cancellation around 0 (the first term left out is 2e-9)
__device__ __forceinline__ float excess(float x) {
  float p = -1.f / 39916800.f;
  const float c[9] = {1.f / 3628800.f, -1.f / 362880.f, 1.f / 40320.f, -1.f / 5040.f, 1.f / 720.f, -1.f / 120.f, 1.f / 24.f, -1.f / 6.f, 0.5f};
#pragma unroll
  for (int i = 0; i < 9; ++i) p = fmaf(p, x, c[i]);
  return p * x * x;
}
// wave 0: what the gradient of the row needs, from the sums over the row (`apart`: over the classes outside the list).  Returns
// which of the lane's two entries are the first of their class.
struct First {
  bool at[2];
};
__device__ __forceinline__ First row_state(const DistillArgs& A, int r, Sums dn, ListScratch& L) {
  const int lane = threadIdx.x & 63;
  const float cT = kLog2e / A.temperature, c1 = kLog2e, a = A.label_weight;
  wave_sync();   // read_list's, where one wave has the row and met no barrier since
  First first = {{false, false}};
  Sums tot = dn;
  if (A.apart) {   // the listed classes join the sums, each once
    const float z[2] = {L.z[lane], L.z[lane + 64]};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = lane + 64 * h, i = L.idx[k];
      first.at[h] = i >= 0;
      for_entries(L, A.K, i, [&](int j) { first.at[h] = first.at[h] && j >= k; });
    }
    Sums o = {NINF, 0.f, 0.f, 0.f};
    o.m = wave_max(fmaxf(first.at[0] ? z[0] : NINF, first.at[1] ? z[1] : NINF));
    const float b = o.m == NINF ? 0.f : o.m;
    float s = 0.f, s1 = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (first.at[h]) {
        s += __builtin_amdgcn_exp2f((z[h] - b) * cT);
        s1 += __builtin_amdgcn_exp2f((z[h] - b) * c1);
      }
    o.s = wave_add(s);
    o.s1 = wave_add(s1);
    tot = merge<true, false>(dn, o, cT, c1);
  }
  if (lane != 0) return first;
  const bool others = dn.m != NINF || dn.s != 0.f;     // classes outside the list (or NaN)
  const float q_rest = others ? L.q_rest : 0.f, Q = L.Q + (A.apart ? q_rest : 0.f);   // none: no tail term
  const bool labelled = A.labels && L.y != A.ignore, skip = A.labels && L.y == A.ignore;
  const bool bad = L.bad || (labelled && (L.y < 0 || L.y >= A.V));
  const bool none = tot.m == NINF && tot.s == 0.f;
  RowState st = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (!skip && !bad && !none) {
    st.cq = (1.f - a) * A.temperature;
    st.m = tot.m;
    st.aT = st.cq * Q / tot.s;
    st.a1 = a / tot.s1;
    st.md = dn.m == NINF ? 0.f : dn.m;
    st.wT = st.aT * rebase(dn.m, tot.m, cT) - (q_rest > 0.f ? st.cq * q_rest / dn.s : 0.f);
    st.w1 = st.a1 * rebase(dn.m, tot.m, c1);
    st.ok = 1.f;
  }
  if (A.state) *(RowState*)(A.state + (int64_t)r * kState) = st;
  L.st = st;
  L.dn = dn;
  L.tot = tot;
  L.others = others;
  L.fixed_loss = !skip && bad ? __builtin_nanf("") : 0.f;
  return first;
}
// wave 0: the loss of the row.  ln q - ln p of an entry is a difference of numbers that are larger than it by the temperature, and
// the loss T^2 times a sum that is smaller by its square: logarithms and their differences are 64 bits.  Where the listed classes
// are apart the sum is taken as that of q d - q + p over the list and the rest of the classes, d = ln q - ln p, which is the same
// (the q and the p have one sum) and has no negative terms: what all p are off by together then hardly shows.
__device__ __forceinline__ void row_loss(const DistillArgs& A, int r, const First& first, const ListScratch& L) {
  const int lane = threadIdx.x & 63;
  wave_sync();
  if (L.st.ok == 0.f) {
    if (lane == 0) A.row_loss[r] = L.fixed_loss;
    return;
  }
  const float T_ = A.temperature, cT = kLog2e / T_, a = A.label_weight;
  const double inv_t = 1. / (double)T_, norm = L.norm;
  const Sums dn = L.dn, tot = L.tot;
  const double ln_s = wide_ln_of(tot.s);
  const float inv_s = 1.f / tot.s;
  float kl = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (64 * h >= A.K) break;
    const float z = L.z[lane + 64 * h], q = L.q[lane + 64 * h];
    const double x = ((double)z - (double)tot.m) * inv_t;
    const float d = (float)((double)L.l[lane + 64 * h] - norm - x + ln_s);   // where q > 0
    if (!A.apart) {
      kl += q != 0.f ? q * d : 0.f;
    } else {
      const float p = first.at[h] ? __builtin_amdgcn_exp2f((z - tot.m) * cT) * inv_s : 0.f;
      if (q == 0.f) kl += p;
      else kl += first.at[h] && fabsf(d) < 1.f ? q * excess(d) : q * (d - 1.f) + p;
    }
  }
  kl = wave_add(kl);
  const float q_rest = L.others ? L.q_rest : 0.f;
  double over = 0.;   // what the q are off a sum of 1, in the tail form without a tail
  if (A.tail && q_rest == 0.f)
    over = wave_add((L.idx[lane] >= 0 ? exp((double)L.l[lane]) : 0.) + (L.idx[lane + 64] >= 0 ? exp((double)L.l[lane + 64]) : 0.)) - 1.;
  if (lane != 0) return;
  if (A.apart) {
    const float p = L.others ? dn.s * rebase(dn.m, tot.m, cT) * inv_s : 0.f;
    if (q_rest > 0.f) {
      const float d = (float)(wide_ln_of(q_rest) - wide_ln_of(dn.s) - ((double)dn.m - (double)tot.m) * inv_t + ln_s);
      kl += fabsf(d) < 1.f ? q_rest * excess(d) : q_rest * (d - 1.f) + p;
    } else if (A.tail) {
      kl += p + (float)over;
    } else {
      kl = L.Q == 0.f ? 0.f : kl + p;    // 0: nothing listed
    }
  }
  float loss = a == 1.f ? 0.f : (1.f - a) * T_ * T_ * kl;
  if (a != 0.f) loss += a * (float)(wide_ln_of(tot.s1) - ((double)L.zy - (double)tot.m));
  A.row_loss[r] = loss;
}

// one bit a class of the row (a byte a granule) says that the class is listed; where the listed classes are apart such a class
// leaves the registers as -inf, so that the sums run over the others
template <typename T, int G>
__device__ __forceinline__ void mark_listed(const Row<T>& row, int K, const ListScratch& L, unsigned* bits) {
  constexpr int E = Gran<T>::E;
  const int tid = threadIdx.x;
  for (int w = tid; w < (row.nq + 3) / 4; w += G) bits[w] = 0;
  __syncthreads();
  for (int k = tid; k < K; k += G) {
    const int i = L.idx[k];
    if (i < 0) continue;
    const int q = (i + row.a) / E, e = (i + row.a) % E;
    atomicOr(&bits[q >> 2], 1u << ((q & 3) * 8 + e));
  }
  __syncthreads();
}
template <typename T> struct DropListed {
  const unsigned char* marks;
  __device__ __forceinline__ u32x4_t operator()(u32x4_t d, int q) const {
    constexpr int E = Gran<T>::E;
    const unsigned b = marks[q];
    if (b == 0) return d;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = (b >> e) & 1 ? NINF : Gran<T>::at(d, e);
    return Gran<T>::pack(x);
  }
};

// dz of a class outside the list, from the row's state; two exponentials where the label's softmax has another temperature
struct Dense {
  float md, cT, wT, w1;
  bool two;
  __device__ __forceinline__ Dense(const DistillArgs& A, const RowState& st, float g) {
    md = st.md;
    cT = kLog2e / A.temperature;
    two = A.temperature != 1.f && A.label_weight != 0.f;
    wT = g * (A.temperature == 1.f ? st.wT + st.w1 : st.wT);
    w1 = g * st.w1;
  }
  __device__ __forceinline__ float one(float z) const { return wT * __builtin_amdgcn_exp2f((z - md) * cT); }
  __device__ __forceinline__ float both(float z) const { return fmaf(w1, __builtin_amdgcn_exp2f((z - md) * kLog2e), one(z)); }
};
// the entries of the list and the label, written over the dense values of the classes [lo, hi): one thread per different class
template <typename T, int G>
__device__ __forceinline__ void put_entries(const DistillArgs& A, const Row<T>& row, int r, T* out, int lo, int hi, const Dense& dn,
                                            const ListScratch& L, float g) {
  const RowState st = L.st;
  const int y = A.labels && A.label_weight != 0.f ? (int)L.y : -1;   // in range: st.ok
  for (int k = threadIdx.x; k <= A.K; k += G) {
    const int i = k < A.K ? L.idx[k] : y;
    if (i < 0 || i < lo || i >= hi) continue;
    float q = 0.f;
    bool first = true, listed = false;
    for_entries(L, A.K, i, [&](int j) {
      listed = true;
      first = first && j >= k;
      q += L.q[j];
    });
    if (!first) continue;
    const float z = k < A.K ? L.z[k] : L.zy;
    float x;
    if (listed) {
      x = st.aT * __builtin_amdgcn_exp2f((z - st.m) * dn.cT) - st.cq * q;
      if (A.label_weight != 0.f) x = fmaf(st.a1, __builtin_amdgcn_exp2f((z - st.m) * kLog2e), x);
      x *= g;
    } else {
      x = dn.two ? dn.both(z) : dn.one(z);
    }
    if (i == y) x -= A.label_weight * g;
    Gran<T>::put(out + i, x);
  }
}
// the gradient of the granules [qa, qb), read (again) from memory
template <typename T, int G, int NV>
__device__ __forceinline__ void grad_of_segment(const DistillArgs& A, const Row<T>& row, int r, int qa, int qb, const ListScratch& L) {
  T* out = (T*)A.dlogits + A.out_at.offset(r);
  const Segment<T> sg(row, qa, qb);
  if (L.st.ok == 0.f) {
    map_segment<T, G, NV>(row, sg, out, [](float) { return 0.f; });
    return;
  }
  const Dense dn(A, L.st, L.scale);
  if (dn.two) map_segment<T, G, NV>(row, sg, out, [&](float z) { return dn.both(z); });
  else map_segment<T, G, NV>(row, sg, out, [&](float z) { return dn.one(z); });
  barrier_after_stores();   // the entries are written over the dense values
  put_entries<T, G>(A, row, r, out, row.first_class(qa), row.first_class(qb), dn, L, L.scale);
}

template <int G> __device__ __forceinline__ int count_rows(const int64_t* labels, int64_t ignore, int R, int* sh) {
  int c = 0;
  for (int i = 0; i < R; i += G) c += __popcll(__ballot(i + (int)threadIdx.x < R && labels[i + threadIdx.x] != ignore));
  return block_total<G>(c, sh);
}
__device__ __forceinline__ float scale_of(const DistillArgs& A, int r, int counted) {
  float g = A.count_here ? 1.f / (float)max(counted, 1) : A.inv_count ? A.inv_count[0] : A.host_scale;
  if (A.upstream) g *= A.upstream[A.upstream_rows ? r : 0];
  return g;
}

// Rows of any length, where the listed classes are apart with the marks in dynamic LDS (one byte a granule).  With the gradient the row is read a
// second time.
template <typename T, int G, int NV, bool GRAD>
__global__ __launch_bounds__(G) void distill_rows_kernel(DistillArgs A) {
  __shared__ __align__(16) float sh[4 * (G / 64)];
  __shared__ int cnt[16];
  __shared__ ListScratch L;
  extern __shared__ unsigned bits[];
  const int r = blockIdx.x, tid = threadIdx.x;
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  const Segment<T> sg(row, 0, row.nq);
  const float cT = kLog2e / A.temperature, c1 = kLog2e;
  const bool two = A.temperature != 1.f && A.label_weight != 0.f;
  if (tid < 64) read_list<T>(A, row.p, r, L);
  Sums t;
  if (A.apart) {
    __syncthreads();
    mark_listed<T, G>(row, A.K, L, bits);
    const DropListed<T> drop = {(const unsigned char*)bits};
    t = two ? row_sums<T, G, NV, true, false, !GRAD>(row, sg, cT, c1, drop) : row_sums<T, G, NV, false, false, !GRAD>(row, sg, cT, c1, drop);
  } else {
    t = two ? row_sums<T, G, NV, true, false, !GRAD>(row, sg, cT, c1) : row_sums<T, G, NV, false, false, !GRAD>(row, sg, cT, c1);
  }
  if (!two) t.s1 = t.s;   // with one exponential both sums are the same numbers; for T != 1 without labels s1 is not used
  t = block_sums<G, true, false>(t, cT, two ? c1 : cT, sh);
  const int counted = GRAD && A.count_here ? count_rows<G>(A.labels, A.ignore, A.R, cnt) : 0;
  First first;
  if (tid < 64) first = row_state(A, r, t, L);
  if constexpr (GRAD) {
    if (tid == 0) L.scale = scale_of(A, r, counted);
    __syncthreads();
    grad_of_segment<T, G, NV>(A, row, r, 0, row.nq, L);
  }
  if (tid < 64) row_loss(A, r, first, L);
}

// Loss and gradient of rows of up to G * NV granules, which stay in registers between the sums and the gradient: the row is read
// once.
template <typename T, int NV, bool TWO>
__device__ __forceinline__ Sums held_sums(u32x4_t (&d)[NV], u32x4_t& edge, float c, float c1) {
  constexpr int E = Gran<T>::E;
  Sums r = {NINF, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j <= NV; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) r.m = fmaxf(r.m, Gran<T>::at(j < NV ? d[j < NV ? j : 0] : edge, e));
  const float b = r.m == NINF ? 0.f : r.m;
#pragma unroll
  for (int j = 0; j <= NV; ++j) {
    u32x4_t g = j < NV ? d[j < NV ? j : 0] : edge;
    asm volatile("" : "+v"(g));   // unpacked anew: all the row's classes unpacked at once would not fit the registers
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = Gran<T>::at(g, e) - b;
      r.s += __builtin_amdgcn_exp2f(x * c);
      if (TWO) r.s1 += __builtin_amdgcn_exp2f(x * c1);
    }
  }
  return r;
}
template <typename T, int G, int NV>
__global__ __launch_bounds__(G) void distill_held_kernel(DistillArgs A) {
  constexpr int E = Gran<T>::E;
  __shared__ __align__(16) float sh[4 * (G / 64)];
  __shared__ int cnt[16];
  __shared__ ListScratch L;
  extern __shared__ unsigned bits[];
  const int r = blockIdx.x, tid = threadIdx.x;
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  const Segment<T> sg(row, 0, row.nq);
  const float cT = kLog2e / A.temperature, c1 = kLog2e;
  const bool two = A.temperature != 1.f && A.label_weight != 0.f;
  u32x4_t d[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int q = sg.lo + j * G + tid;
    d[j] = no_class<T>();
    if (q < sg.hi) d[j] = __builtin_nontemporal_load(granule(row, q));
  }
  const int eq = edge_granule(row, sg, tid);
  u32x4_t edge = no_class<T>();
  if (eq >= 0) edge = load_edge(row, eq);
  if (tid < 64) read_list<T>(A, row.p, r, L);
  if (A.apart) {
    __syncthreads();
    mark_listed<T, G>(row, A.K, L, bits);
    const DropListed<T> drop = {(const unsigned char*)bits};
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (sg.lo + j * G + tid < sg.hi) d[j] = drop(d[j], sg.lo + j * G + tid);
    if (eq >= 0) edge = drop(edge, eq);
  }
  Sums t = two ? held_sums<T, NV, true>(d, edge, cT, c1) : held_sums<T, NV, false>(d, edge, cT, c1);
  if (!two) t.s1 = t.s;
  t = block_sums<G, true, false>(t, cT, two ? c1 : cT, sh);
  const int counted = A.count_here ? count_rows<G>(A.labels, A.ignore, A.R, cnt) : 0;
  First first;
  if (tid < 64) first = row_state(A, r, t, L);
  if (tid == 0) L.scale = scale_of(A, r, counted);
  __syncthreads();
  T* out = (T*)A.dlogits + A.out_at.offset(r);
  if (L.st.ok == 0.f || !same_granules(row.p, (const T*)out)) {   // (a gradient that lies otherwise in its granules)
    grad_of_segment<T, G, 1>(A, row, r, 0, row.nq, L);
    if (tid < 64) row_loss(A, r, first, L);
    return;
  }
  const Dense dn(A, L.st, L.scale);
  auto put = [&](auto f) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int q = sg.lo + j * G + tid;
      asm volatile("" : "+v"(d[j]));
      if (q < sg.hi) {
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = f(Gran<T>::at(d[j], e));
        __builtin_nontemporal_store(Gran<T>::pack(x), (u32x4_t*)(out + row.first_class(q)));
      }
    }
    if (eq >= 0) {
      float x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = f(Gran<T>::at(edge, e));
      store_granule(row, out, false, eq, x);
    }
  };
  if (dn.two) put([&](float z) { return dn.both(z); });
  else put([&](float z) { return dn.one(z); });
  barrier_after_stores();   // the entries are written over the dense values
  put_entries<T, G>(A, row, r, out, 0, row.V, dn, L, L.scale);
  if (tid < 64) row_loss(A, r, first, L);   // behind the gradient: its registers are free, and nothing waits for it
}

// the gradient alone, from the state that the loss left
template <typename T, int G, int NV>
__global__ __launch_bounds__(G) void distill_grad_kernel(DistillArgs A) {
  __shared__ ListScratch L;
  const int r = blockIdx.x / A.nseg, seg = blockIdx.x - r * A.nseg, tid = threadIdx.x;
  const Row<T> row((const T*)A.logits, A.at, r, A.V);
  const int qa = seg * A.per, qb = min(qa + A.per, row.nq);
  if (qa >= qb) return;
  if (tid < 64) read_list<T>(A, row.p, r, L);
  if (tid == 0) {
    L.st = *(const RowState*)(A.state + (int64_t)r * kState);
    L.scale = scale_of(A, r, 0);
  }
  __syncthreads();
  grad_of_segment<T, G, NV>(A, row, r, qa, qb, L);
}

// 1 / (rows whose label is not `ignore`), 1 where there are none: their losses are 0
__global__ __launch_bounds__(1024) void distill_count_kernel(const int64_t* labels, int64_t ignore, int R, float* inv) {
  __shared__ int cnt[16];
  const int c = count_rows<1024>(labels, ignore, R, cnt);
  if (threadIdx.x == 0) inv[0] = 1.f / (float)max(c, 1);
}
// the sum of the row losses over a count; with labels that of the counted rows, whose reciprocal is left in inv_count
__global__ __launch_bounds__(1024) void distill_total_kernel(const float* rows, const int64_t* labels, int64_t ignore, int R,
                                                             float host_count, float* inv_count, float* loss) {
  __shared__ double sh[16];
  __shared__ int cnt[16];
  double s = 0.;
  for (int i = threadIdx.x; i < R; i += 1024) s += rows[i];
  s = wave_add(s);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  const int c = labels ? count_rows<1024>(labels, ignore, R, cnt) : 0;
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += sh[w];
    if (labels) inv_count[0] = 1.f / (host_count = (float)max(c, 1));
    loss[0] = (float)(s / host_count);
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
int granule_classes(int dtype) { return dtype == VITM_BF16 ? 8 : 4; }
int cover(int a, int b) { return (a + b - 1) / b; }
// granules of a row, at most
int row_granules(int dtype, int V, int slack) { return cover(V + slack, granule_classes(dtype)); }

// Threads a row, and granules a thread and chunk.  One wave takes a row of up to 256 granules (2048 bf16 classes): 16384 rows of
// 2000 take 16 us so, 45 us with 256 threads each.  Longer rows have a workgroup of 256 threads (2048 rows of 32001: 28 us, with
// 1024 threads 31 us), or, where there are no more rows than CUs, of 1024 from 2048 granules on (64 rows with 20 best: 16384 classes
// 8.5 us with 256 threads and 10.4 us with 1024; 65536 classes 18.7 and 14.1 us).  A row is never cut: one row of 131072 classes
// with 20 best takes one workgroup 16 us, 10 of them for the arithmetic; cut into 64 segments and joined it took 23 us in two
// launches.
struct Plan {
  int G, NV;
};
Plan plan_rows(int R, int nq) {
  for (int nv = 1; nv <= 4; nv *= 2)
    if (nq <= 64 * nv) return {64, nv};
  return {nq <= 2048 || R > vitm_cu_count() ? 256 : 1024, 4};
}
// Whether the sums over a row leave the teacher's classes out: the tail form, which asks for the mass outside the list, and
// temperatures above kFlat.  Left in, they leave the loss off by what ln s is off by, 1e-7 or so, times T^2 (2e-6 of a loss of 4 at
// T = 8, and growing); taken out, 4e-7 up to T = 10^4, but loss and gradient of 4096 x 32000 bf16 take 136 us against 108 us,
// 8192 x 1000 fp32 39 against 33.
constexpr float kFlat = 8.f;
int keeps_apart(int tail, float temperature) { return tail || temperature > kFlat; }
// Threads, chunk, and the cut of a row for kernels whose segments do not depend on each other.
constexpr int kMapSpan = 2048;   // most granules of a segment: 94 us without a limit, 70 us with, at 1024 x 50001 fp32
struct Cut {
  int G, NV, nseg, per;
};
Cut cut_rows(int R, int nq) {
  for (int nv = 1; nv <= 4; nv *= 2)
    if (nq <= 64 * nv) return {64, nv, 1, nq};
  const int64_t want = 4 * (int64_t)vitm_cu_count();   // workgroups
  int nseg = (int)(want / R < 1 ? 1 : want / R);
  nseg = nseg < cover(nq, 256) ? nseg : cover(nq, 256);
  nseg = nseg > cover(nq, kMapSpan) ? nseg : cover(nq, kMapSpan);
  const int per = cover(cover(nq, nseg), 256) * 256;
  return {256, 4, cover(nq, per), per};
}
int slack_of(const void* p, int dtype, int64_t ld_outer, int64_t ld, int inner, int R) {
  const int E = granule_classes(dtype);
  const bool whole = ((uintptr_t)p & 15) == 0 && (R == 1 || (inner == 1 ? ld_outer : ld) % E == 0) && (inner >= R || ld_outer % E == 0);
  return whole ? 0 : E - 1;
}

int check_rows(const char* what, const void* logits, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V) {
  VITM_REQUIRE(logits, "%s: null pointer", what);
  VITM_REQUIRE(dtype == VITM_BF16 || dtype == VITM_F32, "%s: dtype %d unsupported (bf16 or fp32)", what, dtype);
  VITM_REQUIRE(R > 0 && inner > 0 && R <= (1 << 30), "%s: bad number of rows %d (inner %d)", what, R, inner);
  VITM_REQUIRE(V > 0 && V <= kMaxClasses, "%s: %d classes, supported are 1 to %d", what, V, kMaxClasses);
  VITM_REQUIRE(ld >= 0 && ld_outer >= 0, "%s: negative row stride", what);
  VITM_REQUIRE(((uintptr_t)logits & (dtype == VITM_BF16 ? 1 : 3)) == 0, "%s: logits not aligned to their type", what);
  return VITM_OK;
}
int check_out(const char* what, const void* out, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V) {
  const int rc = check_rows(what, out, dtype, ld_outer, ld, inner, R, V);
  if (rc != VITM_OK) return rc;
  const int in = inner < R ? inner : R;   // rows that follow each other at ld
  VITM_REQUIRE((in == 1 || ld >= V) && (inner >= R || ld_outer >= (in - 1) * ld + V), "%s: rows of the gradient overlap", what);
  return VITM_OK;
}
// Whether a row of the gradient and a row of the logits share memory.  The gradient's rows are apart and in ascending order
// (check_out), so a row of the logits meets one of them if it meets the last that starts in front of its own end.  Row by row only
// where the two spans meet at all, as of a gradient interleaved with the logits.
bool rows_meet(const void* logits, const void* out, int dtype, const RowsAt& at, const RowsAt& out_at, int R, int V) {
  const int64_t es = dtype == VITM_BF16 ? 2 : 4;
  const int in = at.inner < R ? at.inner : R, blocks = (R - 1) / in + 1;
  const int64_t span = (blocks - 1) * at.ld_outer + (in - 1) * at.ld + V, out_span = out_at.offset(R - 1) + V;
  const int64_t d = ((intptr_t)logits - (intptr_t)out) / es;   // of the first rows
  if (d >= out_span || d + span <= 0) return false;
  for (int r = 0; r < R; ++r) {
    const int64_t a = d + at.offset(r), last = a + V - 1;   // the row's classes, from the gradient's first
    if (last < 0) continue;
    int64_t o = blocks == 1 ? 0 : last / out_at.ld_outer;
    o = o < blocks - 1 ? o : blocks - 1;
    const int64_t in_block = R - o * in < in ? R - o * in : in;
    int64_t i = in == 1 ? 0 : (last - o * out_at.ld_outer) / out_at.ld;
    i = i < in_block - 1 ? i : in_block - 1;
    if (o * out_at.ld_outer + i * out_at.ld + V > a) return true;
  }
  return false;
}
// The gradient of a distillation, T (p - q), is off by what ln s is off by, times T: by 3e-3 of itself at T = 10^4 (V = 40001).
constexpr float kMinTemperature = 1e-6f, kMaxTemperature = 1e6f, kMaxDistillTemperature = 1e4f;
int check_temperature(const char* what, float t, float most = kMaxTemperature) {
  VITM_REQUIRE(t >= kMinTemperature && t <= most, "%s: temperature %g, supported are %g to %g", what, (double)t,
               (double)kMinTemperature, (double)most);
  return VITM_OK;
}
// a grid holds fewer than 2^32 threads
int check_grid(const char* what, int R, int64_t workgroups, int threads) {
  VITM_REQUIRE(workgroups * threads < (1ll << 32), "%s: %d rows exceed one launch", what, R);
  return VITM_OK;
}

#define SCORES_LAUNCH(kernel, grid, threads, lds, args) hipLaunchKernelGGL((kernel), dim3((unsigned)(grid)), dim3(threads), (lds), st, args)
// a kernel of G threads and chunks of NV granules a thread, for the plans there are
#define SCORES_PLAN(P, CALL)                                                                                            \
  do {                                                                                                                  \
    if (P.G == 64 && P.NV == 1) { CALL(64, 1); }                                                                        \
    else if (P.G == 64 && P.NV == 2) { CALL(64, 2); }                                                                   \
    else if (P.G == 64) { CALL(64, 4); }                                                                                \
    else if (P.G == 256) { CALL(256, 4); }                                                                              \
    else { CALL(1024, 4); }                                                                                             \
  } while (0)

Plan plan_log_probs(int R, int nq, int top_k) {
  if (top_k == 0 && nq <= 16) return {nq <= 4 ? 4 : 16, 1};
  const Plan P = plan_rows(R, nq);
  return top_k > 0 && P.G == 256 && nq > kTopChunks * 1024 ? Plan{1024, 4} : P;   // the cells of a row fit LDS
}
template <typename T> int launch_log_probs(const LogProbsArgs& A, const Plan& P, int nq, hipStream_t st) {
  if (A.K == 0) {
#define LP(G, NV) SCORES_LAUNCH((log_probs_kernel<T, G, NV>), cover(A.R, rows_of_group(G)), G * rows_of_group(G), 0, A)
    if (P.G == 4) LP(4, 1);
    else if (P.G == 16) LP(16, 1);
    else SCORES_PLAN(P, LP);
#undef LP
  } else if (P.G == 64) {
    if (P.NV == 1) SCORES_LAUNCH((log_probs_wave_top_kernel<T, 1>), A.R, 64, 0, A);
    else if (P.NV == 2) SCORES_LAUNCH((log_probs_wave_top_kernel<T, 2>), A.R, 64, 0, A);
    else SCORES_LAUNCH((log_probs_wave_top_kernel<T, 4>), A.R, 64, 0, A);
  } else if (P.G == 256) {
    SCORES_LAUNCH((log_probs_top_kernel<T, 256, 4>), A.R, 256, cover(nq, 1024) * 1024, A);
  } else {
    VITM_LDS_OPTIN((log_probs_top_kernel<T, 1024, 4>), kTopChunks * 4096, "vitm_log_probs");
    SCORES_LAUNCH((log_probs_top_kernel<T, 1024, 4>), A.R, 1024, cover(nq, 4096) * 4096, A);
  }
  return VITM_OK;
}
template <typename T> void launch_log_probs_bwd(const LogProbsBwdArgs& A, const Cut& C, hipStream_t st) {
#define LPB(G, NV) SCORES_LAUNCH((log_probs_bwd_kernel<T, G, NV>), (int64_t)A.R * C.nseg, G, 0, A)
  if (C.G == 64 && C.NV == 1) LPB(64, 1);
  else if (C.G == 64 && C.NV == 2) LPB(64, 2);
  else if (C.G == 64) LPB(64, 4);
  else LPB(256, 4);
#undef LPB
}
constexpr int kMarks = 131072;   // most granules of a row: the marks of the tail form
template <typename T, bool GRAD> int launch_distill_rows(const DistillArgs& A, const Plan& P, int nq, hipStream_t st) {
  const int lds = A.apart ? cover(nq, 4) * 4 : 0;
#define DS(G, NV)                                                                                                       \
  if (lds > 32768) VITM_LDS_OPTIN((distill_rows_kernel<T, G, NV, GRAD>), kMarks, "vitm_distill");                       \
  SCORES_LAUNCH((distill_rows_kernel<T, G, NV, GRAD>), A.R, G, lds, A)
  if constexpr (GRAD) {   // shorter rows are held
    if (P.G == 256) { DS(256, 4); }
    else { DS(1024, 4); }
  } else {
    SCORES_PLAN(P, DS);
  }
#undef DS
  return VITM_OK;
}
// Loss and gradient in one kernel.  Rows of up to 1024 granules stay in registers.  Longer ones do too, up to 8192 granules, where
// no classes have to be taken out of the sums (4096 x 32000 bf16: 110 us against 135 us with a second reading; 2048 x 32000 fp32:
// 105 against 128); with the marks of the listed classes the walk is the faster one for long lists (4096 x 50001 bf16: 222 us
// against 246 us held with 64 entries, 248 against 344 with 128, 211 against 203 with 20).  A row of
// 16384 granules fills the registers of a CU, and nothing runs beside its phases: 640 us against 500 us at 4096 x 131072 bf16.
Plan plan_distill_fused(int R, int nq, bool apart) {   // NV = 0: a walk by launch_distill_rows
  if (nq <= 1024 || (!apart && nq <= 8192)) {
    if (nq <= 256) return {64, nq <= 64 ? 1 : nq <= 128 ? 2 : 4};
    if (nq <= 4096) return {256, nq <= 1024 ? 4 : nq <= 2048 ? 8 : 16};
    return {512, 16};
  }
  return {plan_rows(R, nq).G, 0};
}
template <typename T> int launch_distill_fused(const DistillArgs& A, const Plan& P, int nq, hipStream_t st) {
  if (P.NV == 0) return launch_distill_rows<T, true>(A, P, nq, st);
  const int lds = A.apart ? cover(nq, 4) * 4 : 0;
#define DH(G, NV) SCORES_LAUNCH((distill_held_kernel<T, G, NV>), A.R, G, lds, A)
  if (P.G == 64 && P.NV == 1) DH(64, 1);
  else if (P.G == 64 && P.NV == 2) DH(64, 2);
  else if (P.G == 64) DH(64, 4);
  else if (P.G == 512) DH(512, 16);
  else if (P.NV == 4) DH(256, 4);
  else if (P.NV == 8) DH(256, 8);
  else DH(256, 16);
#undef DH
  return VITM_OK;
}
template <typename T> void launch_distill_grad(const DistillArgs& A, const Cut& C, hipStream_t st) {
#define DG(G, NV) SCORES_LAUNCH((distill_grad_kernel<T, G, NV>), (int64_t)A.R * C.nseg, G, 0, A)
  if (C.G == 64 && C.NV == 1) DG(64, 1);
  else if (C.G == 64 && C.NV == 2) DG(64, 2);
  else if (C.G == 64) DG(64, 4);
  else DG(256, 4);
#undef DG
}

}  // namespace

extern "C" int vitm_scores_max_top(void) { return kMaxTop; }
extern "C" int vitm_scores_max_classes(void) { return kMaxClasses; }

extern "C" int vitm_log_probs(const void* logits, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V,
                              float temperature, const int64_t* targets, int n_targets, int64_t ignore_index, int top_k,
                              float* logprobs, float* lse, float* entropy, float* top_logprobs, int64_t* top_indices,
                              float* stats, vitm_stream_t stream) {
  const int rc = check_rows("vitm_log_probs", logits, dtype, ld_outer, ld, inner, R, V);
  if (rc != VITM_OK) return rc;
  if (check_temperature("vitm_log_probs", temperature) != VITM_OK) return VITM_EINVAL;
  VITM_REQUIRE(n_targets >= 0 && n_targets <= kMaxTop, "vitm_log_probs: %d targets a row, supported are 0 to %d", n_targets, kMaxTop);
  VITM_REQUIRE(n_targets == 0 || (targets && logprobs), "vitm_log_probs: null pointer");
  VITM_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= V, "vitm_log_probs: top_k %d, supported are 0 to %d and at most the %d classes",
               top_k, kMaxTop, V);
  VITM_REQUIRE(top_k == 0 || (top_logprobs && top_indices), "vitm_log_probs: null pointer");
  LogProbsArgs A = {};
  A.logits = logits;
  A.at = {ld_outer, ld, inner};
  A.R = R; A.V = V;
  A.inv_t = 1.f / temperature;
  A.targets = targets; A.G = n_targets; A.ignore = ignore_index; A.K = top_k;
  A.logprobs = logprobs; A.lse = lse; A.entropy = entropy; A.top_lp = top_logprobs; A.top_idx = top_indices; A.stats = stats;
  const int nq = row_granules(dtype, V, slack_of(logits, dtype, ld_outer, ld, inner, R));
  const Plan P = plan_log_probs(R, nq, top_k);
  // short rows, several to a wave, are held to the number that a wave each would allow
  if (check_grid("vitm_log_probs", R, R, P.G < 64 ? 64 : P.G) != VITM_OK) return VITM_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  const int rl = dtype == VITM_BF16 ? launch_log_probs<bf16_t>(A, P, nq, st) : launch_log_probs<float>(A, P, nq, st);
  if (rl != VITM_OK) return rl;
  VITM_CHECK_LAUNCH("vitm_log_probs");
  return VITM_OK;
}

extern "C" int vitm_log_probs_bwd(const void* logits, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V,
                                  float temperature, const int64_t* targets, int n_targets, int64_t ignore_index,
                                  const int64_t* top_indices, int top_k, const float* stats, const float* entropy,
                                  const float* g_logprobs, const float* g_lse, const float* g_entropy, const float* g_top,
                                  void* dlogits, int64_t ldd_outer, int64_t ldd, vitm_stream_t stream) {
  int rc = check_rows("vitm_log_probs_bwd", logits, dtype, ld_outer, ld, inner, R, V);
  if (rc == VITM_OK) rc = check_out("vitm_log_probs_bwd", dlogits, dtype, ldd_outer, ldd, inner, R, V);
  if (rc != VITM_OK) return rc;
  if (check_temperature("vitm_log_probs_bwd", temperature) != VITM_OK) return VITM_EINVAL;
  VITM_REQUIRE(stats, "vitm_log_probs_bwd: null pointer");
  VITM_REQUIRE(n_targets >= 0 && n_targets <= kMaxTop && top_k >= 0 && top_k <= kMaxTop, "vitm_log_probs_bwd: %d targets, top_k %d: supported are 0 to %d",
               n_targets, top_k, kMaxTop);
  VITM_REQUIRE(!g_logprobs || targets, "vitm_log_probs_bwd: null pointer");
  VITM_REQUIRE(!g_top || top_indices, "vitm_log_probs_bwd: null pointer");
  VITM_REQUIRE(!g_entropy || entropy, "vitm_log_probs_bwd: null pointer");
  VITM_REQUIRE(!rows_meet(logits, dlogits, dtype, {ld_outer, ld, inner}, {ldd_outer, ldd, inner}, R, V),
               "vitm_log_probs_bwd: logits and gradient in the same memory");
  const Cut C = cut_rows(R, row_granules(dtype, V, slack_of(logits, dtype, ld_outer, ld, inner, R)));
  if (check_grid("vitm_log_probs_bwd", R, (int64_t)R * C.nseg, C.G) != VITM_OK) return VITM_EINVAL;
  LogProbsBwdArgs A = {};
  A.logits = logits;
  A.at = {ld_outer, ld, inner};
  A.R = R; A.V = V; A.nseg = C.nseg; A.per = C.per;
  A.inv_t = 1.f / temperature;
  A.targets = targets; A.G = n_targets; A.ignore = ignore_index; A.top_idx = top_indices; A.K = top_k;
  A.stats = stats; A.entropy = entropy;
  A.g_logprobs = g_logprobs; A.g_lse = g_lse; A.g_entropy = g_entropy; A.g_top = g_top;
  A.dlogits = dlogits;
  A.out_at = {ldd_outer, ldd, inner};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == VITM_BF16) launch_log_probs_bwd<bf16_t>(A, C, st);
  else launch_log_probs_bwd<float>(A, C, st);
  VITM_CHECK_LAUNCH("vitm_log_probs_bwd");
  return VITM_OK;
}

extern "C" int vitm_distill_state_floats(void) { return kState; }

namespace {
int distill_args(const char* what, DistillArgs& A, const void* logits, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V,
                 float temperature, float label_weight, int tail, const float* teacher, const int64_t* indices, int K,
                 const int64_t* labels, int64_t ignore_index) {
  const int rc = check_rows(what, logits, dtype, ld_outer, ld, inner, R, V);
  if (rc != VITM_OK) return rc;
  if (check_temperature(what, temperature, kMaxDistillTemperature) != VITM_OK) return VITM_EINVAL;
  VITM_REQUIRE(label_weight >= 0.f && label_weight <= 1.f, "%s: label weight must lie in [0, 1]", what);
  VITM_REQUIRE(label_weight == 0.f || labels, "%s: a label weight needs labels", what);
  VITM_REQUIRE(teacher && indices, "%s: null pointer", what);
  VITM_REQUIRE(K > 0 && K <= kMaxTop, "%s: a teacher's list of %d classes, supported are 1 to %d", what, K, kMaxTop);
  A.logits = logits;
  A.at = {ld_outer, ld, inner};
  A.R = R; A.V = V;
  A.temperature = temperature; A.label_weight = label_weight; A.tail = tail ? 1 : 0;
  A.apart = keeps_apart(A.tail, temperature);
  A.teacher = teacher; A.indices = indices; A.K = K;
  A.labels = labels; A.ignore = ignore_index;
  A.host_scale = 1.f;
  return VITM_OK;
}
}  // namespace

extern "C" int vitm_distill(const void* logits, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V, float temperature,
                            float label_weight, int tail, const float* teacher_logprobs, const int64_t* teacher_indices, int K,
                            const int64_t* labels, int64_t ignore_index, int reduction, float* row_loss, float* loss,
                            float* inv_count, float* state, void* dlogits, int64_t ldd_outer, int64_t ldd,
                            vitm_stream_t stream) {
  DistillArgs A = {};
  const int rc = distill_args("vitm_distill", A, logits, dtype, ld_outer, ld, inner, R, V, temperature, label_weight, tail,
                              teacher_logprobs, teacher_indices, K, labels, ignore_index);
  if (rc != VITM_OK) return rc;
  VITM_REQUIRE(row_loss, "vitm_distill: null pointer");
  VITM_REQUIRE(reduction >= VITM_REDUCE_NONE && reduction <= VITM_REDUCE_SUM, "vitm_distill: unknown reduction %d", reduction);
  VITM_REQUIRE(reduction == VITM_REDUCE_NONE || loss, "vitm_distill: null pointer");
  VITM_REQUIRE(reduction != VITM_REDUCE_MEAN || !labels || inv_count, "vitm_distill: the mean over labelled rows needs inv_count");
  if (dlogits) {
    const int rd = check_out("vitm_distill", dlogits, dtype, ldd_outer, ldd, inner, R, V);
    if (rd != VITM_OK) return rd;
    VITM_REQUIRE(!rows_meet(logits, dlogits, dtype, {ld_outer, ld, inner}, {ldd_outer, ldd, inner}, R, V),
                 "vitm_distill: logits and gradient in the same memory");
  }
  const int nq = row_granules(dtype, V, slack_of(logits, dtype, ld_outer, ld, inner, R));
  const Plan P = dlogits ? plan_distill_fused(R, nq, A.apart) : plan_rows(R, nq);
  if (check_grid("vitm_distill", R, R, P.G) != VITM_OK) return VITM_EINVAL;
  A.row_loss = row_loss;
  A.state = state;
  A.dlogits = dlogits;
  A.out_at = {ldd_outer, ldd, inner};
  hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == VITM_BF16;
  if (reduction == VITM_REDUCE_MEAN) {
    A.host_scale = 1.f / (float)R;
    if (labels && dlogits) {   // the gradient needs the number of counted rows; up to 1024 labels a workgroup counts by itself
      if (R <= 1024) {
        A.count_here = 1;
      } else {
        hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(1024), 0, st, labels, ignore_index, R, inv_count);
        A.inv_count = inv_count;
      }
    }
  }
  const int rl = dlogits ? (bf ? launch_distill_fused<bf16_t>(A, P, nq, st) : launch_distill_fused<float>(A, P, nq, st))
                         : (bf ? launch_distill_rows<bf16_t, false>(A, P, nq, st) : launch_distill_rows<float, false>(A, P, nq, st));
  if (rl != VITM_OK) return rl;
  if (reduction != VITM_REDUCE_NONE)
    hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(1024), 0, st, (const float*)row_loss,
                       reduction == VITM_REDUCE_MEAN ? labels : nullptr, ignore_index, R, reduction == VITM_REDUCE_MEAN ? (float)R : 1.f,
                       inv_count, loss);
  VITM_CHECK_LAUNCH("vitm_distill");
  return VITM_OK;
}

extern "C" int vitm_distill_bwd(const void* logits, int dtype, int64_t ld_outer, int64_t ld, int inner, int R, int V, float temperature,
                                float label_weight, int tail, const float* teacher_logprobs, const int64_t* teacher_indices, int K,
                                const int64_t* labels, int64_t ignore_index, int reduction, const float* inv_count, const float* state,
                                const float* upstream, void* dlogits, int64_t ldd_outer, int64_t ldd, vitm_stream_t stream) {
  DistillArgs A = {};
  int rc = distill_args("vitm_distill_bwd", A, logits, dtype, ld_outer, ld, inner, R, V, temperature, label_weight, tail,
                        teacher_logprobs, teacher_indices, K, labels, ignore_index);
  if (rc == VITM_OK) rc = check_out("vitm_distill_bwd", dlogits, dtype, ldd_outer, ldd, inner, R, V);
  if (rc != VITM_OK) return rc;
  VITM_REQUIRE(state && upstream, "vitm_distill_bwd: null pointer");
  VITM_REQUIRE(reduction >= VITM_REDUCE_NONE && reduction <= VITM_REDUCE_SUM, "vitm_distill_bwd: unknown reduction %d", reduction);
  VITM_REQUIRE(reduction != VITM_REDUCE_MEAN || !labels || inv_count, "vitm_distill_bwd: the mean over labelled rows needs inv_count");
  VITM_REQUIRE(!rows_meet(logits, dlogits, dtype, {ld_outer, ld, inner}, {ldd_outer, ldd, inner}, R, V),
               "vitm_distill_bwd: logits and gradient in the same memory");
  const Cut C = cut_rows(R, row_granules(dtype, V, slack_of(logits, dtype, ld_outer, ld, inner, R)));
  if (check_grid("vitm_distill_bwd", R, (int64_t)R * C.nseg, C.G) != VITM_OK) return VITM_EINVAL;
  A.nseg = C.nseg; A.per = C.per;
  A.state = (float*)state;
  A.upstream = upstream;
  A.upstream_rows = reduction == VITM_REDUCE_NONE;
  if (reduction == VITM_REDUCE_MEAN) {
    A.host_scale = 1.f / (float)R;
    A.inv_count = labels ? inv_count : nullptr;
  }
  A.dlogits = dlogits;
  A.out_at = {ldd_outer, ldd, inner};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == VITM_BF16) launch_distill_grad<bf16_t>(A, C, st);
  else launch_distill_grad<float>(A, C, st);
  VITM_CHECK_LAUNCH("vitm_distill_bwd");
  return VITM_OK;
}
