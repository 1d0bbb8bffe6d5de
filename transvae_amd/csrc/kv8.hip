// Keys and values held in 8 bits: store (quantise rows as they are written), load (read them back) and attention over them.
//
// A cache is a pool of pages.  One page holds `page` tokens of every head: codes (n_pages, h, page, dk), one byte each, in
// e4m3 (1 sign, 4 exponent, 3 mantissa bits, largest 448, no infinity), and one exponent byte per (page, head), bias 127:
//     value = code * 2^(exponent - 127).
// Why a power of two: e4m3 is itself floating point, so a finer scale would not add precision inside its normal range (2^-6 ..
// 448), while a power of two makes scaling, un-scaling and re-scaling exact: a code is ONE rounding of the value it was made
// from, and pulling the rows of a page down to a larger exponent only rounds what drops into the subnormals.
// The exponent is the smallest with amax * 2^-e <= 448, held to [-100, 119] so that no value of a cache can overflow fp32.
#include "common.h"

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int E_BIAS = 127, E_MIN = 27, E_MAX = 246;
constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;              // of 256 threads: a grid counts its threads in 32 bits

struct F16 { _Float16 v; };
struct B16 { uint16_t v; };

// 16 bytes of a row as they are, and as floats
template <typename T> struct Raw {
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  __device__ inline void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ inline void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ inline void values(float (&x)[N]) const;
  // what was unpacked from w so far is not kept: a second look unpacks again instead of holding 8 registers for 4
  __device__ inline void forget() { asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w)); }
};
template <> __device__ inline void Raw<float>::values(float (&x)[4]) const {
  x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
}
template <> __device__ inline void Raw<B16>::values(float (&x)[8]) const {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
}
template <> __device__ inline void Raw<F16>::values(float (&x)[8]) const {
  _Float16 h[8];
  *reinterpret_cast<uint4*>(h) = w;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ inline void load4(const float* p, float (&x)[4]) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
  }
  static __device__ inline void store4(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
  static __device__ inline void put(float* p, float x) { *p = x; }
};
template <> struct Elem<B16> {
  static __device__ inline void load4(const B16* p, float (&x)[4]) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(t.x << 16); x[1] = __uint_as_float(t.x & 0xFFFF0000u);
    x[2] = __uint_as_float(t.y << 16); x[3] = __uint_as_float(t.y & 0xFFFF0000u);
  }
  static __device__ inline uint16_t cvt(float x) {         // round to nearest even; NaN stays NaN
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
  }
  static __device__ inline void put(B16* p, float x) { p->v = cvt(x); }
  static __device__ inline void store4(B16* p, const float (&x)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(cvt(x[0]) | (uint32_t)cvt(x[1]) << 16, cvt(x[2]) | (uint32_t)cvt(x[3]) << 16);
  }
};
template <> struct Elem<F16> {
  static __device__ inline void load4(const F16* p, float (&x)[4]) {
    _Float16 h[4];
    *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)h[i];
  }
  static __device__ inline void put(F16* p, float x) { p->v = (_Float16)x; }
  static __device__ inline void store4(F16* p, const float (&x)[4]) {
    _Float16 h[4] = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
  }
};

__device__ inline float exp_scale(int e) { return __uint_as_float((uint32_t)e << 23); }          // 2^(e - 127)
__device__ inline float inv_scale(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }  // 2^(127 - e)

// Magnitudes are compared as whole numbers (the bits without the sign): one comparison also finds infinities and NaN, which
// are rare enough for a second look.
constexpr uint32_t INF_BITS = 0x7F800000u;
__device__ inline uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ inline uint32_t finite_magnitude(float x) {
  const uint32_t u = magnitude(x);
  return u < INF_BITS ? u : 0u;
}
// stored exponent for a largest magnitude (448 = 1.75 * 2^8: a mantissa above 1.75 carries into the exponent)
__device__ inline int need_exp(uint32_t top) {
  const int e = (int)((top + 0x1FFFFFu) >> 23) - 8;
  return e < E_MIN ? E_MIN : e > E_MAX ? E_MAX : e;
}
__device__ inline uint32_t pack4(const float (&y)[4]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  return w;
}
// codes of four values.  `odd`: the page's rows hold a non-finite value (NaN is stored: the format has no infinity, and a saturated
// one would read back as an ordinary number) or take the largest exponent (which cannot hold every float: those saturate).
// Otherwise the scale itself keeps every value within +-448.
__device__ inline uint32_t encode4(const float (&x)[4], float inv, bool odd) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] * inv;
  if (odd) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = magnitude(x[i]) >= INF_BITS ? __uint_as_float(0x7FC00000u) : fminf(fmaxf(y[i], -448.f), 448.f);
  }
  return pack4(y);
}
__device__ inline void unpack4(uint32_t w, float (&x)[4]) {
  const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
}

// where a sequence's pages are
struct Pages {
  const int32_t* table;      // (n, per_seq) page ids, or NULL: page b * per_seq + i
  int per_seq, n_pages;
  __device__ inline int at(int b, int slot) const {
    const int p = table ? table[(size_t)b * per_seq + slot] : b * per_seq + slot;
    return p >= 0 && p < n_pages ? p : -1;                   // -1: no such page, nothing is read or written
  }
};
// The same in two halves and without a branch, so that a lookup is in flight while something else is computed: ask() loads a
// table entry (any one where there is no table: `spare` is readable memory), page() makes the id of it.
struct PageRow {
  const int32_t* row;
  int base, last, n_pages;
  bool tabled;
  __device__ inline PageRow(const Pages& p, int b, const void* spare)
      : row(p.table ? p.table + (size_t)b * p.per_seq : reinterpret_cast<const int32_t*>(spare)), base(b * p.per_seq), last(p.per_seq - 1),
        n_pages(p.n_pages), tabled(p.table != nullptr) {}
  __device__ inline int ask(int slot) const { return row[tabled ? (slot < last ? slot : last) : 0]; }
  __device__ inline int page(int raw, int slot, bool want) const {
    const int p = tabled ? raw : base + slot;
    return want && p >= 0 && p < n_pages ? p : -1;
  }
};

template <int CTRL> __device__ inline float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
// sum / maximum over groups of N neighbouring lanes (every lane of a group gets it): quad permutes, mirrors of 8 and 16, then swaps
template <int N> __device__ inline float group_sum(float x) {
  if (N >= 2) x += dpp<0xB1>(x);
  if (N >= 4) x += dpp<0x4E>(x);
  if (N >= 8) x += dpp<0x141>(x);
  if (N >= 16) x += dpp<0x140>(x);
  return x;
}
template <int CTRL> __device__ inline uint32_t dpp(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true); }
template <int N> __device__ inline uint32_t group_max(uint32_t x) {
  if (N >= 2) x = max(x, dpp<0xB1>(x));
  if (N >= 4) x = max(x, dpp<0x4E>(x));
  if (N >= 8) x = max(x, dpp<0x141>(x));
  if (N >= 16) x = max(x, dpp<0x140>(x));
  if (N >= 32) x = max(x, (uint32_t)__shfl_xor((int)x, 16, 64));
  if (N >= 64) x = max(x, (uint32_t)__shfl_xor((int)x, 32, 64));
  return x;
}

// x / d for x < 2^31 and a divisor that the host knows: with 2^(s-1) < d <= 2^s, m = ceil(2^(31+s) / d) fits 32 bits and
// (x m) >> (31 + s) is exact (m exceeds 2^(31+s) / d by less than 1, x times that is less than 2^31 <= 2^(31+s) / d)
struct Divisor {
  uint32_t d, m, s;
  explicit Divisor(uint32_t by) : d(by), m(0), s(0) {
    while ((1u << s) < by) ++s;
    m = (uint32_t)((((uint64_t)1 << (31 + s)) + by - 1) / by);
  }
  __device__ inline uint32_t div(uint32_t x) const { return (uint32_t)(((uint64_t)x * m) >> (31 + s)); }
};

// ------------------------------------------------------------------------------------------------ store
struct StoreArgs {
  const void* src[2];
  int64_t ldb[2], ldt[2], ldh[2];
  uint8_t* codes[2];
  uint8_t* exps[2];
  Pages pages;
  const int32_t* start;
  const int32_t* count;
  Divisor by_h;
  int start0, n, T, h, page, slots;
};

// the rows in front of the new ones, from their old scale to a larger one: each value is rounded again; N codes a lane
template <int N>
__device__ inline void rescale_rows(uint8_t* dst, int r0, int dk, int step, int old, int e) {
  int d = old - e;
  d = d > -40 ? d : -40;                                                // beyond that everything rounds to zero
  const float f = exp_scale(E_BIAS + d);
  for (int i = 0; i < r0; i += step) {
    uint32_t* w = reinterpret_cast<uint32_t*>(dst + (size_t)i * dk);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      float x[4];
      unpack4(w[j], x);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] *= f;
      w[j] = pack4(x);
    }
  }
}

template <typename T> __device__ inline uint32_t top_of(const Raw<T>& r, bool strange) {
  float x[Raw<T>::N];
  r.values(x);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < Raw<T>::N; ++i) top = max(top, strange ? finite_magnitude(x[i]) : magnitude(x[i]));
  return top;
}
template <typename T> __device__ inline void put_codes(uint8_t* dst, const Raw<T>& r, float inv, bool odd) {
  float x[Raw<T>::N];
  r.values(x);
  uint32_t w[Raw<T>::N / 4];
#pragma unroll
  for (int i = 0; i < Raw<T>::N; i += 4) {
    const float y[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
    w[i / 4] = encode4(y, inv, odd);
  }
  if (Raw<T>::N == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
  else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[Raw<T>::N / 4 - 1]);
}

// A few rows a sequence (T <= 4: a decode step, drafted tokens).  The lanes that one row's 16-byte pieces take hold the K and
// the V rows of one (sequence, head) in registers: their maxima, the page's exponents, the codes.  Bound by latency more than
// by the rows' bytes, hence both sides in one thread (16384 x 4 heads x 64 fp32, one row: a wave per (sequence, head, side) 69 us,
// these lane groups with a side each 16 us, with both 12 us = 3.4 TB/s).
template <typename T, int DK>
__global__ __launch_bounds__(256) void kv8_append_kernel(StoreArgs a) {
  constexpr int N = Raw<T>::N, LPR = DK / N;
  const int sub = threadIdx.x % LPR;
  const uint32_t unit = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (unit >= (uint32_t)a.n * a.h) return;
  const int b = (int)a.by_h.div(unit), head = (int)unit - b * a.h;
  const int64_t beg = a.start ? a.start[b] : a.start0;
  int cnt = a.count ? a.count[b] : a.T;
  cnt = cnt < a.T ? cnt : a.T;
  if (beg < 0 || cnt <= 0) return;
  Raw<T> x[2][4];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const T* src = reinterpret_cast<const T*>(a.src[side]) + (int64_t)b * a.ldb[side] + (int64_t)head * a.ldh[side] + N * sub;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t < cnt) x[side][t].load(src + t * a.ldt[side]);
      else x[side][t].zero();
    }
  }
  const int shift = 31 - __clz(a.page);
  for (int t0 = 0; t0 < cnt;) {                                         // page after page: two at most
    const int64_t slot = (beg + t0) >> shift;
    if (slot >= a.pages.per_seq) return;
    const int r0 = (int)((beg + t0) & (a.page - 1)), t1 = cnt - t0 < a.page - r0 ? cnt : t0 + a.page - r0;
    const int id = a.pages.at(b, (int)slot);
    if (id >= 0) {
      const size_t ph = (size_t)id * a.h + head;
      int old[2];
#pragma unroll
      for (int side = 0; side < 2; ++side) old[side] = r0 > 0 ? a.exps[side][ph] : 0;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        uint8_t* dst = a.codes[side] + ph * a.page * DK + N * sub;
        uint32_t top = 0;
        bool strange = false;
        for (int look = 0; look < 2; ++look) {                          // a second time only where something is not finite
          top = 0;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if (t >= t0 && t < t1) top = max(top, top_of(x[side][t], strange));
            x[side][t].forget();
          }
          top = group_max<LPR>(top);
          if (top < INF_BITS) break;
          strange = true;
        }
        int e = need_exp(top);
        if (old[side] >= e) e = old[side] < E_MAX ? old[side] : E_MAX;
        else if (r0 > 0) rescale_rows<N>(dst, r0, DK, 1, old[side], e);
        const float inv = inv_scale(e);
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (t >= t0 && t < t1) put_codes(dst + (size_t)(r0 + t - t0) * DK, x[side][t], inv, strange || e == E_MAX);
        if (sub == 0) a.exps[side][ph] = (uint8_t)e;
      }
    }
    t0 = t1;
  }
}

// Many rows a sequence: TPU threads per (sequence, touched page, head), K or V.  A thread keeps its first KEEP 16-byte pieces in
// registers as they came, so the rows are read once; a wave a page where eight of them suffice, a block of four else.  KEEP follows
// the page: pieces that are never there cost their instructions and registers all the same (264 x 968 rows of 5 heads: 16 x 32
// bf16 a page, 1 / 16 pieces 64 / 166 us; 32 x 64 fp32, 8 / 16 165 / 222; 64 x 128 bf16, four waves with 4 / one with 16 179 / 213).
template <typename T, int DK, int TPU, int KEEP>
__global__ __launch_bounds__(256) void kv8_store_kernel(StoreArgs a) {
  constexpr int N = Raw<T>::N, LPR = DK / N, RPI = TPU / LPR;                   // values a piece, lanes a row, rows a step
  __shared__ uint32_t red[4];
  const int tid = threadIdx.x % TPU, side = blockIdx.y;
  uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * (256 / TPU) + threadIdx.x / TPU);
  const int head = (int)(unit % a.h);
  unit /= a.h;
  const int slot = (int)(unit % a.slots), b = (int)(unit / a.slots);
  if (b >= a.n) return;                                                 // whole units leave: a block of one unit leaves together
  const int64_t beg = a.start ? a.start[b] : a.start0;
  int cnt = a.count ? a.count[b] : a.T;
  cnt = cnt < a.T ? cnt : a.T;
  if (beg < 0 || cnt <= 0) return;
  const int shift = 31 - __clz(a.page);
  const int64_t pslot = (beg >> shift) + slot;
  if (pslot >= a.pages.per_seq) return;
  const int64_t p0 = pslot << shift;                                    // first position of the page
  const int r0 = (int)(beg > p0 ? beg - p0 : 0);                        // rows [r0, r1) of the page are new
  const int64_t left = beg + cnt - p0;
  const int r1 = (int)(left < a.page ? left : a.page);
  if (r0 >= r1) return;
  const int id = a.pages.at(b, (int)pslot);
  if (id < 0) return;
  const int sub = tid % LPR, rg = tid / LPR;
  const T* src = reinterpret_cast<const T*>(a.src[side]) + (int64_t)b * a.ldb[side] + (int64_t)head * a.ldh[side] + N * sub + (p0 - beg) * a.ldt[side];
  const size_t ph = (size_t)id * a.h + head;
  uint8_t* dst = a.codes[side] + ph * a.page * DK + N * sub;
  const int old = r0 > 0 ? a.exps[side][ph] : 0;
  Raw<T> x[KEEP];
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int r = r0 + rg + k * RPI;
    if (r < r1) x[k].load(src + r * a.ldt[side]);
    else x[k].zero();
  }
  uint32_t top = 0;
  bool strange = false;
  for (int look = 0; look < 2; ++look) {                                // a second time only where something is not finite
    top = 0;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
      top = max(top, top_of(x[k], strange));
      x[k].forget();
    }
    for (int r = r0 + rg + KEEP * RPI; r < r1; r += RPI) {
      Raw<T> y;
      y.load(src + r * a.ldt[side]);
      top = max(top, top_of(y, strange));
    }
    top = group_max<64>(top);
    if (TPU == 256) {
      __syncthreads();                                                  // also: every thread has read the old exponent
      if ((tid & 63) == 0) red[tid >> 6] = top;
      __syncthreads();
      top = max(max(red[0], red[1]), max(red[2], red[3]));
    }
    if (top < INF_BITS) break;
    strange = true;
  }
  int e = need_exp(top);
  if (old >= e) e = old < E_MAX ? old : E_MAX;
  else if (rg < r0) rescale_rows<N>(dst + (size_t)rg * DK, r0 - rg, DK, RPI, old, e);
  const float inv = inv_scale(e);
  const bool odd = strange || e == E_MAX;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int r = r0 + rg + k * RPI;
    if (r < r1) put_codes(dst + (size_t)r * DK, x[k], inv, odd);
  }
  for (int r = r0 + rg + KEEP * RPI; r < r1; r += RPI) {
    Raw<T> y;
    y.load(src + r * a.ldt[side]);
    put_codes(dst + (size_t)r * DK, y, inv, odd);
  }
  if (tid == 0) a.exps[side][ph] = (uint8_t)e;
}

// ------------------------------------------------------------------------------------------------ load
struct LoadArgs {
  const uint8_t* codes[2];
  const uint8_t* exps[2];
  void* out[2];
  Pages pages;
  const int32_t* start;
  const int32_t* count;
  Divisor by_T, by_h;
  uint32_t total;
  int start0, T, h, page;
};

// A thread makes four times 16 bytes of the result (4 or 8 values), a block's width apart and all in flight together.  Blocks go
// through the result in its own order: writes are three quarters of the traffic and more, and are whole runs of all heads (24 x 4000
// x 8 x 128 bf16: 118 us so, 128 us in the order of the pages).  The result is written past the caches: kept in them it only
// delays the end of the launch (500 x 127 x 4 x 64 fp32: 40 us through the caches, 25 us past them).
template <typename T, int DK>
__global__ __launch_bounds__(256) void kv8_load_kernel(LoadArgs a) {
  constexpr int N = 16 / sizeof(T), LPR = DK / N, U = 4;
  const int side = blockIdx.y;
  const int shift = 31 - __clz(a.page);
  const uint32_t i0 = blockIdx.x * (256 * U) + threadIdx.x;
  int id[U];
  uint32_t b[U], head[U], t[U], sub[U];
  int64_t pos[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = i0 + 256 * u < a.total ? i0 + 256 * u : 0;
    const uint32_t row = i / LPR, bt = a.by_h.div(row);
    sub[u] = i % LPR;
    head[u] = row - bt * a.h;
    b[u] = a.by_T.div(bt);
    t[u] = bt - b[u] * a.T;
    pos[u] = (int64_t)(a.start ? a.start[b[u]] : a.start0) + t[u];
    const int cnt = a.count ? a.count[b[u]] : a.T;
    const bool live = (int)t[u] < cnt && pos[u] >= 0 && (pos[u] >> shift) < a.pages.per_seq;
    id[u] = live ? a.pages.at((int)b[u], (int)(pos[u] >> shift)) : -1;
  }
  uint32_t w[U][N / 4];
  int e[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t ph = (size_t)(id[u] < 0 ? 0 : id[u]) * a.h + head[u];
    const uint8_t* p = a.codes[side] + (ph * a.page + ((int)pos[u] & (a.page - 1))) * DK + N * sub[u];
    w[u][0] = w[u][N / 4 - 1] = 0;
    e[u] = E_BIAS;
    if (id[u] >= 0) {
      if (N == 4) w[u][0] = *reinterpret_cast<const uint32_t*>(p);
      else *reinterpret_cast<uint2*>(w[u]) = *reinterpret_cast<const uint2*>(p);
      e[u] = a.exps[side][ph];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (i0 + 256 * u >= a.total) continue;
    const float s = exp_scale(e[u]);
    T out[N];
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      float y[4];
      unpack4(w[u][k / 4], y);
#pragma unroll
      for (int v = 0; v < 4; ++v) Elem<T>::put(out + k + v, y[v] * s);
    }
    T* o = reinterpret_cast<T*>(a.out[side]) + (size_t)(i0 + 256 * u) * N;
    __builtin_nontemporal_store(*reinterpret_cast<const uintx4*>(out), reinterpret_cast<uintx4*>(o));
  }
}

// ------------------------------------------------------------------------------------------------ attend
struct AttnArgs {
  const void* q;
  void* o;
  int64_t ldqb, ldqi, ldqh, ldob, ldoi, ldoh;
  const uint8_t* codes[2];
  const uint8_t* exps[2];
  Pages pages;
  const int32_t* lens;
  const uint8_t* mask;
  float* ws;                 // splits > 1: (rows, splits, dk) sums, then (rows, splits, 2) {max, sum of weights}
  int64_t rows, ld_mask;
  int mask_w, len0, causal, n, h, G, Lq, page, splits, chunk;
  float scale;               // of the scores, times log2(e)
};

__device__ inline int seq_len(const AttnArgs& a, int b) {
  int64_t len = a.lens ? a.lens[b] : a.len0;
  const int64_t cap = (int64_t)a.pages.per_seq * a.page;
  len = len < cap ? len : cap;
  return (int)(len > 0 ? len : 0);
}

// the value of lane ^ D for D = 2, 4, 8 (within 16 lanes) and, through row swaps, 16 and 32
template <int D> __device__ inline float lane_xor(float x, int lane) {
  if (D == 1) return dpp<0xB1>(x);
  if (D == 2) return dpp<0x4E>(x);
  if (D == 4) return dpp<0x1B>(dpp<0x141>(x));
  if (D == 8) return dpp<0x128>(x);
  const uintx2 r = D == 16 ? __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)
                           : __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(lane & D ? r[0] : r[1]);
}
// maximum / sum over the lanes that differ in the bits from log2(FROM) up, the same in all of them
template <int FROM> __device__ inline float across_max(float x, int lane) {
  if (FROM <= 2) x = fmaxf(x, lane_xor<2>(x, lane));
  if (FROM <= 4) x = fmaxf(x, lane_xor<4>(x, lane));
  if (FROM <= 8) x = fmaxf(x, lane_xor<8>(x, lane));
  x = fmaxf(x, lane_xor<16>(x, lane));
  return fmaxf(x, lane_xor<32>(x, lane));
}
template <int FROM> __device__ inline float across_sum(float x, int lane) {
  if (FROM <= 2) x += lane_xor<2>(x, lane);
  if (FROM <= 4) x += lane_xor<4>(x, lane);
  if (FROM <= 8) x += lane_xor<8>(x, lane);
  x += lane_xor<16>(x, lane);
  return x + lane_xor<32>(x, lane);
}
// 2 N values a lane -> N: a row swap hands the lower lanes the other half's first N, the upper ones the last N
template <int D, int N> __device__ inline void fold_rows(float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uintx2 r = D == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i + N]), false, false)
                             : __builtin_amdgcn_permlane16_swap(__float_as_uint(x[i]), __float_as_uint(x[i + N]), false, false);
    x[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
}
template <int D, int N> __device__ inline void fold_lanes(float (&x)[16], int lane) {
  const bool up = (lane & D) != 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float keep = up ? x[i + N] : x[i], send = up ? x[i] : x[i + N];
    x[i] = keep + lane_xor<D>(send, lane);
  }
}

// One query row at a time, without matrix instructions: DK / 16 lanes share a key (16 codes each), 64 / (DK / 16) keys an
// instruction, four such groups of keys in flight.  Every lane group keeps a softmax of its own (running maximum, sum, its 16
// dimensions); they meet once at the end, by halving what a lane holds.  A group of keys lies in one page (two at DK = 32 and
// 16 tokens a page), so its address is wave-uniform; keys that are not visible read the group's first row with the others.
template <typename T, int DK, int KW>
__global__ __launch_bounds__(256) void kv8_attn_row_kernel(AttnArgs a) {
  constexpr int LPK = DK / 16, NK = 64 / LPK, U = 4, KPI = NK * U, NV = DK >= 64 ? DK / 64 : 1;
  __shared__ float sm[KW == 1 ? 1 : 4][64 * NV + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t row = KW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  const int kw = KW == 1 ? 0 : wave;
  if (row >= a.rows) return;                                            // KW == 4: one row per block, uniform
  const int64_t this_row = row;
  const int g = (int)((uint32_t)row % (uint32_t)a.G);
  row = (uint32_t)row / (uint32_t)a.G;
  const int i = (int)((uint32_t)row % (uint32_t)a.Lq);
  row = (uint32_t)row / (uint32_t)a.Lq;
  const int head = (int)((uint32_t)row % (uint32_t)a.h), b = (int)((uint32_t)row / (uint32_t)a.h);
  const int part = lane % LPK, kg = lane / LPK;
  int end = seq_len(a, b) - (a.causal ? a.Lq - 1 - i : 0);
  const int split = blockIdx.y;
  const int64_t beg = (int64_t)split * a.chunk;
  if (end > beg + a.chunk) end = (int)(beg + a.chunk);
  float qr[16];
  const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.ldqb + (int64_t)i * a.ldqi + (int64_t)(head * a.G + g) * a.ldqh + 16 * part;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float x[4];
    Elem<T>::load4(q + 4 * c, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) qr[4 * c + e] = x[e];
  }
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int d = 0; d < 16; ++d) o[d] = 0.f;
  const PageRow pages(a.pages, b, a.codes[0]);
  const int shift = 31 - __clz(a.page), pm = a.page - 1;
  const uint8_t* mk = a.mask + (int64_t)b * a.ld_mask;
  const int row_off = (kg & (NK > 16 ? 15 : NK - 1)) * DK + 16 * part;
  for (int64_t j0 = beg + (int64_t)kw * KPI; j0 < end; j0 += (int64_t)KW * KPI) {
    uint4 kc[U], vc[U];
    int raw[U][2], ek[U], ev[U];
    bool vis[U];
    bool none = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = j0 + u * NK;
      raw[u][0] = pages.ask(t < end ? (int)(t >> shift) : 0);
      if (NK > 16) raw[u][1] = pages.ask(t + 16 < end ? (int)((t + 16) >> shift) : 0);
      vis[u] = kg < end - t;
    }
    if (a.mask) {
      uint8_t mb[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = j0 + u * NK + kg;
        vis[u] = vis[u] && j < a.mask_w;
        mb[u] = mk[vis[u] ? j : 0];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) vis[u] = vis[u] && mb[u] != 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) none = none && !vis[u];
    if (__all(none)) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = j0 + u * NK;
      const int id0 = pages.page(raw[u][0], (int)(t >> shift), t < end);
      int id = id0;
      if (NK > 16) {
        const int id1 = pages.page(raw[u][1], (int)((t + 16) >> shift), t + 16 < end);
        id = kg >= 16 ? id1 : id0;
      }
      vis[u] = vis[u] && id >= 0;
      const size_t ph = (size_t)(id < 0 ? 0 : id) * a.h + head;
      const size_t at = ph * a.page * DK + (NK > 16 ? ((int)t + (kg & 16)) & pm : (int)t & pm) * DK;
      const int off = vis[u] ? row_off : 16 * part;
      kc[u] = *reinterpret_cast<const uint4*>(a.codes[0] + at + off);
      vc[u] = *reinterpret_cast<const uint4*>(a.codes[1] + at + off);
      ek[u] = a.exps[0][ph];
      ev[u] = a.exps[1][ph];
    }
    float s[U];
    float mn = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = -INFINITY;
      if (!__any(vis[u])) continue;
      const uint32_t w[4] = {kc[u].x, kc[u].y, kc[u].z, kc[u].w};
      float acc = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float x[4];
        unpack4(w[c], x);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = fmaf(x[e], qr[4 * c + e], acc);
      }
      acc = group_sum<LPK>(acc) * (exp_scale(ek[u]) * a.scale);
      s[u] = vis[u] ? acc : -INFINITY;
      mn = fmaxf(mn, s[u]);
    }
    if (__any(mn > m + 8.f)) {                                          // weights may exceed 1 by 2^8 before the maximum is raised
      mn = fmaxf(mn, m);
      const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int d = 0; d < 16; ++d) o[d] *= al;
    }
    const float ms = m == -INFINITY ? 0.f : m;                          // nothing seen so far: every weight is 0
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!__any(vis[u])) continue;
      const float p = __builtin_amdgcn_exp2f(s[u] - ms);
      l += p;
      const float pv = vis[u] ? p * exp_scale(ev[u]) : 0.f;
      const uint32_t w[4] = {vis[u] ? vc[u].x : 0u, vis[u] ? vc[u].y : 0u, vis[u] ? vc[u].z : 0u, vis[u] ? vc[u].w : 0u};   // 0 * NaN would not vanish
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float x[4];
        unpack4(w[c], x);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * c + e] = fmaf(x[e], pv, o[4 * c + e]);
      }
    }
  }
  // the lane groups meet: 16 dimensions a lane become NV
  float M = across_max<LPK>(m, lane);
  const float f = __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
  l = across_sum<LPK>(l * f, lane);
#pragma unroll
  for (int d = 0; d < 16; ++d) o[d] *= f;
  fold_rows<32, 8>(o);
  fold_rows<16, 4>(o);
  if (LPK <= 8) fold_lanes<8, 2>(o, lane);
  if (LPK <= 4) fold_lanes<4, 1>(o, lane);
  if (LPK <= 2) o[0] += lane_xor<2>(o[0], lane);
  const int d0 = 16 * part + (lane >> 5) * 8 + (lane >> 4 & 1) * 4 + (LPK <= 8 ? (lane >> 3 & 1) * 2 : 0) + (LPK <= 4 ? lane >> 2 & 1 : 0);
  if (KW > 1) {
#pragma unroll
    for (int c = 0; c < NV; ++c) sm[wave][c * 64 + lane] = o[c];
    if (lane == 0) { sm[wave][64 * NV] = M; sm[wave][64 * NV + 1] = l; }
    __syncthreads();
    if (wave != 0) return;
    M = fmaxf(fmaxf(sm[0][64 * NV], sm[1][64 * NV]), fmaxf(sm[2][64 * NV], sm[3][64 * NV]));
    const float z = M == -INFINITY ? 0.f : M;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c) o[c] = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float r = __builtin_amdgcn_exp2f(sm[w][64 * NV] - z);
      l += r * sm[w][64 * NV + 1];
#pragma unroll
      for (int c = 0; c < NV; ++c) o[c] += r * sm[w][c * 64 + lane];
    }
  }
  if (LPK == 2 && (lane & 2)) return;                                   // two lanes hold the same dimension
  if (a.splits > 1) {
    float* dst = a.ws + (this_row * a.splits + split) * DK + d0;
#pragma unroll
    for (int c = 0; c < NV; ++c) dst[c] = o[c];
    if (lane == 0) {
      float* ml = a.ws + a.rows * a.splits * DK + (this_row * a.splits + split) * 2;
      ml[0] = M;
      ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;                           // no visible key: zeros
  T* dst = reinterpret_cast<T*>(a.o) + (int64_t)b * a.ldob + (int64_t)i * a.ldoi + (int64_t)(head * a.G + g) * a.ldoh + d0;
#pragma unroll
  for (int c = 0; c < NV; ++c) Elem<T>::put(dst + c, o[c] * inv);
}

// ---- several query rows at once, on the matrix cores
typedef __bf16 bfx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bfx8 __attribute__((ext_vector_type(8)));

union Frag {                 // eight bf16 of one lane: an operand of v_mfma_f32_16x16x32_bf16
  uint32_t u[4];
  bfx2 h[4];
  bfx8 v;
};
// how many bf16 pieces a query, and a weight of the softmax, is cut into.  A code is exact in bf16, so only the other operand decides
// the products' precision: fp32 = three pieces of 8 bits (exact).  16-bit queries are exact in one (bf16) or two (fp16).  Their
// weights take two, both rounded: within 2^-17, far below the half step of 2^-8 or 2^-11 by which the result is rounded.  One piece
// (2^-8, what a bf16 result's own rounding is) would let the error against 64 bits grow by 14 % (48 sequences up to 8 k, 32 / 8
// heads x 128 bf16: 1.63e-3 -> 1.85e-3 of the norm) for 0 to 9 % of the time (48 sequences 92 us either way, 12 x 50 queries 49 us
// with one, 53 with two, 57 with three; 512 queries of one sequence 69 / 75 / 83).
template <typename T> struct Pieces;
template <> struct Pieces<float> { static constexpr int Q = 3, P = 3; };
template <> struct Pieces<F16> { static constexpr int Q = 2, P = 2; };
template <> struct Pieces<B16> { static constexpr int Q = 1, P = 2; };

// 8 values into N pieces.  One or two: each rounds to nearest what is left (two: within 2^-17, and exact for fp16).  Three: each takes
// the next 8 bits, cut off, which leaves nothing of 24.
template <int N>
__device__ inline void cut_pieces(const float (&x)[8], Frag (&f)[N]) {
  if constexpr (N <= 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const floatx2 t = {x[2 * i], x[2 * i + 1]};
      f[0].h[i] = __builtin_convertvector(t, bfx2);
      if (N == 2) {
        const floatx2 r = {x[2 * i] - __uint_as_float(f[0].u[i] << 16), x[2 * i + 1] - __uint_as_float(f[0].u[i] & 0xFFFF0000u)};
        f[N - 1].h[i] = __builtin_convertvector(r, bfx2);
      }
    }
    return;
  }
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[k].u[i] = __builtin_amdgcn_perm(__float_as_uint(r[2 * i + 1]), __float_as_uint(r[2 * i]), 0x07060302u);
      if (k + 1 < N) {
        r[2 * i] -= __uint_as_float(__float_as_uint(r[2 * i]) & 0xFFFF0000u);
        r[2 * i + 1] -= __uint_as_float(__float_as_uint(r[2 * i + 1]) & 0xFFFF0000u);
      }
    }
  }
}
__device__ inline float quad_max(float x) {        // over the four lanes of a column (lane & 15)
  uintx2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float quad_sum(float x) {
  uintx2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The codes of 32 tokens as one lane (c = lane & 15, quad = lane >> 4) loads them.  For the scores: token rows c and 16 + c, 16
// codes of every 64.  For the second product: W = DK / 16 codes of the tokens 4 quad .. + 3 and 16 + 4 quad .. + 3, which are
// those whose scores the lane will hold.  The two halves of 16 tokens lie in one page each, so both addresses are wave-uniform
// plus an offset that never changes, and the exponents are wave-uniform too.
template <int DK>
struct CodeTile {
  static constexpr int W = DK / 16, KN = W >= 4 ? W : 2, VW = W >= 4 ? DK / 64 : 1;     // dwords of a lane's token row, and of W codes
  uint32_t k[2][KN];
  uint32_t v[8][VW];
  int ek[2], ev[2];

  // id0, id1: pages of the two halves
  __device__ inline void load(const AttnArgs& a, int head, int id0, int id1, int64_t t0, uint32_t koff, uint32_t voff) {
    const int pm = a.page - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const size_t ph = (size_t)(i ? id1 : id0) * a.h + head;
      const size_t at = (ph * a.page + ((int)(t0 + 16 * i) & pm)) * DK;
      const uint8_t* p = a.codes[0] + at + koff;
      if (DK == 32) {
        *reinterpret_cast<uint2*>(k[i]) = *reinterpret_cast<const uint2*>(p);
      } else {
#pragma unroll
        for (int w = 0; w < DK / 64; ++w) *reinterpret_cast<uint4*>(k[i] + 4 * w) = *reinterpret_cast<const uint4*>(p + 64 * w);
      }
      p = a.codes[1] + at + voff;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t* d = v[4 * i + j];
        if (W == 2) d[0] = *reinterpret_cast<const uint16_t*>(p + j * DK);
        else if (W == 4) d[0] = *reinterpret_cast<const uint32_t*>(p + j * DK);
        else if (W == 8) *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(p + j * DK);
        else *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(p + j * DK);
      }
      ek[i] = a.exps[0][ph];
      ev[i] = a.exps[1][ph];
    }
  }
};
__device__ inline int token_of(int i, int quad) { return (i >> 2) * 16 + 4 * quad + (i & 3); }      // of a lane's i-th score, within the 32

// Eight tokens' W codes as operands of the second product: group g is dimension W c + g of the lane's tokens, in bf16, scaled.
template <int DK>
__device__ inline void value_frag(Frag& f, const uint32_t (&v)[8][CodeTile<DK>::VW], int w, int g, const float (&scale)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {                                         // bytes {x0, y0, x1, y1} or {x2, y2, x3, y3} of two tokens
    const uint32_t two = __builtin_amdgcn_perm(v[2 * i + 1][w], v[2 * i][w], g < 2 ? 0x05010400u : 0x07030602u);
    f.h[i] = g & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(two, scale[i >> 1], true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(two, scale[i >> 1], false);
  }
}

// G * Lq query rows of one (sequence, key head) share its codes: NT tiles of 16 rows a wave.  Both products are taken
// transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane's scores (4 + 4 tokens of one query) are in place as the second
// product's operand and no weight crosses lanes; codes go from memory to registers to the matrix cores (a byte permute turns
// the eight token rows of V into columns), nothing is staged in shared memory.  The running maximum is only raised when a
// score passes it by 2^8: until then weights just exceed 1, which costs no precision and saves the rescaling.
// KW = 4: the block's waves take every fourth group of 32 tokens and meet at the end; KW = 1: every wave has rows of its own.
template <typename T, int DK, int NT, int KW, bool MASKED>
__global__ __launch_bounds__(256, DK == 256 ? 1 : 2) void kv8_attn_tile_kernel(AttnArgs a) {
  constexpr int W = DK / 16, KS = DK / 32, NQ = Pieces<T>::Q, NP = Pieces<T>::P, VW = CodeTile<DK>::VW, VG = W < 4 ? W : 4;
  constexpr int REGS = NT * (4 * W + 2);
  __shared__ float buf[KW == 1 ? 1 : 2 * REGS * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, quad = lane >> 4;
  const int M = a.G * a.Lq, mt = (M + 16 * NT - 1) / (16 * NT);
  const int kw = KW == 1 ? 0 : wave;
  // KW == 4: the tiles of one (sequence, key head, part) read the same codes, so they go to one die, one behind the other: blocks
  // are dealt to the eight dies in turn, and each has a cache of its own (8 sequences of 60000 tokens, 8 key heads x 128, 64 rows
  // a key head: with the tiles on different dies 293 us in bf16 and 528 in fp32, 266 and 421 us so; no difference where all codes fit
  // the memory-side cache: 12 sequences of 4000 tokens, 200 rows a key head, 54 us)
  const uint32_t groups = (uint32_t)a.n * a.h * a.splits;
  uint32_t group, tile;
  if (KW == 1) {
    const uint32_t unit = blockIdx.x * 4 + wave;
    group = unit / mt;
    tile = unit - group * mt;
  } else {
    const uint32_t at = blockIdx.x >> 3;
    group = at / mt * 8 + (blockIdx.x & 7);
    tile = at % mt;
  }
  if (group >= groups) return;                                          // KW == 4: one group a block, uniform
  const int split = (int)(group % a.splits);
  group /= a.splits;
  const int head = (int)(group % a.h), b = (int)(group / a.h), r0 = (int)tile * 16 * NT;
  const int len = seq_len(a, b);
  const int64_t beg = (int64_t)split * a.chunk;
  auto end_of = [&](int r) {                                            // tokens that row r sees, in this part
    const int64_t e = len - (a.causal ? a.Lq - 1 - r / a.G : 0);
    return (int)(e < beg + a.chunk ? e : beg + a.chunk);
  };
  const int rl = r0 + 16 * NT - 1 < M ? r0 + 16 * NT - 1 : M - 1;
  const int most = end_of(rl), least = end_of(r0);
  // the sign of the scale goes into the queries: the largest raw score then is the largest score
  const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f, scale = a.scale == 0.f ? 1.f : fabsf(a.scale);
  Frag qf[NT][KS][NQ];
  int end[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + c;
    end[t] = r < M ? end_of(r) : 0;
    const int rr = r < M ? r : M - 1;
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.ldqb + (int64_t)(rr / a.G) * a.ldqi + (int64_t)(head * a.G + rr % a.G) * a.ldqh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = DK == 32 ? 8 * quad : 64 * (s >> 1) + 16 * quad + 8 * (s & 1);
      float x[8], y[4];
      Elem<T>::load4(q + d, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = y[i] * sign;
      Elem<T>::load4(q + d + 4, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 + i] = y[i] * sign;
      cut_pieces<NQ>(x, qf[t][s]);
    }
  }
  floatx4 o[NT][W];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int g = 0; g < W; ++g) o[t][g] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const int shift = 31 - __clz(a.page), pm = a.page - 1;
  const PageRow pages(a.pages, b, a.codes[0]);
  const int64_t step = 32 * KW;
  int64_t t0 = beg + 32 * kw;
  auto ask = [&](int64_t tok) { return pages.ask(tok < most ? (int)(tok >> shift) : 0); };
  auto page = [&](int raw, int64_t tok) { return pages.page(raw, (int)(tok >> shift), tok < most); };
  // the mask of 32 tokens: a byte a lane, then a bit each
  const uint8_t* mk = a.mask + (MASKED ? (int64_t)b * a.ld_mask : 0);
  auto ask_mask = [&](int64_t tok) {
    const int64_t j = tok + (lane & 31);
    return MASKED ? (int)mk[j < a.mask_w ? j : 0] : 1;
  };
  auto mask_bits = [&](int raw, int64_t tok) { return MASKED ? (uint32_t)__ballot(raw != 0 && tok + (lane & 31) < a.mask_w) : ~0u; };
  const uint32_t koff = c * DK + (DK == 32 ? 8 : 16) * quad, voff = 4 * quad * DK + W * c;
  bool strange = false;
  // page ids (the same for all lanes) and masks are looked up two groups ahead, codes loaded one group ahead; where there is no page,
  // or 16 tokens are masked, page 0 is read instead, and a group with nothing else is passed over
  CodeTile<DK> tile0, tile1;
  int ra = ask(t0), rb = ask(t0 + 16), rm = ask_mask(t0);
  uint32_t bits = mask_bits(rm, t0);
  int id0 = bits & 0xFFFF ? page(ra, t0) : -1, id1 = bits >> 16 ? page(rb, t0 + 16) : -1;
  ra = ask(t0 + step), rb = ask(t0 + step + 16), rm = ask_mask(t0 + step);
  tile0.load(a, head, id0 < 0 ? 0 : id0, id1 < 0 ? 0 : id1, t0, koff, voff);
  auto group_of_32 = [&](CodeTile<DK>& cur, CodeTile<DK>& nxt) {
    const uint32_t next_bits = mask_bits(rm, t0 + step);
    const int nd0 = next_bits & 0xFFFF ? page(ra, t0 + step) : -1, nd1 = next_bits >> 16 ? page(rb, t0 + step + 16) : -1;
    ra = ask(t0 + 2 * step), rb = ask(t0 + 2 * step + 16), rm = ask_mask(t0 + 2 * step);
    nxt.load(a, head, nd0 < 0 ? 0 : nd0, nd1 < 0 ? 0 : nd1, t0 + step, koff, voff);
    if (MASKED && id0 < 0 && id1 < 0) {
      id0 = nd0, id1 = nd1, bits = next_bits;
      t0 += step;
      return;
    }
    // raw scores: sc[t][i][e] is the lane's query c of tile t against token t0 + 16 i + 4 quad + e
    floatx4 sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {                                      // 2 NT sums side by side: each waits for its own last step only
      Frag kf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kf[i].h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(cur.k[i][2 * s], 1.f, false);
        kf[i].h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(cur.k[i][2 * s], 1.f, true);
        kf[i].h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(cur.k[i][2 * s + 1], 1.f, false);
        kf[i].h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(cur.k[i][2 * s + 1], 1.f, true);
      }
#pragma unroll
      for (int p = NQ - 1; p >= 0; --p) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            sc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i].v, qf[t][s][p].v, sc[t][i], 0, 0, 0);
        }
      }
    }
    const float ks[2] = {exp_scale(cur.ek[0]) * scale, exp_scale(cur.ek[1]) * scale};
    float vs[2] = {exp_scale(cur.ev[0]), exp_scale(cur.ev[1])};
    const bool plain = t0 + 32 <= least && bits == ~0u && id0 >= 0 && id1 >= 0;  // every row of the unit sees all 32 tokens
    if (!plain) {
      // bit i: the lane's i-th token exists and is not masked
      const uint32_t seen = (id0 >= 0 ? bits >> 4 * quad & 0x0Fu : 0u) | (id1 >= 0 ? (bits >> (16 + 4 * quad) & 0x0Fu) << 4 : 0u);
      // codes that no row sees must not be NaN (0 * NaN is not 0); nor may those that only some rows see: they are taken out
      // here and put back behind the loop.  Half a page that nobody sees may hold any exponent.
      const bool some = least < most && t0 + 32 > least;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool dead = !(t0 + token_of(i, quad) < most) || !(seen >> i & 1);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t x = dead ? 0u : cur.v[i][w];
          if (some) {
            const uint32_t hit = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
            strange = strange || hit != 0;
            x &= ~((hit >> 7) * 0xFFu);
          }
          cur.v[i][w] = x;
        }
      }
      if (!(seen & 0x0Fu)) vs[0] = 1.f;
      if (!(seen & 0xF0u)) vs[1] = 1.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t left = end[t] - t0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(token_of(i, quad) < left) || !(seen >> i & 1)) sc[t][i >> 2][i & 3] = -INFINITY;
      }
    }
    Frag pf[NT][NP];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float top = fmaxf(fmaxf(sc[t][i][0], sc[t][i][1]), fmaxf(sc[t][i][2], sc[t][i][3]));
        mx = fmaxf(mx, top == -INFINITY ? top : top * ks[i]);           // the exponent of half a page that nobody sees does not count
      }
      if (__any(mx > m[t] + 8.f)) {
        mx = fmaxf(m[t], quad_max(mx));
        const float al = __builtin_amdgcn_exp2f(m[t] - (mx == -INFINITY ? 0.f : mx));
        m[t] = mx;
        l[t] *= al;
#pragma unroll
        for (int g = 0; g < W; ++g) o[t][g] *= al;
      }
      const float ms = m[t] == -INFINITY ? 0.f : m[t];
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(sc[t][i >> 2][i & 3], ks[i >> 2], -ms);
      if (!plain) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sc[t][i >> 2][i & 3] == -INFINITY ? -INFINITY : x[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i]);
        l[t] += x[i];
      }
      cut_pieces<NP>(x, pf[t]);
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
#pragma unroll
      for (int g = 0; g < VG; ++g) {
        Frag vf;
        value_frag<DK>(vf, cur.v, w, g, vs);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int p = NP - 1; p >= 0; --p)
            o[t][4 * w + g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf.v, pf[t][p].v, o[t][4 * w + g], 0, 0, 0);
        }
      }
    }
    id0 = nd0, id1 = nd1, bits = next_bits;
    t0 += step;
  };
  while (t0 < most) {
    group_of_32(tile0, tile1);
    if (t0 >= most) break;
    group_of_32(tile1, tile0);
  }
  if (__any(strange)) {                                                 // NaN for the rows that see it: token by token, rare
    for (int64_t g0 = beg + 32 * kw; g0 < most; g0 += step) {
      if (g0 + 32 <= least) continue;
      for (int64_t j = g0; j < g0 + 32 && j < most; ++j) {
        const int id = page(ask(j), j);
        if (id < 0 || (MASKED && (j >= a.mask_w || mk[j] == 0))) continue;
        const uint8_t* p = a.codes[1] + (((size_t)id * a.h + head) * a.page + ((int)j & pm)) * DK + 4 * W * quad;
#pragma unroll
        for (int i = 0; i < 4 * W; ++i) {                               // dimension W e + g of the lane's 4 W
          const bool nan = (p[i] & 0x7F) == 0x7F;
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (nan && j < end[t]) o[t][i % W][i / W] = __uint_as_float(0x7FC00000u);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) l[t] = quad_sum(l[t]);
  if (KW > 1) {                                                         // waves 2, 3 hand over to 0, 1, then 1 to 0
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
      float* dst = buf + (wave & (half - 1)) * REGS * 64 + lane;
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int g = 0; g < W; ++g) {
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[(t * (4 * W + 2) + 4 * g + e) * 64] = o[t][g][e];
          }
          dst[(t * (4 * W + 2) + 4 * W) * 64] = m[t];
          dst[(t * (4 * W + 2) + 4 * W + 1) * 64] = l[t];
        }
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float m2 = dst[(t * (4 * W + 2) + 4 * W) * 64], l2 = dst[(t * (4 * W + 2) + 4 * W + 1) * 64];
          const float mm = fmaxf(m[t], m2), z = mm == -INFINITY ? 0.f : mm;
          const float f1 = __builtin_amdgcn_exp2f(m[t] - z), f2 = __builtin_amdgcn_exp2f(m2 - z);
          m[t] = mm;
          l[t] = l[t] * f1 + l2 * f2;
#pragma unroll
          for (int g = 0; g < W; ++g) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][g][e] = o[t][g][e] * f1 + dst[(t * (4 * W + 2) + 4 * g + e) * 64] * f2;
          }
        }
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = r0 + 16 * t + c;
    if (r >= M) continue;
    const int64_t row = ((int64_t)b * a.h + head) * M + r;
    float* part = a.splits > 1 ? a.ws + (row * a.splits + split) * DK + 4 * W * quad : nullptr;
    T* dst = reinterpret_cast<T*>(a.o) + (int64_t)b * a.ldob + (int64_t)(r / a.G) * a.ldoi + (int64_t)(head * a.G + r % a.G) * a.ldoh + 4 * W * quad;
    const float inv = part ? 1.f : l[t] == 0.f ? 0.f : 1.f / l[t];
#pragma unroll
    for (int i = 0; i < 4 * W; i += 4) {                                // dimension W e + g of the lane's 4 W
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = o[t][(i + e) % W][(i + e) / W] * inv;
      if (part) *reinterpret_cast<float4*>(part + i) = make_float4(y[0], y[1], y[2], y[3]);
      else Elem<T>::store4(dst + i, y);
    }
    if (part && quad == 0) {
      float* ml = a.ws + a.rows * a.splits * DK + (row * a.splits + split) * 2;
      ml[0] = m[t];
      ml[1] = l[t];
    }
  }
}

// joins few parts of many rows: a thread per four dimensions of a row
template <typename T>
__global__ __launch_bounds__(256) void kv8_attn_join_few_kernel(AttnArgs a, int dk) {
  const int per = dk >> 2;
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, r = at / per, d = at - r * per;
  if (r >= a.rows) return;
  const uint32_t g = r % a.G, rest = r / a.G, i = rest % a.Lq, bh = rest / a.Lq, head = bh % a.h, b = bh / a.h;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + a.rows * a.splits * dk) + (size_t)r * a.splits;
  const float4* part = reinterpret_cast<const float4*>(a.ws + (size_t)r * a.splits * dk) + d;
  float M = -INFINITY;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, ml[s].x);
  const float z = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < a.splits; ++s) {
    const float2 o = ml[s];
    const float f = __builtin_amdgcn_exp2f(o.x - z);
    const float4 v = part[(size_t)s * per];
    l = fmaf(f, o.y, l);
    acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;                           // no visible key: zeros
  T* dst = reinterpret_cast<T*>(a.o) + (int64_t)b * a.ldob + (int64_t)i * a.ldoi + (int64_t)(head * a.G + g) * a.ldoh + 4 * d;
  const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  Elem<T>::store4(dst, y);
}

// joins the parts of a split row: a block a row; DK / 4 threads hold four dimensions each, the others take every so-manieth part
template <typename T>
__global__ __launch_bounds__(256) void kv8_attn_join_kernel(AttnArgs a, int dk) {
  __shared__ float w[1024], red[4];
  __shared__ float4 sums[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int g = (int)(row % a.G);
  int64_t rest = row / a.G;
  const int i = (int)(rest % a.Lq);
  rest /= a.Lq;
  const int head = (int)(rest % a.h), b = (int)(rest / a.h);
  const float* ml = a.ws + a.rows * a.splits * dk + row * a.splits * 2;
  float M = -INFINITY;
  for (int s = tid; s < a.splits; s += 256) M = fmaxf(M, w[s] = ml[2 * s]);
  M = wave_max(M);
  if (lane == 0) red[wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float z = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  for (int s = tid; s < a.splits; s += 256) {
    w[s] = __builtin_amdgcn_exp2f(w[s] - z);
    l += w[s] * ml[2 * s + 1];
  }
  l = wave_sum(l);
  __syncthreads();
  if (lane == 0) red[wave] = l;
  __syncthreads();
  l = (red[0] + red[1]) + (red[2] + red[3]);
  const int per = dk >> 2, d = tid % per, p0 = tid / per, np = 256 / per;
  const float4* part = reinterpret_cast<const float4*>(a.ws + row * a.splits * dk) + d;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = p0; s < a.splits; s += np) {
    const float4 v = part[(size_t)s * per];
    const float f = w[s];
    acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
  }
  sums[tid] = acc;
  __syncthreads();
  if (tid >= per) return;
  for (int k = 1; k < np; ++k) {
    const float4 v = sums[tid + k * per];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;                           // no visible key: zeros
  T* dst = reinterpret_cast<T*>(a.o) + (int64_t)b * a.ldob + (int64_t)i * a.ldoi + (int64_t)(head * a.G + g) * a.ldoh + 4 * d;
  const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  Elem<T>::store4(dst, y);
}

bool page_ok(int page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }
bool dk_ok(int dk) { return dk == 32 || dk == 64 || dk == 128 || dk == 256; }
int type_bytes(int dtype) { return dtype == TVAE_F32 ? 4 : dtype == TVAE_BF16 || dtype == TVAE_F16 ? 2 : 0; }

// the checks that the three entry points share
int check_cache(const char* who, const uint8_t* kc, const uint8_t* vc, const uint8_t* ke, const uint8_t* ve, int n_pages,
                const int32_t* table, int per_seq, int n, int h, int dk, int page, int dtype) {
  TVAE_CHECK(kc && vc && ke && ve, TVAE_E_NULL, "%s: null cache pointer", who);
  TVAE_CHECK(type_bytes(dtype), TVAE_E_DTYPE, "%s: dtype %d is not TVAE_F32, TVAE_BF16 or TVAE_F16", who, dtype);
  TVAE_CHECK(n >= 0 && h > 0 && dk_ok(dk) && page_ok(page), TVAE_E_SHAPE,
             "%s: need n >= 0, h >= 1, dk in {32, 64, 128, 256}, page a power of two in [16, 256] (n=%d h=%d dk=%d page=%d)", who, n, h, dk, page);
  TVAE_CHECK(n_pages >= 1 && per_seq >= 1 && (int64_t)per_seq * page <= INT32_MAX, TVAE_E_SHAPE,
             "%s: bad page counts (n_pages=%d, %d a sequence of %d tokens)", who, n_pages, per_seq, page);
  TVAE_CHECK(table || (int64_t)n * per_seq <= n_pages, TVAE_E_SHAPE, "%s: %d sequences of %d pages do not fit %d pages", who, n, per_seq, n_pages);
  TVAE_CHECK(aligned16(kc) && aligned16(vc), TVAE_E_SHAPE, "%s: cache codes must be 16-byte aligned", who);
  return TVAE_OK;
}
bool rows_ok(const void* p, int64_t ldb, int64_t ldt, int64_t ldh, int dtype) {
  const int64_t m = 16 / type_bytes(dtype);
  return aligned16(p) && ldb % m == 0 && ldt % m == 0 && ldh % m == 0;
}

template <typename T, int DK>
void launch_store_dk(const StoreArgs& a, int units, hipStream_t s) {
  constexpr int N = Raw<T>::N;
  if (a.T <= 4) hipLaunchKernelGGL((kv8_append_kernel<T, DK>), dim3(cdiv(units, 256 * N / DK)), dim3(256), 0, s, a);
  else if (a.page * DK <= 64 * N) hipLaunchKernelGGL((kv8_store_kernel<T, DK, 64, 1>), dim3(cdiv(units, 4), 2), dim3(256), 0, s, a);
  else if (a.page * DK <= 64 * 4 * N) hipLaunchKernelGGL((kv8_store_kernel<T, DK, 64, 4>), dim3(cdiv(units, 4), 2), dim3(256), 0, s, a);
  else if (a.page * DK <= 64 * 8 * N) hipLaunchKernelGGL((kv8_store_kernel<T, DK, 64, 8>), dim3(cdiv(units, 4), 2), dim3(256), 0, s, a);
  else if (a.page * DK <= 256 * 4 * N) hipLaunchKernelGGL((kv8_store_kernel<T, DK, 256, 4>), dim3(units, 2), dim3(256), 0, s, a);
  else if (a.page * DK <= 256 * 8 * N) hipLaunchKernelGGL((kv8_store_kernel<T, DK, 256, 8>), dim3(units, 2), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv8_store_kernel<T, DK, 256, 16>), dim3(units, 2), dim3(256), 0, s, a);
}
template <typename T>
void launch_store(const StoreArgs& a, int dk, int units, hipStream_t s) {
  if (dk == 32) launch_store_dk<T, 32>(a, units, s);
  else if (dk == 64) launch_store_dk<T, 64>(a, units, s);
  else if (dk == 128) launch_store_dk<T, 128>(a, units, s);
  else launch_store_dk<T, 256>(a, units, s);
}
template <typename T>
void launch_load(const LoadArgs& a, int dk, hipStream_t s) {
  const dim3 grid((a.total + 1023) / 1024, 2);
  if (dk == 32) hipLaunchKernelGGL((kv8_load_kernel<T, 32>), grid, dim3(256), 0, s, a);
  else if (dk == 64) hipLaunchKernelGGL((kv8_load_kernel<T, 64>), grid, dim3(256), 0, s, a);
  else if (dk == 128) hipLaunchKernelGGL((kv8_load_kernel<T, 128>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv8_load_kernel<T, 256>), grid, dim3(256), 0, s, a);
}
template <typename T, int DK>
void launch_row(const AttnArgs& a, hipStream_t s) {
  // a wave a row where the rows fill the chip, else a block a row: rows of different lengths then even out (wave / block, 0 .. keys
  // tokens a row, DK = 64: 2048 rows of 128 keys 10.6 / 12.1 us, of 2048 68 / 53; 8064 rows of 128 17 / 31 us, of 512 50 / 52, of
  // 2048 203 / 182; DK = 256, 4096 rows of 64 19 / 20, of 256 56 / 48)
  if (a.rows * a.splits >= (int64_t)a.chunk * DK / 4 || a.rows > MAX_BLOCKS)
    hipLaunchKernelGGL((kv8_attn_row_kernel<T, DK, 1>), dim3((unsigned)((a.rows + 3) / 4), a.splits), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv8_attn_row_kernel<T, DK, 4>), dim3((unsigned)a.rows, a.splits), dim3(256), 0, s, a);
}
template <typename T, int DK, int NT, bool MASKED>
void launch_tile_as(const AttnArgs& a, hipStream_t s) {
  const int64_t tiles = (a.G * a.Lq + 16 * NT - 1) / (16 * NT), groups = (int64_t)a.n * a.h * a.splits, units = groups * tiles;
  // a wave a unit where units fill the chip or keys are few, else a block a unit, whose waves have to meet at the end (wave / block,
  // 0 .. keys tokens a sequence, 4 query heads a key head, bf16: DK = 128, 4096 units of 128 keys 26 / 53 us, of 1024 123 / 120, of
  // 2048 230 / 203; DK = 256, where a block has its compute unit to itself, 1024 units of 128 keys 17 / 43, of 1024 68 / 82, 2048 units
  // of 1024 126 / 153, of 4096 445 / 389; 132 rows a key head, DK = 64: 1520 units of 300 keys 20 / 27, of 2048 85 / 63)
  if (units >= (int64_t)a.chunk * (DK == 256 ? 1 : 3) || units + 8 * tiles > MAX_BLOCKS)
    hipLaunchKernelGGL((kv8_attn_tile_kernel<T, DK, NT, 1, MASKED>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv8_attn_tile_kernel<T, DK, NT, 4, MASKED>), dim3((unsigned)((groups + 7) / 8 * 8 * tiles)), dim3(256), 0, s, a);
}
// masks are a variant of their own: looked up two groups ahead, a byte a lane and a ballot, they cost 7 to 16 % (23 sequences of 15 k
// tokens, 99 rows a key head, DK = 256, all visible, with / without a mask: one key head bf16 135 / 126 us, two fp32 368 / 317; eight
// byte loads a lane where they are needed took about twice the time)
template <typename T, int DK, int NT>
void launch_tile(const AttnArgs& a, hipStream_t s) {
  if (a.mask) launch_tile_as<T, DK, NT, true>(a, s);
  else launch_tile_as<T, DK, NT, false>(a, s);
}
template <typename T, int DK>
void launch_dk(const AttnArgs& a, hipStream_t s) {
  // tiles of 16 rows a wave: what is unpacked once serves all of them, but two waves a SIMD have to stay (one query sequence of 512
  // tokens, 32 heads, 8 key heads x 128 bf16, 4000 keys: 1 tile 116 us, 2 tiles 81 us = 414 TFLOP/s, 4 tiles, one wave a SIMD, 105 us).
  // A tile takes DK / 32 * pieces * 4 registers of queries, DK / 4 of sums and 8 of scores.
  constexpr int PER = DK / 32 * Pieces<T>::Q * 4 + DK / 4 + 8, MOST = 4 * PER <= 120 ? 4 : 2 * PER <= 120 ? 2 : 1;
  const int M = a.G * a.Lq;
  if (M == 1) launch_row<T, DK>(a, s);
  else if (M <= 16 || MOST == 1) launch_tile<T, DK, 1>(a, s);
  else if (M <= 32 || MOST == 2) launch_tile<T, DK, MOST == 1 ? 1 : 2>(a, s);
  else launch_tile<T, DK, MOST>(a, s);
}
template <typename T>
void launch_attn(const AttnArgs& a, int dk, hipStream_t s) {
  if (dk == 32) launch_dk<T, 32>(a, s);
  else if (dk == 64) launch_dk<T, 64>(a, s);
  else if (dk == 128) launch_dk<T, 128>(a, s);
  else launch_dk<T, 256>(a, s);
  if (a.splits > 16) hipLaunchKernelGGL((kv8_attn_join_kernel<T>), dim3((unsigned)a.rows), dim3(256), 0, s, a, dk);
  else if (a.splits > 1) hipLaunchKernelGGL((kv8_attn_join_few_kernel<T>), dim3((unsigned)((a.rows * (dk / 4) + 255) / 256)), dim3(256), 0, s, a, dk);
}

}  // namespace

extern "C" int tvae_kv8_store(const void* k, int64_t ldkb, int64_t ldkt, int64_t ldkh, const void* v, int64_t ldvb, int64_t ldvt,
                              int64_t ldvh, int dtype, uint8_t* kc, uint8_t* vc, uint8_t* ke, uint8_t* ve, int n_pages,
                              const int32_t* table, int per_seq, const int32_t* start, int start0, const int32_t* count, int n,
                              int T, int h, int dk, int page, void* stream) {
  TVAE_CHECK((k && v) || n == 0 || T == 0, TVAE_E_NULL, "tvae_kv8_store: null pointer");
  const int rc = check_cache("tvae_kv8_store", kc, vc, ke, ve, n_pages, table, per_seq, n, h, dk, page, dtype);
  if (rc) return rc;
  TVAE_CHECK(T >= 0 && start0 >= 0 && (start || (int64_t)start0 + (count ? 0 : T) <= (int64_t)per_seq * page), TVAE_E_SHAPE,
             "tvae_kv8_store: rows %d .. %lld do not fit %d pages of %d tokens", start0, (long long)start0 + T, per_seq, page);
  TVAE_CHECK(rows_ok(k, ldkb, ldkt, ldkh, dtype) && rows_ok(v, ldvb, ldvt, ldvh, dtype), TVAE_E_SHAPE,
             "tvae_kv8_store: k and v rows must be 16-byte aligned");
  if (n == 0 || T == 0) return TVAE_OK;
  const int slots = (T - 1 + page - 1) / page + 1;                      // pages that T rows can touch
  const int64_t units = T <= 4 ? (int64_t)n * h : (int64_t)n * slots * h;
  TVAE_CHECK(units <= MAX_BLOCKS, TVAE_E_SHAPE, "tvae_kv8_store: too many pages in one call");
  StoreArgs a = {{k, v}, {ldkb, ldvb}, {ldkt, ldvt}, {ldkh, ldvh}, {kc, vc}, {ke, ve}, {table, per_seq, n_pages}, start, count,
                 Divisor(h), start0, n, T, h, page, slots};
  if (dtype == TVAE_F32) launch_store<float>(a, dk, (int)units, (hipStream_t)stream);
  else if (dtype == TVAE_BF16) launch_store<B16>(a, dk, (int)units, (hipStream_t)stream);
  else launch_store<F16>(a, dk, (int)units, (hipStream_t)stream);
  TVAE_LAUNCH_CHECK("tvae_kv8_store");
  return TVAE_OK;
}

extern "C" int tvae_kv8_load(const uint8_t* kc, const uint8_t* vc, const uint8_t* ke, const uint8_t* ve, int n_pages,
                             const int32_t* table, int per_seq, const int32_t* start, int start0, const int32_t* count, void* k,
                             void* v, int dtype, int n, int T, int h, int dk, int page, void* stream) {
  TVAE_CHECK((k && v) || n == 0 || T == 0, TVAE_E_NULL, "tvae_kv8_load: null pointer");
  const int rc = check_cache("tvae_kv8_load", kc, vc, ke, ve, n_pages, table, per_seq, n, h, dk, page, dtype);
  if (rc) return rc;
  TVAE_CHECK(T >= 0 && aligned16(k) && aligned16(v), TVAE_E_SHAPE, "tvae_kv8_load: T must not be negative, k and v 16-byte aligned");
  if (n == 0 || T == 0) return TVAE_OK;
  const int64_t total = (int64_t)n * h * T * (dk * type_bytes(dtype) / 16);
  TVAE_CHECK((int64_t)n * h <= INT32_MAX && total <= INT32_MAX, TVAE_E_SHAPE, "tvae_kv8_load: too many rows in one call");
  LoadArgs a = {{kc, vc}, {ke, ve}, {k, v}, {table, per_seq, n_pages}, start, count, Divisor(T), Divisor(h), (uint32_t)total, start0, T, h, page};
  if (dtype == TVAE_F32) launch_load<float>(a, dk, (hipStream_t)stream);
  else if (dtype == TVAE_BF16) launch_load<B16>(a, dk, (hipStream_t)stream);
  else launch_load<F16>(a, dk, (hipStream_t)stream);
  TVAE_LAUNCH_CHECK("tvae_kv8_load");
  return TVAE_OK;
}

extern "C" int tvae_kv8_attn(const void* q, int64_t ldqb, int64_t ldqi, int64_t ldqh, void* o, int64_t ldob, int64_t ldoi,
                             int64_t ldoh, int dtype, const uint8_t* kc, const uint8_t* vc, const uint8_t* ke, const uint8_t* ve,
                             int n_pages, const int32_t* table, int per_seq, const int32_t* lens, int len0,
                             const uint8_t* key_mask, int64_t ld_mask, int mask_w, int causal, int n, int h, int G, int Lq, int dk,
                             int page, float scale, int splits, float* ws, void* stream) {
  TVAE_CHECK((q && o) || n == 0 || Lq == 0, TVAE_E_NULL, "tvae_kv8_attn: null pointer");
  const int rc = check_cache("tvae_kv8_attn", kc, vc, ke, ve, n_pages, table, per_seq, n, h, dk, page, dtype);
  if (rc) return rc;
  TVAE_CHECK(G >= 1 && Lq >= 0 && (int64_t)h * G <= INT32_MAX, TVAE_E_SHAPE, "tvae_kv8_attn: need G >= 1 and Lq >= 0 (G=%d Lq=%d)", G, Lq);
  TVAE_CHECK(rows_ok(q, ldqb, ldqi, ldqh, dtype) && rows_ok(o, ldob, ldoi, ldoh, dtype), TVAE_E_SHAPE,
             "tvae_kv8_attn: q and o rows must be 16-byte aligned");
  TVAE_CHECK(lens || (len0 >= 0 && len0 <= (int64_t)per_seq * page), TVAE_E_SHAPE, "tvae_kv8_attn: %d keys do not fit %d pages of %d tokens",
             len0, per_seq, page);
  TVAE_CHECK(!key_mask || (mask_w >= 0 && ld_mask >= mask_w), TVAE_E_SHAPE, "tvae_kv8_attn: bad mask shape");
  const int64_t rows = (int64_t)n * Lq * h * G;
  TVAE_CHECK(splits >= 1 && splits <= 1024 && (splits == 1 || rows == 0 || (ws && aligned16(ws))), TVAE_E_SHAPE,
             "tvae_kv8_attn: 1 .. 1024 splits, more than one with a 16-byte aligned workspace");
  TVAE_CHECK((splits > 1 ? rows : (rows + 3) / 4) <= MAX_BLOCKS && rows * splits <= 4 * MAX_BLOCKS, TVAE_E_SHAPE, "tvae_kv8_attn: too many query rows in one call");
  if (rows == 0) return TVAE_OK;
  const int64_t cap = lens ? (int64_t)per_seq * page : len0;
  int64_t chunk = ((cap + splits - 1) / splits + 127) / 128 * 128;
  chunk = chunk < INT32_MAX ? chunk : INT32_MAX;
  if (key_mask && mask_w == 0) { key_mask = ke; ld_mask = 0; }           // no byte of it counts, but one is read
  AttnArgs a = {q, o, ldqb, ldqi, ldqh, ldob, ldoi, ldoh, {kc, vc}, {ke, ve}, {table, per_seq, n_pages}, lens, key_mask, ws, rows,
                ld_mask, mask_w, len0, causal, n, h, G, Lq, page, splits, (int)chunk, scale * 1.44269504088896341f};
  if (dtype == TVAE_F32) launch_attn<float>(a, dk, (hipStream_t)stream);
  else if (dtype == TVAE_BF16) launch_attn<B16>(a, dk, (hipStream_t)stream);
  else launch_attn<F16>(a, dk, (hipStream_t)stream);
  TVAE_LAUNCH_CHECK("tvae_kv8_attn");
  return TVAE_OK;
}
