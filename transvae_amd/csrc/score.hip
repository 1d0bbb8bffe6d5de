// Log probabilities of given tokens, entropies and most likely alternatives of rows of logits, and their gradient.
//
// One pass over a row: every lane keeps a running maximum m, l = sum exp(x - m) and t = sum exp(x - m) (x - m), rescaled when
// its maximum grows; then with M the row's maximum   ln p_y = x_y - M - ln l,   H = ln l - t / l.
// (t is taken relative to the maximum: sum p x would cancel against ln-sum-exp when all logits are far from zero.)
// The alternatives ride along: a wave keeps its best `top` as a list sorted across its lanes and looks at a vector of logits
// again only if it holds something above the list's last entry, which soon is rare: a row of V values in any random order
// enters top * (1 + ln(V / top)) values a wave.
#include "common.h"

namespace {

struct F16 { _Float16 v; };
struct B16 { uint16_t v; };
constexpr float LOG2E = 1.44269504088896341f;
constexpr int SHORT = 256;                                 // classes that 32 lanes hold in registers (8 a lane)
constexpr int NO_KEY = INT32_MIN;                          // below every value
constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;              // of 256 threads: a grid counts its threads in 32 bits

__device__ inline float value_of(float x) { return x; }
__device__ inline float value_of(B16 x) { return __uint_as_float((uint32_t)x.v << 16); }
__device__ inline float value_of(F16 x) { return (float)x.v; }
__device__ inline void put(float* p, float x) { *p = x; }
__device__ inline void put(F16* p, float x) { p->v = (_Float16)x; }
__device__ inline void put(B16* p, float x) {              // round to nearest even; NaN stays NaN
  const uint32_t u = __float_as_uint(x);
  p->v = (u & 0x7FFFFFFFu) > 0x7F800000u ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

template <typename T> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};

// order of the alternatives as whole numbers: -0 equals +0, NaN is above everything
__device__ inline int key_of(float x) {
  if (x != x) return INT32_MAX;
  const int u = __float_as_int(x + 0.f);
  return u < 0 ? u ^ 0x7FFFFFFF : u;
}
__device__ inline float of_key(int k) { return k == INT32_MAX ? __int_as_float(0x7FC00000) : __int_as_float(k < 0 ? k ^ 0x7FFFFFFF : k); }

template <int CTRL> __device__ inline int dpp(int x) { return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xF, 0xF, false); }
template <int CTRL> __device__ inline float dppf(float x) { return __int_as_float(dpp<CTRL>(__float_as_int(x))); }
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
// the value of lane ^ D, without shared memory: quad permutes, mirrors of 8 (^ 7) and 16 (^ 15) lanes, row swaps
template <int D> __device__ inline int lane_xor(int x, int lane) {
  if (D == 1) return dpp<0xB1>(x);
  if (D == 2) return dpp<0x4E>(x);
  if (D == 4) return dpp<0x1B>(dpp<0x141>(x));
  if (D == 8) return dpp<0x141>(dpp<0x140>(x));
  const uintx2 r = D == 16 ? __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false)
                           : __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
  return (int)(lane & D ? r[0] : r[1]);
}
template <int D> __device__ inline float lane_xorf(float x, int lane) { return __int_as_float(lane_xor<D>(__float_as_int(x), lane)); }

struct Sums {
  float m = -INFINITY, l = 0.f, t = 0.f;
  __device__ inline void grow(float to) {                  // to > m
    if (l != 0.f) {                                        // also a NaN
      const float d = m - to, r = __builtin_amdgcn_exp2f(d * LOG2E);
      t = r * (t + l * fmaxf(d, -1e30f));
      l *= r;
    }
    m = to;
  }
  __device__ inline void add(float x) {                    // m is at least x, or x is NaN
    const float d = x - (m == -INFINITY ? 0.f : m), e = __builtin_amdgcn_exp2f(d * LOG2E);
    l += e;
    t = fmaf(e, fmaxf(d, -1e30f), t);                      // -inf adds 0, not 0 * inf
  }
  __device__ inline void add_finite(float x) {             // x - m is finite (x > -inf, x <= m < 1e30), or x is NaN
    const float d = x - m, e = __builtin_amdgcn_exp2f(d * LOG2E);
    l += e;
    t = fmaf(e, d, t);
  }
  __device__ inline void over_wave(int lane) {             // every lane ends with the sums of all
    float M = m;
    M = fmaxf(M, dppf<0xB1>(M));
    M = fmaxf(M, dppf<0x4E>(M));
    M = fmaxf(M, dppf<0x141>(M));
    M = fmaxf(M, dppf<0x140>(M));
    M = fmaxf(M, lane_xorf<16>(M, lane));
    M = fmaxf(M, lane_xorf<32>(M, lane));
    if (M > m) grow(M);
    l = total(l, lane);
    t = total(t, lane);
  }
  static __device__ inline float total(float x, int lane) {
    x += dppf<0xB1>(x);
    x += dppf<0x4E>(x);
    x += dppf<0x141>(x);
    x += dppf<0x140>(x);
    x += lane_xorf<16>(x, lane);
    return x + lane_xorf<32>(x, lane);
  }
  __device__ inline void join(float m2, float l2, float t2) {
    if (m2 > m) grow(m2);
    if (l2 != 0.f) {
      const float d = m2 - (m == -INFINITY ? 0.f : m), r = __builtin_amdgcn_exp2f(d * LOG2E);
      l += r * l2;
      t += r * (t2 + l2 * fmaxf(d, -1e30f));
    }
  }
};

// the n-th largest of the lanes' keys (n = 1 .. 64), for many by a bitonic sort across the wave, descending
template <int SIZE, int D> __device__ inline void sort_step(int& k, int lane) {
  const int other = lane_xor<D>(k, lane);
  const bool up = (lane & SIZE) != 0, low = (lane & D) == 0;
  k = (low != up) ? max(k, other) : min(k, other);
}
template <int SIZE, int D> __device__ inline void sort_steps(int& k, int lane) {
  sort_step<SIZE, D>(k, lane);
  if constexpr (D > 1) sort_steps<SIZE, D / 2>(k, lane);
}
__device__ inline int max_key(int k, int lane) {
  k = max(k, dpp<0xB1>(k));
  k = max(k, dpp<0x4E>(k));
  k = max(k, dpp<0x141>(k));
  k = max(k, dpp<0x140>(k));
  k = max(k, lane_xor<16>(k, lane));
  return max(k, lane_xor<32>(k, lane));
}
__device__ inline int nth_key(int k, int lane, int n) {
  if (n <= 8) {                                            // n maxima taken out one by one are fewer steps than the sort's 21
    for (int i = 1; i < n; ++i) {
      const int m = max_key(k, lane);
      if (lane == __ffsll((unsigned long long)__ballot(k == m)) - 1) k = NO_KEY;
    }
    return max_key(k, lane);
  }
  sort_steps<2, 1>(k, lane);
  sort_steps<4, 2>(k, lane);
  sort_steps<8, 4>(k, lane);
  sort_steps<16, 8>(k, lane);
  sort_steps<32, 16>(k, lane);
  sort_steps<64, 32>(k, lane);
  return __builtin_amdgcn_readlane(k, n - 1);
}

// A wave's best: lane i < top holds the i-th (by descending key, then ascending class).
struct TopList {
  int key = NO_KEY, idx = INT32_MAX;
  __device__ inline void insert(int k, int i, int lane, int top) {      // k, i uniform
    const int pos = __popcll(__ballot(lane < top && (key > k || (key == k && idx < i))));
    if (pos >= top) return;
    const int ku = dpp<0x138>(key), iu = dpp<0x138>(idx);  // one lane up (wave_shr:1)
    if (lane > pos) { key = ku; idx = iu; }
    if (lane == pos) { key = k; idx = i; }
  }
  __device__ inline int entry(int n) const { return __builtin_amdgcn_readlane(key, n); }
};
// the largest float below every value of key k: v > bar_below(k) is key(v) >= k, NaN included
__device__ inline float bar_below(int k) {
  if (k == NO_KEY) return __int_as_float(0x7FC00000);      // nothing is <= NaN
  return of_key(k == 0 ? -2 : k - 1);                      // -1 is the key that -0 does not have
}

struct ScoreArgs {
  const void* logits;
  const int64_t* tokens;
  float *logp, *entropy, *stat, *top_logp, *ws;
  int64_t* top_ids;
  int64_t ld, ld_tok, tok_sub, rows, V, ld_logp, ld_ent, seg_len;
  int top, segs;
};

// how many of n (key, idx) pairs in shared memory stand in front of `me`
__device__ inline int rank_of(int2 me, const int2* cand, int n) {
  int rank = 0;
#pragma unroll 8
  for (int o = 0; o < n; ++o) rank += cand[o].x > me.x || (cand[o].x == me.x && cand[o].y < me.y);
  return rank;
}

// the class asked for and its logit: two loads one after the other, which start with the row's own, not at its end
template <typename T> struct Asked {
  int64_t y = -1;
  bool known = false;
  T x = {};
  __device__ inline void ask(const ScoreArgs& a, int64_t row) {
    if (a.tokens) y = a.tokens[row * a.ld_tok] - a.tok_sub;
  }
  __device__ inline void fetch(const ScoreArgs& a, int64_t row) {
    known = y >= 0 && y < a.V;
    if (known) x = reinterpret_cast<const T*>(a.logits)[row * a.ld + y];
  }
};

// what is known of a whole row -> its results.  cand: n (key, idx) pairs in shared memory, of which the best `top` are taken.
template <typename T>
__device__ inline void finish_row(const ScoreArgs& a, int64_t row, const Sums& s, const Asked<T>& own, const int2* cand, int n, int tid, int threads) {
  const float L = logf(s.l);
  const bool none = s.l == 0.f;                            // -inf everywhere
  if (tid == 0) {
    float lp = 0.f;
    if (own.known) lp = none ? -INFINITY : s.l != s.l ? s.l : value_of(own.x) - s.m - L;
    a.logp[row * a.ld_logp] = lp;
    a.entropy[row * a.ld_ent] = none ? 0.f : L - s.t / s.l;
    if (a.stat) {
      a.stat[2 * row] = s.m;
      a.stat[2 * row + 1] = L;
    }
  }
  for (int c = tid; c < n; c += threads) {
    const int2 me = cand[c];
    if (me.x == NO_KEY) continue;
    const int rank = rank_of(me, cand, n);
    if (rank < a.top) {
      a.top_ids[row * a.top + rank] = me.y;
      a.top_logp[row * a.top + rank] = none ? -INFINITY : s.l != s.l ? s.l : of_key(me.x) - s.m - L;
    }
  }
}

// W waves share a row (or one part of it); W == 1: a block has four rows.
template <typename T, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void score_kernel(ScoreArgs a) {
  constexpr int NV = Vec<T>::N, H = 8 / NV;
  __shared__ float sums[W == 1 ? 4 : W][3];
  __shared__ int2 cand[W == 1 ? 4 : W][64];
  // W > 1: each full wave's `share`-th best key so far.  The shares are `top` values, so `top` values of the row reach the least of
  // them; a stale one is only lower, so the waves do not wait for each other to read them
  __shared__ int pub[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  const int kw = W == 1 ? 0 : wave;
  const bool live = row < a.rows;
  const int seg = blockIdx.y;
  Sums s;
  TopList top;
  Asked<T> asked;
  if (a.segs == 1 && live) asked.ask(a, row);
  if (live) {
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
    const int64_t c0 = seg * a.seg_len < a.V ? seg * a.seg_len : a.V, c1 = c0 + a.seg_len < a.V ? c0 + a.seg_len : a.V;
    int64_t head = ((16 - ((uintptr_t)(x + c0) & 15)) & 15) / sizeof(T);              // values up to a 16-byte border
    if (head > c1 - c0) head = c1 - c0;
    const int64_t body = (c1 - c0 - head) / NV, tail = c0 + head + body * NV;
    // waves that begin with 64 vectors share the bar; one with fewer would hold it down (2745 classes in two parts: 76 us with it)
    const int full = W == 1 || body < 128 ? 1 : body < W * 64 ? (int)(body >> 6) : W;
    const int share = (a.top + full - 1) / full;
    // Enters what of v[0 .. N) (lane o's values are classes base + o * N ..) can be among the best.  `own`: the last entry of the
    // wave's list; what equals it is a higher class than all entries and stays out.  `floor`: a key that at least `top` values of
    // the row reach; what equals it may still count.
    int own = NO_KEY, floor = NO_KEY;
    float bar = __int_as_float(0x7FC00000);
    auto set_bar = [&]() { bar = floor > own ? bar_below(floor) : own == NO_KEY ? __int_as_float(0x7FC00000) : of_key(own); };
    auto enter = [&](auto& v, float vm, bool in, int base) {
      constexpr int N = sizeof(v) / sizeof(float);
      const bool odd = s.l != s.l;                         // a NaN went by: the maximum may have passed over it
      if (!__any(in && (odd || !(vm <= bar)))) return;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        uint64_t todo = __ballot(in && !(v[e] <= bar));
        if (!todo) continue;
        const int k = key_of(v[e]);
        while (todo) {
          const int o = __ffsll((unsigned long long)todo) - 1;
          todo &= todo - 1;
          top.insert(__builtin_amdgcn_readlane(k, o), base + o * N + e, lane, a.top);
        }
      }
      own = top.entry(a.top - 1);
      if (W > 1 && kw < full) {
        const int q = top.entry(share - 1);
        if (lane == 0 && q != NO_KEY) __hip_atomic_store(&pub[wave], q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      set_bar();
    };
    auto single = [&](int64_t c0, int n) {                 // one value a lane
      const bool in = lane < n;
      float v[1] = {in ? value_of(x[c0 + lane]) : -INFINITY};
      if (in) {
        if (v[0] > s.m) s.grow(v[0]);
        s.add(v[0]);
      }
      if (a.top) enter(v, v[0], in, (int)c0);
    };
    const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + c0 + head);
    if (kw == 0 && head) single(c0, (int)head);
    bool opening = a.top > 0;
    // eight values a lane and step, the next eight in flight meanwhile (sixteen cost 16-bit logits their occupancy: 4096 x 32000
    // bf16 with 4 alternatives 100 us against 91)
    constexpr int64_t STEP = (int64_t)W * 64;
    int64_t i0 = (int64_t)kw * 64;
    uint4 ahead[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      ahead[h] = make_uint4(0, 0, 0, 0);
      if (i0 + h * STEP + lane < body) ahead[h] = *reinterpret_cast<const uint4*>(xv + i0 + h * STEP + lane);
    }
    if (a.segs == 1) asked.fetch(a, row);
    for (; i0 < body || opening; i0 += H * STEP) {
      float v[H][NV];
      float vm[H], least = INFINITY;
      bool in[H];
      const bool whole = i0 + (H - 1) * STEP + 64 <= body; // every lane has its values: the same for all of them
#pragma unroll
      for (int h = 0; h < H; ++h) {
        vm[h] = -INFINITY;
        in[h] = whole || i0 + h * STEP + lane < body;
        Vec<T> t;
        *reinterpret_cast<uint4*>(t.x) = ahead[h];
#pragma unroll
        for (int e = 0; e < NV; ++e) v[h][e] = value_of(t.x[e]);
      }
      if (!whole) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
          for (int e = 0; e < NV; ++e) v[h][e] = in[h] ? v[h][e] : -INFINITY;
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int e = 0; e < NV; ++e) {
          vm[h] = fmaxf(vm[h], v[h][e]);
          least = fminf(least, v[h][e]);
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (i0 + (H + h) * STEP + lane < body) ahead[h] = *reinterpret_cast<const uint4*>(xv + i0 + (H + h) * STEP + lane);
      const float both = fmaxf(vm[0], vm[H - 1]);
      if (both > s.m) s.grow(both);
      if (__all(least > -INFINITY && s.m < 1e30f && s.m > -INFINITY)) {       // else more care: -inf, or a difference that overflows to it, adds 0, not 0 * inf
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
          for (int e = 0; e < NV; ++e) s.add_finite(v[h][e]);
        }
      } else {
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
          for (int e = 0; e < NV; ++e) s.add(v[h][e]);
        }
      }
      if (a.top) {
        if (opening) {                                     // every wave of the block comes by here once
          const int q = kw < full ? nth_key(key_of(both), lane, share) : INT32_MAX;
          if (W > 1) {
            if (lane == 0) __hip_atomic_store(&pub[wave], q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __syncthreads();
          } else {
            floor = q;
            set_bar();
          }
          opening = false;
        }
        const bool odd = s.l != s.l;                       // a NaN went by: the maximum may have passed over it
        if (__any(odd || !(both <= bar))) {
          if (W > 1) {                                     // how far the others are is only looked up when it matters
            int f = INT32_MAX;
#pragma unroll
            for (int w = 0; w < W; ++w) f = min(f, __hip_atomic_load(&pub[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            if (f > floor) {
              floor = f;
              set_bar();
            }
          }
#pragma unroll
          for (int h = 0; h < H; ++h) enter(v[h], vm[h], in[h], (int)(c0 + head + (i0 + h * STEP) * NV));
        }
      }
    }
    if (kw == 0 && tail < c1) single(tail, (int)(c1 - tail));
  }
  s.over_wave(lane);
  if (lane == 0) { sums[wave][0] = s.m; sums[wave][1] = s.l; sums[wave][2] = s.t; }
  if (lane < a.top) cand[W == 1 ? wave : 0][W == 1 ? lane : wave * a.top + lane] = make_int2(top.key, top.idx);
  __syncthreads();
  if (!live) return;
  Sums all;
  if (W == 1) {
    all.m = sums[wave][0]; all.l = sums[wave][1]; all.t = sums[wave][2];
  } else {
    for (int w = 0; w < W; ++w) all.join(sums[w][0], sums[w][1], sums[w][2]);
  }
  const int n = W == 1 ? a.top : W * a.top, tid = W == 1 ? lane : (int)threadIdx.x, threads = W == 1 ? 64 : 64 * W;
  const int2* c = cand[W == 1 ? wave : 0];
  if (a.segs == 1) {
    finish_row<T>(a, row, all, asked, c, n, tid, threads);
    return;
  }
  // workspace: the parts' best (key, idx), then {m, l, t} of every part
  const int64_t at = row * a.segs + seg;
  float* part = a.ws + a.rows * a.segs * 2 * a.top + at * 3;
  if (tid == 0) { part[0] = all.m; part[1] = all.l; part[2] = all.t; }
  int2* best = reinterpret_cast<int2*>(a.ws) + at * a.top;
  for (int i = tid; i < a.top; i += threads) best[i] = make_int2(NO_KEY, 0);
  __syncthreads();                                                      // W > 1 whenever segs > 1: the whole block is here
  for (int i = tid; i < n; i += threads) {
    const int2 me = c[i];
    if (me.x == NO_KEY) continue;
    const int rank = rank_of(me, c, n);
    if (rank < a.top) best[rank] = me;
  }
}

// Joins the parts of a row: a block a row, a thread an entry of the parts' lists.  The lists are sorted, so if `lists` of them have
// an entry j that reaches a bar, lists * j values do: what stays below the bar of lists * j >= top cannot be among the best.  What is
// left (few more than `top`) is ranked all against all; only where it is more than the block's threads (equal logits) do the waves
// go through it with a sorted list each.  (Against going through all entries with sorted lists, whole calls: 100003 classes fp16, one
// row, 20 / 64 alternatives 35 / 98 -> 23 / 53 us, 3 rows with 8: this kernel 8.7 -> 5.4 us.)
template <typename T>
__global__ __launch_bounds__(256) void score_join_kernel(ScoreArgs a) {
  __shared__ float sums[4][3];
  __shared__ int2 cand[4 * 64];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.segs * a.top;
  const int2* best = reinterpret_cast<const int2*>(a.ws) + row * n;
  const float* part = a.ws + a.rows * a.segs * 2 * a.top + row * a.segs * 3;
  if (tid == 0) count = 0;
  Asked<T> asked;
  asked.ask(a, row);
  const int lists = a.segs < 64 ? a.segs : 64, j = (a.top + lists - 1) / lists;
  int bar = NO_KEY;
  int2 first = make_int2(NO_KEY, 0);
  if (a.top) {
    if (lane < lists) bar = best[lane * a.top + j - 1].x;
    if (tid < n) first = best[tid];
  }
  asked.fetch(a, row);
  Sums s;
  for (int g = tid; g < a.segs; g += 256) s.join(part[(int64_t)g * 3], part[(int64_t)g * 3 + 1], part[(int64_t)g * 3 + 2]);
  s.over_wave(lane);
  if (lane == 0) { sums[wave][0] = s.m; sums[wave][1] = s.l; sums[wave][2] = s.t; }
  if (a.top) bar = nth_key(bar, lane, (a.top + j - 1) / j);
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const int2 me = i == tid ? first : best[i];
    if (me.x == NO_KEY || me.x < bar) continue;
    const int at = __hip_atomic_fetch_add(&count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    if (at < 256) cand[at] = me;
  }
  __syncthreads();
  Sums all;
  for (int w = 0; w < 4; ++w) all.join(sums[w][0], sums[w][1], sums[w][2]);
  int left = count;
  if (left > 256) {
    __syncthreads();                                       // all have read `count`, and none reads `cand` before the next barrier
    TopList top;
    for (int i0 = 0; i0 < n; i0 += 256) {
      const int2 e = i0 + tid < n ? best[i0 + tid] : make_int2(NO_KEY, 0);
      const int last = top.entry(a.top - 1);
      uint64_t todo = __ballot(e.x != NO_KEY && e.x >= (last > bar ? last : bar));
      while (todo) {
        const int o = __ffsll((unsigned long long)todo) - 1;
        todo &= todo - 1;
        top.insert(__builtin_amdgcn_readlane(e.x, o), __builtin_amdgcn_readlane(e.y, o), lane, a.top);
      }
    }
    if (lane < a.top) cand[wave * a.top + lane] = make_int2(top.key, top.idx);
    left = 4 * a.top;
    __syncthreads();
  }
  finish_row<T>(a, row, all, asked, cand, left, tid, 256);
}

// Rows of at most 256 classes: 32 lanes a row, E values a lane, everything in registers.  The alternatives are taken out one
// after the other, a maximum over the lanes each.
__device__ inline float max32(float x) {                   // over the 32 lanes of a half wave
  x = fmaxf(x, dppf<0xB1>(x));
  x = fmaxf(x, dppf<0x4E>(x));
  x = fmaxf(x, dppf<0x141>(x));
  x = fmaxf(x, dppf<0x140>(x));
  const uintx2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float sum32(float x) {
  x += dppf<0xB1>(x);
  x += dppf<0x4E>(x);
  x += dppf<0x141>(x);
  x += dppf<0x140>(x);
  const uintx2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline void better(int& k, int& i, int k2, int i2) {
  const bool b = k2 > k || (k2 == k && i2 < i);
  k = b ? k2 : k;
  i = b ? i2 : i;
}
__device__ inline void best32(int& k, int& i) {
  better(k, i, dpp<0xB1>(k), dpp<0xB1>(i));
  better(k, i, dpp<0x4E>(k), dpp<0x4E>(i));
  better(k, i, dpp<0x141>(k), dpp<0x141>(i));
  better(k, i, dpp<0x140>(k), dpp<0x140>(i));
  const uintx2 rk = __builtin_amdgcn_permlane16_swap((uint32_t)k, (uint32_t)k, false, false);
  const uintx2 ri = __builtin_amdgcn_permlane16_swap((uint32_t)i, (uint32_t)i, false, false);
  k = (int)rk[0];
  i = (int)ri[0];
  better(k, i, (int)rk[1], (int)ri[1]);
}

// (key, class) pairs of the 32 lanes of a half wave in descending order: a bitonic sort, 15 steps
template <int SIZE, int D> __device__ inline void sort_pairs(int& k, int& i, int lane) {
  const int k2 = lane_xor<D>(k, lane), i2 = lane_xor<D>(i, lane);
  const bool mine = k > k2 || (k == k2 && i < i2), up = (lane & 31 & SIZE) != 0, low = (lane & D) == 0;
  const bool keep = mine == (low != up);
  k = keep ? k : k2;
  i = keep ? i : i2;
  if constexpr (D > 1) sort_pairs<SIZE, D / 2>(k, i, lane);
}

template <typename T, int E>
__global__ __launch_bounds__(256) void score_short_kernel(ScoreArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const bool live = row < a.rows;                          // both halves of a wave go through the same steps
  const T* x = reinterpret_cast<const T*>(a.logits) + (live ? row : 0) * a.ld;
  float v[E];
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = lane + 32 * e;
    v[e] = c < a.V ? value_of(x[c]) : -INFINITY;
    m = fmaxf(m, v[e]);
  }
  const int64_t y = a.tokens && live ? a.tokens[row * a.ld_tok] - a.tok_sub : -1;
  m = max32(m);
  float l = 0.f, t = 0.f;
  const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = v[e] - ms, w = __builtin_amdgcn_exp2f(d * LOG2E);
    l += w;
    t = fmaf(w, fmaxf(d, -1e30f), t);
  }
  l = sum32(l);
  t = sum32(t);
  const bool none = l == 0.f;
  const float L = logf(l);
  const bool token = y >= 0 && y < a.V;
  float lp = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e == (token ? (int)y : -1)) lp = none ? -INFINITY : l != l ? l : v[e] - m - L;
  if (live && (token ? lane == ((int)y & 31) : lane == 0)) a.logp[row * a.ld_logp] = lp;
  if (live && lane == 0) {
    a.entropy[row * a.ld_ent] = none ? 0.f : L - t / l;
    if (a.stat) {
      a.stat[2 * row] = m;
      a.stat[2 * row + 1] = L;
    }
  }
  if (a.top == 0) return;
  if (E == 1) {                                            // one value a lane: sorted at once (63000 x 25, 20 alternatives: 53 -> 17 us)
    int k = lane < a.V ? key_of(v[0]) : NO_KEY, i = lane;
    sort_pairs<2, 1>(k, i, lane);
    sort_pairs<4, 2>(k, i, lane);
    sort_pairs<8, 4>(k, i, lane);
    sort_pairs<16, 8>(k, i, lane);
    sort_pairs<32, 16>(k, i, lane);
    if (live && lane < a.top) {
      a.top_ids[row * a.top + lane] = i;
      a.top_logp[row * a.top + lane] = none ? -INFINITY : l != l ? l : of_key(k) - m - L;
    }
    return;
  }
  int key[E];
#pragma unroll
  for (int e = 0; e < E; ++e) key[e] = lane + 32 * e < a.V ? key_of(v[e]) : NO_KEY;
  for (int n0 = 0; n0 < a.top; n0 += 32) {                 // lane i keeps alternative n0 + i
    int mk = NO_KEY, mi = 0;
    const int n1 = a.top - n0 < 32 ? a.top - n0 : 32;
    for (int n = 0; n < n1; ++n) {
      int k = NO_KEY, i = INT32_MAX;
#pragma unroll
      for (int e = 0; e < E; ++e) better(k, i, key[e], lane + 32 * e);
      best32(k, i);
      if (lane == n) { mk = k; mi = i; }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + 32 * e == i) key[e] = NO_KEY;
    }
    if (live && lane < n1) {
      a.top_ids[row * a.top + n0 + lane] = mi;
      a.top_logp[row * a.top + n0 + lane] = none ? -INFINITY : l != l ? l : of_key(mk) - m - L;
    }
  }
}

// ------------------------------------------------------------------------------------------------ gradient
struct ScoreBwdArgs {
  const void* logits;
  void* dx;
  const int64_t *tokens, *top_ids;
  const float *stat, *entropy, *g_logp, *g_entropy, *g_top;
  int64_t ld, ld_tok, tok_sub, rows, V, ld_ent, seg_len;
  int top;
};

constexpr float NO_WEIGHT = -128.f;                        // e^-128 is 0 in fp32: below it ln p only has to stay finite when g_H multiplies it

// One read and one write a value: p = exp((x - M) - L), dx = -p (pull + g_H (ln p + H)) with pull = g_l + sum g_t; the few
// classes that are the token or an alternative get their own gradient on top, added by the thread that holds the class.
template <typename T>
__global__ __launch_bounds__(256) void score_bwd_kernel(ScoreBwdArgs a) {
  constexpr int NV = Vec<T>::N;
  __shared__ float extra[65];
  __shared__ int64_t which[65];
  __shared__ float pull_s;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t c0 = (int64_t)blockIdx.y * a.seg_len, c1 = c0 + a.seg_len < a.V ? c0 + a.seg_len : a.V;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  T* dx = reinterpret_cast<T*>(a.dx) + row * a.V;
  if (tid < 64) {
    int64_t y = a.tokens && a.g_logp ? a.tokens[row * a.ld_tok] - a.tok_sub : -1;
    if (y >= a.V) y = -1;
    const float gl = y >= 0 ? a.g_logp[row] : 0.f;
    const bool alt = a.g_top && tid < a.top;
    const float gt = alt ? a.g_top[row * a.top + tid] : 0.f;
    const int64_t id = alt ? a.top_ids[row * a.top + tid] : -1;
    const bool same = alt && id == y;                                   // the token is an alternative too
    if (tid < 64) { which[1 + tid] = id; extra[1 + tid] = gt + (same ? gl : 0.f); }
    const bool any = __ballot(same) != 0;
    const float sum = wave_sum(gt);
    if (tid == 0) { which[0] = any ? -1 : y; extra[0] = gl; pull_s = gl + sum; }
  }
  __syncthreads();
  const float pull = pull_s, M = a.stat[2 * row], L = a.stat[2 * row + 1], H = a.entropy[row * a.ld_ent];
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const bool none = M == -INFINITY && L == -INFINITY;                   // a row of -inf: no gradient
  auto grad = [&](float v) {
    const float lp = (v - M) - L;
    const float p = __builtin_amdgcn_exp2f(lp * LOG2E);
    const float r = -p * (pull + gh * (fmaxf(lp, NO_WEIGHT) + H));
    return none || v == -INFINITY ? 0.f : r;
  };
  int64_t head = ((16 - ((uintptr_t)(x + c0) & 15)) & 15) / sizeof(T);
  if (head > c1 - c0) head = c1 - c0;
  const int64_t body = (c1 - c0 - head) / NV, tail = c0 + head + body * NV;
  const bool even = (((uintptr_t)(dx + c0 + head)) & 15) == 0;          // rows of x and dx on the same 16-byte phase
  for (int64_t c = c0 + tid; c < c0 + head; c += 256) put(dx + c, grad(value_of(x[c])));
  for (int64_t i = tid; i < body; i += 256) {
    Vec<T> t;
    *reinterpret_cast<uint4*>(t.x) = *reinterpret_cast<const uint4*>(x + c0 + head + i * NV);
#pragma unroll
    for (int e = 0; e < NV; ++e) put(&t.x[e], grad(value_of(t.x[e])));
    T* d = dx + c0 + head + i * NV;
    if (even) {
      *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(t.x);
    } else {
#pragma unroll
      for (int e = 0; e < NV; ++e) d[e] = t.x[e];
    }
  }
  for (int64_t c = tail + tid; c < c1; c += 256) put(dx + c, grad(value_of(x[c])));
  __syncthreads();                                                      // the rewrites below come after the stores above
  if (tid < 65 && tid <= a.top) {
    const int64_t c = which[tid];
    if (c >= c0 && c < c1) {
      const float v = value_of(x[c]);
      if (!none && v != -INFINITY) put(dx + c, grad(v) + extra[tid]);
    }
  }
}

// Rows of at most 256 classes: 32 lanes a row; what a class gets of its own is added up in shared memory first.
template <typename T>
__global__ __launch_bounds__(256) void score_short_bwd_kernel(ScoreBwdArgs a) {
  __shared__ float own[8][SHORT];
  const int lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 8 + slot;
  const bool live = row < a.rows;
  for (int c = lane; c < a.V; c += 32) own[slot][c] = 0.f;
  __syncthreads();
  float pull = 0.f;
  if (live && a.g_logp && a.tokens) {
    const int64_t y = a.tokens[row * a.ld_tok] - a.tok_sub;
    if (y >= 0 && y < a.V) {
      pull = a.g_logp[row];
      if (lane == 0) own[slot][y] = pull;
    }
  }
  __syncthreads();
  float sum = 0.f;
  if (live)
    for (int t = lane; t < a.top; t += 32) {                            // the alternatives are different classes
      const float g = a.g_top[row * a.top + t];
      const int64_t id = a.top_ids[row * a.top + t];
      if (id >= 0 && id < a.V) own[slot][id] += g;
      sum += g;
    }
  pull += sum32(sum);
  __syncthreads();
  if (!live) return;
  const float M = a.stat[2 * row], L = a.stat[2 * row + 1], H = a.entropy[row * a.ld_ent], gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const bool none = M == -INFINITY && L == -INFINITY;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  T* dx = reinterpret_cast<T*>(a.dx) + row * a.V;
  for (int c = lane; c < a.V; c += 32) {
    const float v = value_of(x[c]), lp = (v - M) - L, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    const float r = own[slot][c] - p * (pull + gh * (fmaxf(lp, NO_WEIGHT) + H));
    put(dx + c, none || v == -INFINITY ? 0.f : r);
  }
}

int type_bytes(int dtype) { return dtype == TVAE_F32 ? 4 : dtype == TVAE_BF16 || dtype == TVAE_F16 ? 2 : 0; }

template <typename T>
void launch_score(const ScoreArgs& a, hipStream_t s) {
  if (a.V <= SHORT) {
    const dim3 grid((unsigned)((a.rows + 7) / 8)), block(256);
    if (a.V <= 32) hipLaunchKernelGGL((score_short_kernel<T, 1>), grid, block, 0, s, a);
    else if (a.V <= 64) hipLaunchKernelGGL((score_short_kernel<T, 2>), grid, block, 0, s, a);
    else if (a.V <= 128) hipLaunchKernelGGL((score_short_kernel<T, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((score_short_kernel<T, 8>), grid, block, 0, s, a);
    return;
  }
  // a wave a row where the rows are many or short, else a block: the start and the end of a row are then paid once instead of four
  // times (bf16, 4 alternatives, wave / block: 20000 x 4000 58 / 92 us, 4096 x 32000 74 / 83, 2048 x 16000 29 / 28; fp32, 20
  // alternatives: 1024 x 4000 25 / 21, 500 x 600 13 / 42)
  if (a.segs == 1 && (a.V <= 2048 || a.rows >= 4096)) hipLaunchKernelGGL((score_kernel<T, 1>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((score_kernel<T, 4>), dim3((unsigned)a.rows, a.segs), dim3(256), 0, s, a);
  if (a.segs > 1) hipLaunchKernelGGL((score_join_kernel<T>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
}

template <typename T>
void launch_bwd(const ScoreBwdArgs& a, hipStream_t s) {
  if (a.V <= SHORT) hipLaunchKernelGGL(score_short_bwd_kernel<T>, dim3((unsigned)((a.rows + 7) / 8)), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(score_bwd_kernel<T>, dim3((unsigned)a.rows, (unsigned)((a.V + a.seg_len - 1) / a.seg_len)), dim3(256), 0, s, a);
}

}  // namespace

extern "C" int tvae_token_logp(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t ld_tok, int64_t tok_sub,
                               int64_t rows, int64_t V, int top, float* logp, int64_t ld_logp, float* entropy, int64_t ld_ent,
                               float* stat, float* top_logp, int64_t* top_ids, int segs, float* ws, void* stream) {
  TVAE_CHECK(rows >= 0 && V >= 1 && V <= INT32_MAX && ld >= V && top >= 0 && top <= 64 && top <= V, TVAE_E_SHAPE,
             "tvae_token_logp: need rows >= 0, 1 <= V <= ld, top in [0, min(V, 64)] (rows=%lld V=%lld ld=%lld top=%d)", (long long)rows,
             (long long)V, (long long)ld, top);
  TVAE_CHECK(type_bytes(dtype), TVAE_E_DTYPE, "tvae_token_logp: dtype %d is not TVAE_F32, TVAE_BF16 or TVAE_F16", dtype);
  if (rows == 0) return TVAE_OK;
  TVAE_CHECK(logits && logp && entropy && (top == 0 || (top_logp && top_ids)), TVAE_E_NULL, "tvae_token_logp: null pointer");
  TVAE_CHECK((uintptr_t)logits % type_bytes(dtype) == 0, TVAE_E_SHAPE, "tvae_token_logp: logits are not aligned to their type");
  TVAE_CHECK(segs >= 1 && segs <= 1024 && (segs == 1 || (ws && (uintptr_t)ws % 8 == 0)), TVAE_E_SHAPE,
             "tvae_token_logp: 1 .. 1024 parts, more than one with a workspace aligned to 8 bytes");
  TVAE_CHECK((V <= SHORT ? (rows + 7) / 8 : rows) <= MAX_BLOCKS, TVAE_E_SHAPE, "tvae_token_logp: too many rows in one call (%lld)", (long long)rows);
  const int64_t seg_len = ((V + segs - 1) / segs + 7) / 8 * 8;
  ScoreArgs a = {logits, tokens, logp, entropy, stat, top_logp, ws, top_ids, ld, ld_tok, tok_sub, rows, V, ld_logp, ld_ent, seg_len, top, segs};
  if (dtype == TVAE_F32) launch_score<float>(a, (hipStream_t)stream);
  else if (dtype == TVAE_BF16) launch_score<B16>(a, (hipStream_t)stream);
  else launch_score<F16>(a, (hipStream_t)stream);
  TVAE_LAUNCH_CHECK("tvae_token_logp");
  return TVAE_OK;
}

extern "C" int tvae_token_logp_bwd(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t ld_tok, int64_t tok_sub,
                                   int64_t rows, int64_t V, int top, const float* stat, const float* entropy, int64_t ld_ent,
                                   const int64_t* top_ids, const float* g_logp, const float* g_entropy, const float* g_top, void* dx,
                                   void* stream) {
  TVAE_CHECK(rows >= 0 && V >= 1 && V <= INT32_MAX && ld >= V && top >= 0 && top <= 64 && top <= V, TVAE_E_SHAPE,
             "tvae_token_logp_bwd: need rows >= 0, 1 <= V <= ld, top in [0, min(V, 64)] (rows=%lld V=%lld ld=%lld top=%d)", (long long)rows,
             (long long)V, (long long)ld, top);
  TVAE_CHECK(type_bytes(dtype), TVAE_E_DTYPE, "tvae_token_logp_bwd: dtype %d is not TVAE_F32, TVAE_BF16 or TVAE_F16", dtype);
  if (rows == 0) return TVAE_OK;
  TVAE_CHECK(logits && stat && entropy && dx && (!g_top || top == 0 || top_ids), TVAE_E_NULL, "tvae_token_logp_bwd: null pointer");
  TVAE_CHECK((uintptr_t)logits % type_bytes(dtype) == 0 && (uintptr_t)dx % type_bytes(dtype) == 0, TVAE_E_SHAPE,
             "tvae_token_logp_bwd: logits or dx are not aligned to their type");
  TVAE_CHECK((V <= SHORT ? (rows + 7) / 8 : rows) <= MAX_BLOCKS, TVAE_E_SHAPE, "tvae_token_logp_bwd: too many rows in one call (%lld)", (long long)rows);
  const int64_t seg_len = 16384;
  TVAE_CHECK((V + seg_len - 1) / seg_len <= 65535, TVAE_E_SHAPE, "tvae_token_logp_bwd: V too large (%lld)", (long long)V);
  ScoreBwdArgs a = {logits, dx, tokens, top_ids, stat, entropy, g_logp, g_entropy, g_top, ld, ld_tok, tok_sub, rows, V, ld_ent, seg_len,
                    g_top ? top : 0};
  if (dtype == TVAE_F32) launch_bwd<float>(a, (hipStream_t)stream);
  else if (dtype == TVAE_BF16) launch_bwd<B16>(a, (hipStream_t)stream);
  else launch_bwd<F16>(a, (hipStream_t)stream);
  TVAE_LAUNCH_CHECK("tvae_token_logp_bwd");
  return TVAE_OK;
}
