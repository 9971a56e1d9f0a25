// Layer norm over the rows of a matrix, and its gradients.
//
//   mu = mean(x), s2 = mean((x - mu)^2), r = 1 / sqrt(s2 + eps), xh = (x - mu) r,  y = xh w + b
//   q = dy w,  dx = r (q - mean(q) - xh mean(q xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Rows are fp32, bf16 or fp16, the weights fp32 or of the rows' type; everything between is fp32 and each
// result is rounded once.  The variance is taken about the mean (two passes over registers): E[x^2] - mu^2
// would cancel for rows whose mean is large against their spread.
//
// Bound: HBM.  Forward 2 e bytes an element, backward 3 e (e = element size), ~8 and ~14 flop an element.  So
// a row is read once and stays in registers, as the 16-byte vectors that it came in: TPR threads hold it (16,
// or 64 to 1024; row_threads_fwd / row_threads_bwd), longer rows are read again, from L2 for the most part.
//
// Measured (MI355X; a copy of 1 GiB runs at 5.3 TB/s on it): forward 256000 x 800 fp32 284 us = 5.8 TB/s, 8192 x 4096
// bf16 24, 4000 x 800 fp32 6, one row 1.8; backward of the first three 436 (5.6 TB/s), 41 and 12 us with the slabs' sum.
// 100 M elements, 100 to 16384 columns: forward 4.2 to 5.2 TB/s in 16 bits, 5.0 to 5.7 in 32; backward 3.9 to 5.1 and
// 4.7 to 5.5, lowest where a row fills its threads badly (513, 1200 columns).  100 M elements in longer rows: forward
// 4.4 TB/s at 20000 to 30000 fp32 columns, 3.3 to 3.5 at 40000 to 50000 of 16 bits (8 vectors a thread), 2.3 at 100000 of
// either, read again twice; backward 2.0 to 2.3 from 16385 on.
#include <type_traits>

#include "common.h"

namespace iadmm {

// 16 bytes of T in four words (elements of 16 bits as members would take a register each).
template <typename T> struct Pack {
  static constexpr int n = 16 / sizeof(T);
  uint32_t w[4];
};
template <typename T> IADMM_DEV float get(const Pack<T>& p, int j) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(p.w[j]);
  } else if constexpr (std::is_same<T, __bf16>::value) {
    return __uint_as_float(j & 1 ? p.w[j / 2] & 0xFFFF0000u : p.w[j / 2] << 16);
  } else {
    const uint16_t b = static_cast<uint16_t>(j & 1 ? p.w[j / 2] >> 16 : p.w[j / 2]);
    return static_cast<float>(__builtin_bit_cast(_Float16, b));
  }
}
template <typename T> IADMM_DEV void set(Pack<T>& p, const float (&v)[Pack<T>::n]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      p.w[k] = __float_as_uint(v[k]);
    } else {
      const T t[2] = {static_cast<T>(v[2 * k]), static_cast<T>(v[2 * k + 1])};
      __builtin_memcpy(&p.w[k], t, 4);
    }
  }
}

// Rows of odd length start at any multiple of the element size: the memory pipe takes 16-byte accesses there.
//
// Where a thread's vector would reach over the row's end (or lies behind it), it takes the row's last 16 bytes
// instead: every access is whole, and none has a branch of its own, which would keep a row's loads from being in
// flight together (8192 rows of 4096 bf16: 48 us with branches, 26 without).  The elements that its neighbours
// hold too are its first `dup`: they count in no sum, and their result is stored twice, with the same bits.
struct Place {
  uint32_t at;  // column of its first element
  int dup;
};
template <typename T> IADMM_DEV Place place(int c, int cols) {
  constexpr int V = Pack<T>::n;
  const int last = cols - V, at = c < last ? c : last;
  return Place{static_cast<uint32_t>(at), c - at};
}
// 16 bytes from element `at` (32 bits of offset beside a base that a wave shares: no arithmetic in 64 bits per access).
template <typename T> IADMM_DEV Pack<T> load_whole(const T* p, uint32_t at) {
  Pack<T> r;
  __builtin_memcpy(&r, reinterpret_cast<const char*>(p) + at * static_cast<uint32_t>(sizeof(T)), 16);
  return r;
}
template <typename T> IADMM_DEV void store_whole(T* p, uint32_t at, const Pack<T>& r) {
  __builtin_memcpy(reinterpret_cast<char*>(p) + at * static_cast<uint32_t>(sizeof(T)), &r, 16);
}

// n elements from p; what lies behind is 0.  For rows shorter than a vector and for the long rows' kernels.
template <typename T> IADMM_DEV Pack<T> load_pack(const T* p, int64_t n) {
  Pack<T> r;
  if (n >= Pack<T>::n) {
    __builtin_memcpy(&r, p, 16);
  } else {
    using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    const U* q = reinterpret_cast<const U*>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        r.w[k] = k < n ? q[k] : 0u;
      } else {
        r.w[k] = 2 * k < n ? q[2 * k] : 0u;
        if (2 * k + 1 < n) r.w[k] |= static_cast<uint32_t>(q[2 * k + 1]) << 16;
      }
    }
  }
  return r;
}
template <typename T> IADMM_DEV void store_pack(T* p, const Pack<T>& r, int64_t n) {
  if (n >= Pack<T>::n) {
    __builtin_memcpy(p, &r, 16);
  } else {
    using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    U* q = reinterpret_cast<U*>(p);
#pragma unroll
    for (int j = 0; j < Pack<T>::n; ++j)
      if (j < n) q[j] = static_cast<U>(sizeof(T) == 4 ? r.w[j * sizeof(T) / 4] : r.w[j / 2] >> (j & 1) * 16);
  }
}

// V weights from column c, of type T or fp32; `none` where there are none.  WHOLE: all within the row.  KIND: which
// of these it is, where the caller has asked already (outside its loop, whose loads a branch would keep apart).
enum { kAnyKind, kFloats, kSame };
template <typename T, bool WHOLE = false, int KIND = kAnyKind>
IADMM_DEV void load_weights(const void* w, bool f32, int64_t c, int64_t cols, float none, float* out) {
  constexpr int V = Pack<T>::n;
  const int64_t n = WHOLE ? V : cols - c;
  f32 = KIND == kFloats || (KIND == kAnyKind && f32);
  if (KIND == kAnyKind && !w) {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = none;
  } else if (sizeof(T) == 4 || f32) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      const float* p = static_cast<const float*>(w) + 4 * k;
      const Pack<float> a = WHOLE ? load_whole(p, static_cast<uint32_t>(c)) : load_pack(p + c, n - 4 * k);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[4 * k + j] = get(a, j);
    }
  } else {
    const T* p = static_cast<const T*>(w);
    const Pack<T> a = WHOLE ? load_whole(p, static_cast<uint32_t>(c)) : load_pack(p + c, n);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = get(a, j);
  }
}

// Sums of v over the TPR threads of a row, in every one of them.  Within 16 lanes and then a wave by adds whose second
// operand comes from another lane, a few cycles each (through LDS a step waits for some hundred); over the waves
// through LDS, `red` holding one value per wave of the workgroup; the caller alternates between two such arrays,
// so one barrier is enough (a wave writes an array again only after every wave has passed the other array's barrier).
template <int CTRL> IADMM_DEV float add_from(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int N> IADMM_DEV float sum_lanes(float v) {  // over N neighbours, up to 16, in each of them
  if (N >= 2) v = add_from<0xB1>(v);    // within quads: 1 lane apart,
  if (N >= 4) v = add_from<0x4E>(v);    // 2 lanes apart
  if (N >= 8) v = add_from<0x141>(v);   // half rows mirrored
  if (N >= 16) v = add_from<0x140>(v);  // rows mirrored
  return v;
}
// Over lanes 16, 32 and 48 apart: halves, then rows of 16, change places between a register and its copy.
IADMM_DEV float sum_rows16(float v) {
  const uint32_t a = __float_as_uint(v);
  const auto h = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t b = __float_as_uint(__uint_as_float(h[0]) + __uint_as_float(h[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
template <int TPR, int K> IADMM_DEV void row_sum(float (&v)[K], float* red) {
  static_assert(TPR == 16 || (TPR >= kWave && TPR <= 1024), "");
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = sum_lanes<16>(v[k]);
    if constexpr (TPR >= kWave) {
      v[k] = add_from<0x143>(add_from<0x142>(v[k]));  // row_bcast 15, 31: lane 63 has the wave's
      v[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v[k]), 63));
    }
  }
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    __syncthreads();
    const float* r = red + (wave / W * W + threadIdx.x % W) * K;
#pragma unroll
    for (int k = 0; k < K; ++k)
      v[k] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sum_lanes<W>(r[k]))));
  }
}

// What the threads of a wave share: their row's number, and the first column of their vector i (TPR < 64: of all rows).
template <int TPR> IADMM_DEV int shared(int v) { return TPR >= kWave ? __builtin_amdgcn_readfirstlane(v) : v; }
template <typename T, int TPR> IADMM_DEV int first_col(int i) {
  return (i * TPR + (TPR > kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x % TPR) : 0)) * Pack<T>::n;
}

struct LnFwd {
  int64_t rows, cols, ldx;
  const void *x, *w, *b;
  void* y;
  float *mean, *rstd;
  float eps;
  int w32;
};

// Forward.  Bound by HBM from some thousand rows on, by the launch and one trip to memory and back below.
// One row per TPR threads, NV vectors each; SHORT: rows shorter than a vector (TPR = 16, NV = 1).
template <typename T, int TPR, int NV, bool SHORT>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) ln_fwd_kernel(LnFwd a) {
  constexpr int V = Pack<T>::n, BLOCK = TPR > 256 ? TPR : 256, R = BLOCK / TPR;
  __shared__ float red[2][BLOCK / kWave];
  const int lane = threadIdx.x % TPR, cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  // (no loop over rows: the weights would be loaded before it and stay in 2 registers an element)
  const int64_t row = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * R + shared<TPR>(threadIdx.x / TPR);
  const bool on = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + (on ? row : 0) * a.ldx;
  Pack<T> p[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * V;
    p[i] = SHORT ? load_pack(x + c, cols - c) : load_whole(x, place<T>(c, cols).at);
  }
  // Vector by vector, so that a path has 8 + NV additions.  Whether element j of vector i counts only the row's last
  // vectors ask.
  auto sum = [&](auto term) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      float t = 0.0f;
      if ((i + 1) * TPR * V <= cols) {
#pragma unroll
        for (int j = 0; j < V; ++j) t += term(get(p[i], j));
      } else {
        const int dup = SHORT ? 0 : place<T>(c, cols).dup;
#pragma unroll
        for (int j = 0; j < V; ++j) t += j >= dup && j < (SHORT ? cols - c : V) ? term(get(p[i], j)) : 0.0f;
      }
      s += t;
    }
    return s;
  };
  float s[1] = {sum([](float v) { return v; })};
  row_sum<TPR, 1>(s, red[0]);
  const float mu = s[0] * inv;
  s[0] = sum([mu](float v) { return (v - mu) * (v - mu); });
  row_sum<TPR, 1>(s, red[1]);
  const float r = 1.0f / sqrtf(s[0] * inv + a.eps);
  if (!on) return;
  T* y = static_cast<T*>(a.y) + row * a.cols;
  auto finish = [&](auto kind) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      const uint32_t at = SHORT ? c : place<T>(c, cols).at;
      float w[V], b[V];
      load_weights<T, !SHORT, kind()>(a.w, a.w32, at, a.cols, 1.0f, w);
      load_weights<T, !SHORT, kind()>(a.b, a.w32, at, a.cols, 0.0f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = fmaf((get(p[i], j) - mu) * r, w[j], b[j]);
      set(p[i], w);
      if (SHORT) store_pack(y + at, p[i], cols - c);
      else if (c < cols) store_whole(y, at, p[i]);
    }
  };
  if (!a.w || !a.b || SHORT) finish(std::integral_constant<int, kAnyKind>());
  else if (sizeof(T) == 4 || a.w32) finish(std::integral_constant<int, kFloats>());
  else finish(std::integral_constant<int, kSame>());
  if (lane == 0 && a.mean) a.mean[row] = mu;
  if (lane == 0 && a.rstd) a.rstd[row] = r;
}

// Rows longer than the registers hold (32768 fp32, 65536 16-bit elements): a workgroup reads its row three times, 4 e bytes
// an element for 2 e, the second and third time from caches.  1000 x 100000: fp32 342 us, bf16 172 (2.3 TB/s of 2 e); 100
// rows of a million fp32 836, as only 100 of 256 CUs have one.
template <typename T> __global__ void __launch_bounds__(1024) ln_fwd_long_kernel(LnFwd a) {
  constexpr int V = Pack<T>::n, TPR = 1024;
  __shared__ float red[2][TPR / kWave];
  const float inv = 1.0f / static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.cols;
    float s[1] = {0.0f};
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.cols; c += TPR * V) {
      const Pack<T> p = load_pack(x + c, a.cols - c);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += get(p, j);
    }
    row_sum<TPR, 1>(s, red[0]);
    const float mu = s[0] * inv;
    s[0] = 0.0f;
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.cols; c += TPR * V) {
      const Pack<T> p = load_pack(x + c, a.cols - c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = c + j < a.cols ? get(p, j) - mu : 0.0f;
        s[0] = fmaf(d, d, s[0]);
      }
    }
    row_sum<TPR, 1>(s, red[1]);
    const float r = 1.0f / sqrtf(s[0] * inv + a.eps);
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.cols; c += TPR * V) {
      Pack<T> p = load_pack(x + c, a.cols - c);
      float w[V], b[V];
      load_weights<T>(a.w, a.w32, c, a.cols, 1.0f, w);
      load_weights<T>(a.b, a.w32, c, a.cols, 0.0f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = fmaf((get(p, j) - mu) * r, w[j], b[j]);
      set(p, w);
      store_pack(y + c, p, a.cols - c);
    }
    if (threadIdx.x == 0 && a.mean) a.mean[row] = mu;
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = r;
  }
}

struct LnBwd {
  int64_t rows, cols, lddy, ldx;
  const void *dy, *x, *w;
  const float *mean, *rstd;
  void* dx;     // or null
  float* slab;  // [gridDim.x][2][cols]: each workgroup's share of dw and db; or null
  int w32;
  void *dw, *db;  // of a workgroup that has all rows: it writes them itself; or null
};

// A workgroup of BLOCK threads takes BLOCK / TPR rows at a time, 1024 threads per CU at most: dw and db grow in
// registers over all its rows, meet once in LDS and leave as one slab, which keeps the slabs' traffic small beside
// the rows' (512 slabs at most).  These sums are fp32, the slabs' are 64 bits: at 256000 x 800 a thread adds 125 rows, and
// dw and db are off by 2e-7 of their size.  Up to 64 threads a row there is no barrier among them, and a wave waits for its
// own rows alone.
template <typename T, int TPR, int NV, int BLOCK, bool SHORT> __global__ void __launch_bounds__(BLOCK) ln_bwd_kernel(LnBwd a) {
  constexpr int V = Pack<T>::n, R = BLOCK / TPR, E = NV * V, SPAN = (TPR < kWave ? TPR : kWave) * V;
  extern __shared__ float lds[];  // [groups][TPR * E]
  __shared__ float red[2][2 * BLOCK / kWave];
  const int lane = threadIdx.x % TPR, group = shared<TPR>(threadIdx.x / TPR), cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  // The weights stay in registers (read again for each row and pass, a wave waits for them four times: 24414 x 4096
  // bf16 136 us, kept 118); at 24 elements a thread they would take those of four waves.
  constexpr bool KEEP = E <= 16;
  float dw[E], db[E], w[KEEP ? NV : 1][V];
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.0f;
  uint32_t again = 0;
  auto weights = [&](int i, float (&to)[V]) {
    const int c = (i * TPR + lane) * V;
    load_weights<T, !SHORT>(a.w, a.w32, (SHORT ? c : place<T>(c, cols).at) + again, cols, 1.0f, to);
  };
  if constexpr (KEEP)
#pragma unroll
    for (int i = 0; i < NV; ++i) weights(i, w[i]);
  int odd = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * R; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * R, odd ^= 1) {
    const int64_t row = row0 + group;
    const bool on = row < a.rows;
    const int64_t from = on ? row : 0;
    const T* x = static_cast<const T*>(a.x) + from * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + from * a.lddy;
    Pack<T> px[NV], pd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * V;
      if constexpr (SHORT) {
        px[i] = load_pack(x + c, cols - c);
        pd[i] = load_pack(dy + c, cols - c);
      } else {
        const uint32_t at = place<T>(c, cols).at;
        px[i] = load_whole(x, at);
        pd[i] = load_whole(dy, at);
      }
    }
    const float mu = a.mean[from], r = a.rstd[from];
    float s[2] = {0.0f, 0.0f};
    // xh and q are made twice from the row's 16-byte packs: as fp32 they would take twice to four times the registers
    if (on) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V, first = first_col<T, TPR>(i);
        if (first >= cols) continue;
        if constexpr (!KEEP) weights(i, w[0]);
        const float (&wi)[V] = w[KEEP ? i : 0];
        const Place to = SHORT ? Place{static_cast<uint32_t>(c), 0} : place<T>(c, cols);
        auto add = [&](int j, bool own) {
          const float d = get(pd[i], j), h = (get(px[i], j) - mu) * r, q = d * wi[j];
          s[0] = own ? s[0] + q : s[0];
          s[1] = own ? fmaf(q, h, s[1]) : s[1];
          dw[i * V + j] = fmaf(d, h, dw[i * V + j]);  // (what is not its own it leaves behind below)
          db[i * V + j] += d;
        };
        if (first + SPAN > cols) {  // only the wave that holds the row's end has to ask
          const int left = SHORT ? cols - c : V;
#pragma unroll
          for (int j = 0; j < V; ++j) add(j, j >= to.dup && j < left);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) add(j, true);
        }
      }
    }
    row_sum<TPR, 2>(s, red[odd]);
    if constexpr (!KEEP) asm volatile("" : "+s"(again));  // (0: so that they are not kept after all)
    if (a.dx && on) {
      const float s0 = s[0] * inv, s1 = s[1] * inv;
      T* dx = static_cast<T*>(a.dx) + row * a.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V;
        if (c >= cols) continue;
        const uint32_t at = SHORT ? c : place<T>(c, cols).at;
        if constexpr (!KEEP) weights(i, w[0]);
        const float (&wi)[V] = w[KEEP ? i : 0];
        float v[V];
        Pack<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[j] = r * fmaf(-((get(px[i], j) - mu) * r), s1, fmaf(get(pd[i], j), wi[j], -s0));
        set(p, v);
        if (SHORT) store_pack(dx + at, p, cols - c);
        else store_whole(dx, at, p);
      }
    }
  }
  if (!a.slab && !a.dw && !a.db) return;
  // The groups' sums meet in LDS: first those of a wave's own groups by shuffles, then all at once, and each column
  // adds the groups in their order.  (One group after the other took 16 us for the 16 of 800 columns.)
  constexpr int SHARE = TPR < kWave ? kWave / TPR : 1, PITCH = TPR * E;
  if constexpr (TPR < kWave)
#pragma unroll
    for (int i = 0; i < E; ++i) dw[i] = sum_rows16(dw[i]), db[i] = sum_rows16(db[i]);
  float* out = a.slab + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
    if (group % SHARE == 0) {
      float* to = lds + group / SHARE * PITCH;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * V;
        const float* v = (half ? db : dw) + i * V;
        if (c + V <= cols) {
#pragma unroll
          for (int j = 0; j < V; j += 4)
            *reinterpret_cast<float4*>(to + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else if (c < cols) {  // the last vector's own elements
          const Place p = SHORT ? Place{static_cast<uint32_t>(c), 0} : place<T>(c, cols);
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j >= p.dup && static_cast<int>(p.at) + j < cols) to[p.at + j] = v[j];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += BLOCK) {
      float s = lds[c];
#pragma unroll
      for (int g = 1; g < R / SHARE; ++g) s += lds[g * PITCH + c];
      void* whole = half ? a.db : a.dw;
      if (a.slab) out[half * cols + c] = s;
      else if (whole && (sizeof(T) == 4 || a.w32)) static_cast<float*>(whole)[c] = s;
      else if (whole) static_cast<T*>(whole)[c] = static_cast<T>(s);
    }
  }
}

// Long rows: dx from two readings of the row (the second from the L2), dw and db by columns (ln_bwd_cols_kernel), a
// third: HBM bound, 5 e bytes an element for 3 e.
template <typename T> __global__ void __launch_bounds__(1024) ln_bwd_long_kernel(LnBwd a) {
  constexpr int V = Pack<T>::n, TPR = 1024;
  __shared__ float red[2][2 * TPR / kWave];
  const float inv = 1.0f / static_cast<float>(a.cols);
  int odd = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, odd ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = static_cast<T*>(a.dx) + row * a.cols;
    const float mu = a.mean[row], r = a.rstd[row];
    float s[2] = {0.0f, 0.0f}, w[V];
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.cols; c += TPR * V) {
      const Pack<T> px = load_pack(x + c, a.cols - c), pd = load_pack(dy + c, a.cols - c);
      load_weights<T>(a.w, a.w32, c, a.cols, 1.0f, w);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < a.cols) {
          const float q = get(pd, j) * w[j];
          s[0] += q;
          s[1] = fmaf(q, (get(px, j) - mu) * r, s[1]);
        }
    }
    row_sum<TPR, 2>(s, red[odd]);
    const float s0 = s[0] * inv, s1 = s[1] * inv;
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.cols; c += TPR * V) {
      const Pack<T> px = load_pack(x + c, a.cols - c), pd = load_pack(dy + c, a.cols - c);
      load_weights<T>(a.w, a.w32, c, a.cols, 1.0f, w);
      Pack<T> p;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float q = get(pd, j) * w[j], h = (get(px, j) - mu) * r;
        w[j] = r * (q - fmaf(h, s1, s0));
      }
      set(p, w);
      store_pack(dx + c, p, a.cols - c);
    }
  }
}

// A column has few workgroups where rows are long (one from a million fp32 columns on), so a thread adds up many rows: 32
// at a time in fp32, these sums in 64 bits.  (All of them in fp32: 1024 times the same 1.00003 were off by 208 roundings,
// more than the 48 + rows / 32 that the other kernel keeps to.  No slower: 5000 x 20000 fp32 518 to 525 us both ways.)
template <typename T> __global__ void __launch_bounds__(256) ln_bwd_cols_kernel(LnBwd a) {
  constexpr int V = Pack<T>::n, RUN = 32;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * V;
  if (c >= a.cols) return;
  double all_dw[V], all_db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) all_dw[j] = all_db[j] = 0.0;
  float dw[V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.0f;
  int run = RUN;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const Pack<T> px = load_pack(static_cast<const T*>(a.x) + row * a.ldx + c, a.cols - c);
    const Pack<T> pd = load_pack(static_cast<const T*>(a.dy) + row * a.lddy + c, a.cols - c);
    const float mu = a.mean[row], r = a.rstd[row];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = get(pd, j);
      dw[j] = fmaf(d, (get(px, j) - mu) * r, dw[j]);
      db[j] += d;
    }
    if (--run == 0) {
      run = RUN;
#pragma unroll
      for (int j = 0; j < V; ++j) all_dw[j] += dw[j], all_db[j] += db[j], dw[j] = db[j] = 0.0f;
    }
  }
  float* out = a.slab + static_cast<int64_t>(blockIdx.y) * 2 * a.cols + c;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (c + j < a.cols) {
      out[j] = static_cast<float>(all_dw[j] + dw[j]);
      out[a.cols + j] = static_cast<float>(all_db[j] + db[j]);
    }
}

// dw, db = the slabs' sums, in 64 bits: 64 columns x 16 runs of slabs per workgroup, so that a thread has 16
// or 32 loads to wait for, and the runs meet in LDS in their order.  2 to 5 us (512 slabs of 4096 columns, 16.8 MB).
template <typename W> __global__ void __launch_bounds__(1024) ln_slab_kernel(const float* slab, int slabs, int64_t cols,
                                                                            W* dw, W* db) {
  __shared__ double part[16][64];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x % 64;
  const int run = threadIdx.x / 64;
  double s = 0.0;
  if (c < 2 * cols)
#pragma unroll 16
    for (int k = run; k < slabs; k += 16) s += static_cast<double>(slab[static_cast<int64_t>(k) * 2 * cols + c]);
  part[run][threadIdx.x % 64] = s;
  __syncthreads();
  if (run == 0 && c < 2 * cols) {
    for (int k = 1; k < 16; ++k) s += part[k][threadIdx.x];
    W* out = c < cols ? dw : db;
    if (out) out[c < cols ? c : c - cols] = static_cast<W>(static_cast<float>(s));
  }
}

constexpr int kCUs = 256;
constexpr int64_t kMaxCols = 1 << 24;  // (ln_slab_kernel's grid has 32 threads a column, of 2^32)
constexpr int64_t kMaxHeld = 16384;  // elements of a row that a workgroup of the backward kernel holds

// Forward: threads per row.  Fewer take their sums with less waiting, but each has more to load: up to 3 vectors each
// in a wave, 4 beyond, 8 where there are no more threads (1500 columns of fp32: 64 threads 159 us for 400 MB, 128 147, 256
// 147 with half of them idle; 1200: 150, 145, 149; 8000: 512 threads with 4 vectors 150, 1024 with 3 160, at 7000 133 and
// 130, 16000 of bf16 91 and 99; 16000 of fp32: 1024 threads with 4 145, with the 8 of longer rows 185; 24000 of fp32: 8
// vectors 183, read three times 297, and 64 such rows of 30000 8.1 and 18.3).  16 threads, whose sums stay among neighbours, with rows of 16 bits up to 5 vectors each (513 columns:
// 98 us for 200 MB, 64 threads 141; 800 columns: 86 and 82), of 32 bits up to 2 (400 columns: 163 and 139).
static int row_threads_fwd(int64_t cols, int vec) {
  const int64_t n = (cols + vec - 1) / vec;
  if (n <= 16 * (vec == 8 ? 5 : 2)) return 16;
  return n <= 64 * 3 ? 64 : n <= 128 * 4 ? 128 : n <= 256 * 4 ? 256 : n <= 512 * 4 ? 512 : 1024;
}
// Backward: up to 2 vectors each (3 in a wave, 4 where there are no more threads), beside which the weights and the sums
// of dw and db leave registers for 16 waves a CU.  600 MB of 16 bits: 1200 columns take 142 us with 64 threads and 3
// vectors, 155 with 128 and 2; 5000 columns 171 with 256 and 3 (12 waves), 131 with 512 and 2.
static int row_threads_bwd(int64_t cols, int vec) {
  const int64_t n = (cols + vec - 1) / vec;
  if (n <= 16 * 2) return 16;
  return n <= 64 * 3 ? 64 : n <= 128 * 2 ? 128 : n <= 256 * 2 ? 256 : n <= 512 * 2 ? 512 : 1024;
}
// Workgroups of 512 threads, two per CU, so that one loads while the other waits, where that tells (256 threads a row:
// 2500 columns 128 us, 157 with 1024); elsewhere of 1024, which halves the slabs.
static int bwd_block(int64_t cols, int tpr, int vec) {
  return tpr == 256 || (tpr == 64 && cols > 64 * vec) ? 512 : 1024;
}

// One workgroup alone, without slabs and their sum: up to two rounds of rows (16 rows of 800 fp32: 6.2 us on the GPU and
// 6.3 a call, with slabs 6.4 and 9.8; four rounds, 32 rows: 9.8, with slabs 6.5).
static bool bwd_alone(int64_t rows, int64_t cols, int vec) {
  if (cols > kMaxHeld) return false;
  const int tpr = row_threads_bwd(cols, vec);
  return rows <= bwd_block(cols, tpr, vec) / tpr * 2;
}

static int64_t bwd_slabs(int64_t rows, int64_t cols, int vec) {
  if (rows <= 0 || bwd_alone(rows, cols, vec)) return 0;
  if (cols > kMaxHeld) {  // column kernel: enough row runs for ~4 workgroups per CU
    const int64_t blocks = (cols + 256 * vec - 1) / (256 * vec);
    const int64_t runs = (4 * kCUs + blocks - 1) / blocks;
    return runs < rows ? runs : rows;
  }
  const int tpr = row_threads_bwd(cols, vec);
  const int64_t block = bwd_block(cols, tpr, vec), per = block / tpr, most = 1024 / block * kCUs;
  const int64_t need = (rows + per - 1) / per;
  return need < most ? need : most;
}

template <typename T, int TPR, int NV, bool SHORT = false> static void launch_fwd(const LnFwd& a, hipStream_t st) {
  constexpr int block = TPR > 256 ? TPR : 256, r = block / TPR;
  const int64_t need = (a.rows + r - 1) / r, most = 1 << 20;  // (a grid's x is at most 2^32 threads)
  const dim3 grid(static_cast<unsigned>(need < most ? need : most), static_cast<unsigned>((need + most - 1) / most));
  hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV, SHORT>), grid, dim3(block), 0, st, a);
}

template <typename T> static void fwd(const LnFwd& a, hipStream_t st) {
  constexpr int V = Pack<T>::n;
  const int tpr = row_threads_fwd(a.cols, V);
  const int64_t nv = (a.cols + static_cast<int64_t>(tpr) * V - 1) / (static_cast<int64_t>(tpr) * V);
  if (a.cols < V) {
    launch_fwd<T, 16, 1, true>(a, st);
  } else if (tpr == 16) {
    if constexpr (V == 8)
      if (nv > 2) return nv <= 4 ? launch_fwd<T, 16, 4>(a, st) : launch_fwd<T, 16, 5>(a, st);
    if (nv <= 1) launch_fwd<T, 16, 1>(a, st); else launch_fwd<T, 16, 2>(a, st);
  } else if (tpr == 64) {
    if constexpr (V == 4)
      if (nv <= 1) return launch_fwd<T, 64, 1>(a, st);
    if (nv <= 2) launch_fwd<T, 64, 2>(a, st); else launch_fwd<T, 64, 3>(a, st);
  } else if (tpr == 128) {
    if (nv <= 2) launch_fwd<T, 128, 2>(a, st); else if (nv <= 3) launch_fwd<T, 128, 3>(a, st); else launch_fwd<T, 128, 4>(a, st);
  } else if (tpr == 256) {
    if (nv <= 3) launch_fwd<T, 256, 3>(a, st); else launch_fwd<T, 256, 4>(a, st);
  } else if (tpr == 512) {
    if (nv <= 3) launch_fwd<T, 512, 3>(a, st); else launch_fwd<T, 512, 4>(a, st);
  } else if (nv <= 8) {
    if (nv <= 3) launch_fwd<T, 1024, 3>(a, st); else if (nv <= 4) launch_fwd<T, 1024, 4>(a, st); else launch_fwd<T, 1024, 8>(a, st);
  } else {
    const int64_t most = 1 << 20;
    hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3(static_cast<unsigned>(a.rows < most ? a.rows : most)), dim3(1024), 0,
                       st, a);
  }
}

template <typename T, int TPR, int NV, int BLOCK = 1024, bool SHORT = false> static int launch_bwd(const LnBwd& a, int64_t slabs, hipStream_t st) {
  constexpr int groups = BLOCK / (TPR < kWave ? kWave : TPR);
  constexpr int lds = groups * TPR * NV * Pack<T>::n * static_cast<int>(sizeof(float));
  IADMM_ALLOW_LDS((ln_bwd_kernel<T, TPR, NV, BLOCK, SHORT>), lds + 512);
  hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV, BLOCK, SHORT>), dim3(static_cast<unsigned>(slabs)), dim3(BLOCK), lds, st, a);
  return 0;
}

template <typename T> static int bwd(const LnBwd& a, int64_t slabs, hipStream_t st) {
  constexpr int V = Pack<T>::n;
  if (a.cols > kMaxHeld) {
    const int64_t most = 1 << 20;
    if (a.dx)
      hipLaunchKernelGGL((ln_bwd_long_kernel<T>), dim3(static_cast<unsigned>(a.rows < most ? a.rows : most)), dim3(1024),
                         0, st, a);
    if (a.slab) {
      const int64_t blocks = (a.cols + 256 * V - 1) / (256 * V);
      hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(slabs)),
                         dim3(256), 0, st, a);
    }
    return 0;
  }
  const int tpr = row_threads_bwd(a.cols, V);
  const int64_t nv = (a.cols + static_cast<int64_t>(tpr) * V - 1) / (static_cast<int64_t>(tpr) * V);
  if (a.cols < V) return launch_bwd<T, 16, 1, 1024, true>(a, slabs, st);
  if (tpr == 16) return nv <= 1 ? launch_bwd<T, 16, 1>(a, slabs, st) : launch_bwd<T, 16, 2>(a, slabs, st);
  if (tpr == 64) {
    if (nv <= 1) return launch_bwd<T, 64, 1>(a, slabs, st);
    return nv <= 2 ? launch_bwd<T, 64, 2, 512>(a, slabs, st) : launch_bwd<T, 64, 3, 512>(a, slabs, st);
  }
  if (tpr == 128) return launch_bwd<T, 128, 2>(a, slabs, st);
  if (tpr == 256) return launch_bwd<T, 256, 2, 512>(a, slabs, st);
  if (tpr == 512) return launch_bwd<T, 512, 2>(a, slabs, st);
  if constexpr (V == 4)
    if (nv > 2) return nv <= 3 ? launch_bwd<T, 1024, 3>(a, slabs, st) : launch_bwd<T, 1024, 4>(a, slabs, st);
  return launch_bwd<T, 1024, 2>(a, slabs, st);
}

static bool bad_types(int dtype, int wdtype) {
  return dtype < IADMM_F32 || dtype > IADMM_F16 || (wdtype != IADMM_F32 && wdtype != dtype);
}

}  // namespace iadmm

using namespace iadmm;

extern "C" int iadmm_layer_norm_fwd(int64_t rows, int64_t cols, int dtype, int wdtype, const void* x, int64_t ldx,
                                    const void* w, const void* b, float eps, void* y, float* mean, float* rstd,
                                    void* stream) {
  if (rows < 0 || cols <= 0 || bad_types(dtype, wdtype) || !(eps >= 0.0f) || !(eps < __builtin_inff())) return IADMM_E_ARG;
  if (rows == 0) return IADMM_OK;
  if (!x || !y || ldx < cols) return IADMM_E_ARG;
  if (cols > kMaxCols) return IADMM_E_SIZE;
  const LnFwd a{rows, cols, ldx, x, w, b, y, mean, rstd, eps, wdtype == IADMM_F32};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == IADMM_F32) fwd<float>(a, st);
  else if (dtype == IADMM_BF16) fwd<__bf16>(a, st);
  else fwd<_Float16>(a, st);
  IADMM_CHECK_LAUNCH();
  return IADMM_OK;
}

extern "C" int64_t iadmm_layer_norm_bwd_ws_bytes(int64_t rows, int64_t cols, int dtype) {
  if (rows <= 0 || cols <= 0) return 0;
  return bwd_slabs(rows, cols, dtype == IADMM_F32 ? 4 : 8) * 2 * cols * static_cast<int64_t>(sizeof(float));
}

extern "C" int iadmm_layer_norm_bwd(int64_t rows, int64_t cols, int dtype, int wdtype, const void* dy, int64_t lddy,
                                    const void* x, int64_t ldx, const float* mean, const float* rstd, const void* w,
                                    void* dx, void* dw, void* db, void* ws, int64_t ws_bytes, void* stream) {
  if (rows < 0 || cols <= 0 || bad_types(dtype, wdtype)) return IADMM_E_ARG;
  if (cols > kMaxCols) return IADMM_E_SIZE;
  const bool sums = dw || db;
  if (rows > 0 && (!dy || !x || !mean || !rstd || lddy < cols || ldx < cols)) return IADMM_E_ARG;
  if (sums && ws_bytes < iadmm_layer_norm_bwd_ws_bytes(rows, cols, dtype)) return IADMM_E_ARG;
  if (sums && rows > 0 && !ws && iadmm_layer_norm_bwd_ws_bytes(rows, cols, dtype) > 0) return IADMM_E_ARG;
  if (sums && !aligned16(ws)) return IADMM_E_ALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int vec = dtype == IADMM_F32 ? 4 : 8;
  const bool alone = rows > 0 && bwd_alone(rows, cols, vec);
  const int64_t slabs = bwd_slabs(rows, cols, vec);
  const LnBwd a{rows, cols, lddy, ldx, dy, x, w, mean, rstd, dx, sums && !alone ? static_cast<float*>(ws) : nullptr,
                wdtype == IADMM_F32, alone ? dw : nullptr, alone ? db : nullptr};
  if (rows > 0 && (dx || sums)) {
    const int64_t blocks = alone ? (sums ? 1 : rows) : slabs;  // (alone: some hundred rows at most)
    const int rc = dtype == IADMM_F32 ? bwd<float>(a, blocks, st)
                   : dtype == IADMM_BF16 ? bwd<__bf16>(a, blocks, st) : bwd<_Float16>(a, blocks, st);
    if (rc) return rc;
    IADMM_CHECK_LAUNCH();
  }
  if (sums && !alone) {  // (no rows: the sums are 0)
    const dim3 grid(static_cast<unsigned>((2 * cols + 63) / 64)), block(1024);
    const float* slab = static_cast<const float*>(ws);
    const int n = static_cast<int>(slabs);
    if (wdtype == IADMM_F32)
      hipLaunchKernelGGL((ln_slab_kernel<float>), grid, block, 0, st, slab, n, cols, static_cast<float*>(dw),
                         static_cast<float*>(db));
    else if (wdtype == IADMM_BF16)
      hipLaunchKernelGGL((ln_slab_kernel<__bf16>), grid, block, 0, st, slab, n, cols, static_cast<__bf16*>(dw),
                         static_cast<__bf16*>(db));
    else
      hipLaunchKernelGGL((ln_slab_kernel<_Float16>), grid, block, 0, st, slab, n, cols, static_cast<_Float16*>(dw),
                         static_cast<_Float16*>(db));
    IADMM_CHECK_LAUNCH();
  }
  return IADMM_OK;
}
