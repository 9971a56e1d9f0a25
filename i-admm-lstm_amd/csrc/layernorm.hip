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
// a row is read once and stays in registers: TPR threads hold it, up to 16 elements each, in 16-byte vectors
// (TPR = 16, 64, 256, 1024 for rows up to 256 / 1024 / 4096 / 16384 elements); longer rows are read again,
// from L2 for the most part.
#include "common.h"

namespace iadmm {

typedef unsigned uint4v __attribute__((ext_vector_type(4)));

template <typename T> struct Pack;  // 16 bytes of T, at any address that T may have
template <> struct Pack<float> { static constexpr int n = 4; float v[4]; };
template <> struct Pack<__bf16> { static constexpr int n = 8; __bf16 v[8]; };
template <> struct Pack<_Float16> { static constexpr int n = 8; _Float16 v[8]; };

// n elements from p (n < Pack::n only at a row's end); what lies behind is 0.  Rows of odd length start at
// any multiple of the element size: the memory pipe takes 16-byte loads there.
template <typename T> IADMM_DEV Pack<T> load_pack(const T* p, int64_t n) {
  Pack<T> r;
  if (n >= Pack<T>::n) {
    __builtin_memcpy(&r, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < Pack<T>::n; ++j) r.v[j] = j < n ? p[j] : static_cast<T>(0.0f);
  }
  return r;
}
template <typename T> IADMM_DEV void store_pack(T* p, const Pack<T>& r, int64_t n) {
  if (n >= Pack<T>::n) {
    __builtin_memcpy(p, &r, 16);
  } else {
#pragma unroll
    for (int j = 0; j < Pack<T>::n; ++j)
      if (j < n) p[j] = r.v[j];
  }
}

// V weights from column c (0 behind the end), of type T or fp32; `none` where there are none.
template <typename T> IADMM_DEV void load_weights(const void* w, bool f32, int64_t c, int64_t cols, float none,
                                                  float* out) {
  constexpr int V = Pack<T>::n;
  const int64_t n = cols - c;
  if (!w) {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = none;
  } else if (sizeof(T) == 4 || f32) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      const Pack<float> a = load_pack(static_cast<const float*>(w) + c + 4 * k, n - 4 * k);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[4 * k + j] = a.v[j];
    }
  } else {
    const Pack<T> a = load_pack(static_cast<const T*>(w) + c, n);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = static_cast<float>(a.v[j]);
  }
}

// Sums of v over the TPR threads of a row, in every one of them.  More than a wave: through LDS, `red` holding
// one value per wave of the workgroup; the caller alternates between two such arrays, so one barrier is enough
// (a wave writes an array again only after every wave has passed the other array's barrier).
template <int TPR, int K> IADMM_DEV void row_sum(float (&v)[K], float* red) {
#pragma unroll
  for (int o = (TPR < kWave ? TPR : kWave) / 2; o >= 1; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o, kWave);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave * K + k] = v[k];
    __syncthreads();
    const float* r = red + wave / W * W * K;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = r[k];
      for (int w = 1; w < W; ++w) s += r[w * K + k];
      v[k] = s;
    }
  }
}

struct LnFwd {
  int64_t rows, cols, ldx;
  const void *x, *w, *b;
  void* y;
  float *mean, *rstd;
  float eps;
  int w32;
};

// One row per TPR threads, NV vectors each.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) ln_fwd_kernel(LnFwd a) {
  constexpr int V = Pack<T>::n, BLOCK = TPR > 256 ? TPR : 256, R = BLOCK / TPR;
  __shared__ float red[2][BLOCK / kWave];
  const int lane = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.cols);
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * R; row0 < a.rows; row0 += static_cast<int64_t>(gridDim.x) * R) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool on = row < a.rows;
    const T* x = static_cast<const T*>(a.x) + (on ? row : 0) * a.ldx;
    float v[NV * V];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = static_cast<int64_t>(i * TPR + lane) * V;
      const Pack<T> p = load_pack(x + c, on ? a.cols - c : 0);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = static_cast<float>(p.v[j]);
    }
#pragma unroll
    for (int i = 0; i < NV * V; ++i) s[0] += v[i];
    row_sum<TPR, 1>(s, red[0]);
    const float mu = s[0] * inv;
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int64_t c = static_cast<int64_t>(i * TPR + lane) * V + j;
        v[i * V + j] = c < a.cols ? v[i * V + j] - mu : 0.0f;
        s[0] = fmaf(v[i * V + j], v[i * V + j], s[0]);
      }
    row_sum<TPR, 1>(s, red[1]);
    const float r = 1.0f / sqrtf(s[0] * inv + a.eps);
    if (!on) continue;  // (TPR > 64 has one row per workgroup: nobody is left at a barrier)
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = static_cast<int64_t>(i * TPR + lane) * V;
      if (c >= a.cols) continue;
      float w[V], b[V];
      load_weights<T>(a.w, a.w32, c, a.cols, 1.0f, w);
      load_weights<T>(a.b, a.w32, c, a.cols, 0.0f, b);
      Pack<T> p;
#pragma unroll
      for (int j = 0; j < V; ++j) p.v[j] = static_cast<T>(fmaf(v[i * V + j] * r, w[j], b[j]));
      store_pack(y + c, p, a.cols - c);
    }
    if (lane == 0 && a.mean) a.mean[row] = mu;
    if (lane == 0 && a.rstd) a.rstd[row] = r;
  }
}

// Rows longer than the registers hold: a workgroup reads its row three times.
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
      for (int j = 0; j < V; ++j) s[0] += static_cast<float>(p.v[j]);
    }
    row_sum<TPR, 1>(s, red[0]);
    const float mu = s[0] * inv;
    s[0] = 0.0f;
    for (int64_t c = static_cast<int64_t>(threadIdx.x) * V; c < a.cols; c += TPR * V) {
      const Pack<T> p = load_pack(x + c, a.cols - c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = c + j < a.cols ? static_cast<float>(p.v[j]) - mu : 0.0f;
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
      for (int j = 0; j < V; ++j)
        p.v[j] = static_cast<T>(fmaf((static_cast<float>(p.v[j]) - mu) * r, w[j], b[j]));
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
};

// A workgroup of 1024 threads takes 1024 / TPR rows at a time, at most one workgroup per CU: dw and db grow in
// registers over all its rows, meet once in LDS and leave as one slab, which keeps the slabs' traffic small
// beside the rows' (256 slabs at most).
template <typename T, int TPR, int NV> __global__ void __launch_bounds__(1024) ln_bwd_kernel(LnBwd a) {
  constexpr int V = Pack<T>::n, R = 1024 / TPR, E = NV * V;
  extern __shared__ float lds[];  // [2][cols]
  __shared__ float red[2][2 * 1024 / kWave];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.0f / static_cast<float>(a.cols);
  float dw[E], db[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.0f;
  int odd = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * R; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x) * R, odd ^= 1) {
    const int64_t row = row0 + group;
    const bool on = row < a.rows;
    const int64_t at = on ? row : 0, cols = on ? a.cols : 0;
    const T* x = static_cast<const T*>(a.x) + at * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + at * a.lddy;
    Pack<T> px[NV], pd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = static_cast<int64_t>(i * TPR + lane) * V;
      px[i] = load_pack(x + c, cols - c);
      pd[i] = load_pack(dy + c, cols - c);
    }
    // (0 in the groups behind the last row, whose dy is 0 too: nothing of them reaches the sums)
    const float mu = on ? a.mean[row] : 0.0f, r = on ? a.rstd[row] : 0.0f;
    float s[2] = {0.0f, 0.0f};
    // dy is 0 behind the row's end, and so is all that comes of it there.  xh and q are made twice from the
    // row's 16-byte packs: held as fp32 they spill (128 registers for a workgroup of 1024).
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[V];
      load_weights<T>(a.w, a.w32, static_cast<int64_t>(i * TPR + lane) * V, a.cols, 1.0f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = static_cast<float>(pd[i].v[j]), h = (static_cast<float>(px[i].v[j]) - mu) * r;
        const float q = d * w[j];
        s[0] += q;
        s[1] = fmaf(q, h, s[1]);
        dw[i * V + j] = fmaf(d, h, dw[i * V + j]);
        db[i * V + j] += d;
      }
    }
    row_sum<TPR, 2>(s, red[odd]);
    if (a.dx && on) {
      const float s0 = s[0] * inv, s1 = s[1] * inv;
      T* dx = static_cast<T*>(a.dx) + row * a.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = static_cast<int64_t>(i * TPR + lane) * V;
        if (c >= a.cols) continue;
        float w[V];
        load_weights<T>(a.w, a.w32, c, a.cols, 1.0f, w);
        Pack<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float q = static_cast<float>(pd[i].v[j]) * w[j], h = (static_cast<float>(px[i].v[j]) - mu) * r;
          p.v[j] = static_cast<T>(r * (q - fmaf(h, s1, s0)));
        }
        store_pack(dx + c, p, a.cols - c);
      }
    }
  }
  if (!a.slab) return;
  // the groups add their sums in their order (a wave's own groups by shuffles first)
  constexpr int SHARE = TPR < kWave ? kWave / TPR : 1;
#pragma unroll
  for (int o = kWave / 2; o >= TPR; o >>= 1)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      dw[i] += __shfl_xor(dw[i], o, kWave);
      db[i] += __shfl_xor(db[i], o, kWave);
    }
  for (int g = 0; g < R; g += SHARE) {
    if (group == g) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int64_t c = static_cast<int64_t>(i / V * TPR + lane) * V + i % V;
        if (c < a.cols) {
          lds[c] = g ? lds[c] + dw[i] : dw[i];
          lds[a.cols + c] = g ? lds[a.cols + c] + db[i] : db[i];
        }
      }
    }
    __syncthreads();
  }
  float* out = a.slab + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
  for (int64_t c = threadIdx.x; c < 2 * a.cols; c += 1024) out[c] = lds[c];
}

// Long rows: dx from two readings of the row, dw and db by columns (ln_bwd_cols_kernel).
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
          const float q = static_cast<float>(pd.v[j]) * w[j];
          s[0] += q;
          s[1] = fmaf(q, (static_cast<float>(px.v[j]) - mu) * r, s[1]);
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
        const float q = static_cast<float>(pd.v[j]) * w[j], h = (static_cast<float>(px.v[j]) - mu) * r;
        p.v[j] = static_cast<T>(r * (q - fmaf(h, s1, s0)));
      }
      store_pack(dx + c, p, a.cols - c);
    }
  }
}

template <typename T> __global__ void __launch_bounds__(256) ln_bwd_cols_kernel(LnBwd a) {
  constexpr int V = Pack<T>::n;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * V;
  if (c >= a.cols) return;
  float dw[V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const Pack<T> px = load_pack(static_cast<const T*>(a.x) + row * a.ldx + c, a.cols - c);
    const Pack<T> pd = load_pack(static_cast<const T*>(a.dy) + row * a.lddy + c, a.cols - c);
    const float mu = a.mean[row], r = a.rstd[row];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = static_cast<float>(pd.v[j]);
      dw[j] = fmaf(d, (static_cast<float>(px.v[j]) - mu) * r, dw[j]);
      db[j] += d;
    }
  }
  float* out = a.slab + static_cast<int64_t>(blockIdx.y) * 2 * a.cols + c;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (c + j < a.cols) out[j] = dw[j], out[a.cols + j] = db[j];
}

// dw, db = the slabs' sums, in 64 bits: 64 columns x 16 runs of slabs per workgroup, so that a thread has 16
// loads at most to wait for, and the runs meet in LDS in their order.
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
constexpr int64_t kMaxHeld = 16384;  // elements of a row that a workgroup holds

// Threads per row: as few as hold it with 16 elements each, since fewer meet without a barrier.
static int row_threads(int64_t cols, int vec) {
  if (cols <= 16 * 16) return vec == 8 || cols <= 16 * 8 ? 16 : 64;
  return cols <= 64 * 16 ? 64 : cols <= 256 * 16 ? 256 : 1024;
}

static int64_t bwd_slabs(int64_t rows, int64_t cols, int vec) {
  if (rows <= 0) return 0;
  if (cols > kMaxHeld) {  // column kernel: enough row runs for ~4 workgroups per CU
    const int64_t blocks = (cols + 256 * vec - 1) / (256 * vec);
    const int64_t runs = (4 * kCUs + blocks - 1) / blocks;
    return runs < rows ? runs : rows;
  }
  const int64_t per = 1024 / row_threads(cols, vec);
  const int64_t need = (rows + per - 1) / per;
  return need < kCUs ? need : kCUs;
}

template <typename T, int TPR, int NV> static void launch_fwd(const LnFwd& a, hipStream_t st) {
  constexpr int block = TPR > 256 ? TPR : 256, r = block / TPR;
  const int64_t need = (a.rows + r - 1) / r, most = 1 << 20;
  hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV>), dim3(static_cast<unsigned>(need < most ? need : most)), dim3(block), 0,
                     st, a);
}

template <typename T> static void fwd(const LnFwd& a, hipStream_t st) {
  constexpr int V = Pack<T>::n, M = 16 / V;  // vectors of 16 elements
  if (a.cols > kMaxHeld) {
    const int64_t most = 1 << 20;
    hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3(static_cast<unsigned>(a.rows < most ? a.rows : most)), dim3(1024), 0,
                       st, a);
    return;
  }
  const int tpr = row_threads(a.cols, V);
  const int64_t nv = (a.cols + static_cast<int64_t>(tpr) * V - 1) / (static_cast<int64_t>(tpr) * V);
  if (tpr == 16) {
    if (nv <= 1) launch_fwd<T, 16, 1>(a, st); else launch_fwd<T, 16, 2>(a, st);
  } else if (tpr == 64) {
    if (nv <= 1) launch_fwd<T, 64, 1>(a, st); else if (nv <= 2) launch_fwd<T, 64, 2>(a, st); else launch_fwd<T, 64, M>(a, st);
  } else if (tpr == 256) {
    if (nv <= M / 2) launch_fwd<T, 256, M / 2>(a, st); else launch_fwd<T, 256, M>(a, st);
  } else {
    if (nv <= M / 2) launch_fwd<T, 1024, M / 2>(a, st); else launch_fwd<T, 1024, M>(a, st);
  }
}

template <typename T, int TPR, int NV> static int launch_bwd(const LnBwd& a, int64_t slabs, hipStream_t st) {
  const int lds = static_cast<int>(2 * a.cols * sizeof(float));
  IADMM_ALLOW_LDS((ln_bwd_kernel<T, TPR, NV>), lds + 512);
  hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV>), dim3(static_cast<unsigned>(slabs)), dim3(1024), lds, st, a);
  return 0;
}

template <typename T> static int bwd(const LnBwd& a, int64_t slabs, hipStream_t st) {
  constexpr int V = Pack<T>::n, M = 16 / V;
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
  const int tpr = row_threads(a.cols, V);
  const int64_t nv = (a.cols + static_cast<int64_t>(tpr) * V - 1) / (static_cast<int64_t>(tpr) * V);
  if (tpr == 16) return nv <= 1 ? launch_bwd<T, 16, 1>(a, slabs, st) : launch_bwd<T, 16, 2>(a, slabs, st);
  if (tpr == 64)
    return nv <= 1 ? launch_bwd<T, 64, 1>(a, slabs, st)
                   : nv <= 2 ? launch_bwd<T, 64, 2>(a, slabs, st) : launch_bwd<T, 64, M>(a, slabs, st);
  if (tpr == 256) return nv <= M / 2 ? launch_bwd<T, 256, M / 2>(a, slabs, st) : launch_bwd<T, 256, M>(a, slabs, st);
  return nv <= M / 2 ? launch_bwd<T, 1024, M / 2>(a, slabs, st) : launch_bwd<T, 1024, M>(a, slabs, st);
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
  if (cols > (int64_t{1} << 31)) return IADMM_E_SIZE;
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
  if (cols > (int64_t{1} << 31)) return IADMM_E_SIZE;
  const bool sums = dw || db;
  if (rows > 0 && (!dy || !x || !mean || !rstd || lddy < cols || ldx < cols)) return IADMM_E_ARG;
  if (sums && ws_bytes < iadmm_layer_norm_bwd_ws_bytes(rows, cols, dtype)) return IADMM_E_ARG;
  if (sums && rows > 0 && !ws) return IADMM_E_ARG;
  if (sums && !aligned16(ws)) return IADMM_E_ALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t slabs = bwd_slabs(rows, cols, dtype == IADMM_F32 ? 4 : 8);
  const LnBwd a{rows, cols, lddy, ldx, dy, x, w, mean, rstd, dx, sums ? static_cast<float*>(ws) : nullptr,
                wdtype == IADMM_F32};
  if (rows > 0 && (dx || sums)) {
    const int rc = dtype == IADMM_F32 ? bwd<float>(a, slabs, st)
                   : dtype == IADMM_BF16 ? bwd<__bf16>(a, slabs, st) : bwd<_Float16>(a, slabs, st);
    if (rc) return rc;
    IADMM_CHECK_LAUNCH();
  }
  if (sums) {  // (no rows: the sums are 0)
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
