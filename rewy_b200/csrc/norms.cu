// Root-mean-square norms before and after a block, fused with what stands beside them, and their gradients.
//
//   gated     y = n(x) w act(g), or with gate_first n(x act(g)) w;       n(v) = v r, r = 1 / sqrt(mean v^2 + eps)
//   residual  r_out = residual + s x;  y = n(r_out) w                    s a number or one per channel
//   backward  with dn the gradient of n:  dv = r (dn - n mean(dn n));  dw = sum over the rows of dn's other factor
//
// One pass over the rows, bound by HBM: a row lies in the registers of the 16 to 1024 threads that share it (8 neighbouring
// elements per access), so that its sum of squares needs no second read; the backward takes mean(dn n) = r mean(dn v) from the
// same exchange as the sum of squares and so needs neither r nor a second exchange.  Rows of up to 128 elements (heads) share a
// warp.  The weight, its gradient and the scale's stay in registers over the rows that a CTA takes; the CTAs' sums are added by
// a second kernel in one order.  The residual backward adds residual + s x up again in FP32 instead of reading the rounded sum
// that the forward returned: n then is what the forward normalised, at the price of one more input read.
// Measured in BF16: gated, 131072 rows of 128: forward 19 us (5.4 TB/s), backward 32 (5.3 TB/s); residual, 8192 rows of 4096 with a
// scale per channel: forward 51 us (5.3 TB/s), backward 93 (4.3 TB/s).  Before: rows loaded into registers 30, 68, 84, 302; through
// shared memory, two or three rows ahead, 28, 48, 64, 117; without a division per row and with 16-bit elements converted in pairs
// 20, 33, 54, 104; sums over the warps of a row by lanes instead of by every thread, now.
#include "layer.cuh"

namespace rewy {
namespace {

constexpr int E = 8;  // elements per access

struct NormParams {
  RewyNormArgs a;
  bool wide;
  float* partial;  // [CTAs][2][D]
  float inv_D;
};

// (rows at one distance need no division; fewer than 2^32 rows a short one)
__device__ __forceinline__ long long row_start(long long r, long long inner, long long rows, const int64_t (&stride)[2]) {
  if (inner >= rows) return r * stride[1];
  const long long o = rows <= 0xffffffffLL ? (long long)((unsigned)r / (unsigned)inner) : r / inner;
  return o * stride[0] + (r - o * inner) * stride[1];
}

// Sums over the TPR threads of a row; `red` is written alternately so that one barrier per row is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], float* red, int parity) {
  constexpr int LANES = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int m = LANES / 2; m > 0; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; i++) x[i] += __shfl_xor_sync(0xffffffffu, x[i], m);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32, ALL = (TPR > 256 ? TPR : 256) / 32;
    const int warp = threadIdx.x >> 5, first = warp / WARPS * WARPS;
    float* to = red + parity * ALL * N;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; i++) to[warp * N + i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to[(first + (threadIdx.x & (WARPS - 1))) * N + i];
#pragma unroll
    for (int m = WARPS / 2; m > 0; m >>= 1)
#pragma unroll
      for (int i = 0; i < N; i++) x[i] += __shfl_xor_sync(0xffffffffu, x[i], m);
  }
}

template <int TPR, int NV>
struct Layout {
  static constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR, COLS = TPR * NV * E, RED = TPR > 32 ? 2 * THREADS / 32 * 2 : 1;
  __device__ static __forceinline__ int column(int v) { return (v * TPR + threadIdx.x % TPR) * E; }
};

// The rows that a CTA works on next, on their way through shared memory: every thread copies the elements that it will read
// itself, so that no barrier stands between, and no registers hold what is under way.  Rows that do not fit twice are loaded
// when they are needed.  Elements of TA stand in the first NA of the inputs, of TB in the others.
template <class TA, int NA, class TB, int NB, int TPR, int NV>
struct Stream {
  using Y = Layout<TPR, NV>;
  static constexpr int BYTES_A = NV * E * sizeof(TA), BYTES_B = NV * E * sizeof(TB), STAGE = Y::THREADS * (NA * BYTES_A + NB * BYTES_B);
  static constexpr int ROOM = (220 * 1024 - Y::COLS * 8) / STAGE, WANT = STAGE <= 32 * 1024 ? 3 : 2, STAGES = ROOM >= WANT ? WANT : ROOM >= 2 ? 2 : 0;
  static constexpr int BYTES = STAGES * STAGE;
  const TA* a[NA];
  const TB* b[NB > 0 ? NB : 1];
  Pack<TA, E> pa[NA][NV];
  Pack<TB, E> pb[NB > 0 ? NB : 1][NV];
  unsigned char* smem;
  bool wide;

  template <class T>
  __device__ __forceinline__ T* slot(int stage, int i, int v) const {
    const int before = sizeof(T) == sizeof(TA) && i < NA ? i * BYTES_A : NA * BYTES_A + (i - NA) * BYTES_B;
    return reinterpret_cast<T*>(smem + stage * STAGE + Y::THREADS * before) + (v * Y::THREADS + threadIdx.x) * E;
  }
  template <class T>
  __device__ __forceinline__ void copy(T* to, const T* from, int valid) {
    if (wide && valid >= E) {
#pragma unroll
      for (int i = 0; i < E * (int)sizeof(T) / 16; i++) {
        const unsigned dst = (unsigned)__cvta_generic_to_shared(reinterpret_cast<uint4*>(to) + i);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<const uint4*>(from) + i) : "memory");
      }
      return;
    }
    Pack<T, E> x;
    load_some<T, E>(x, from, valid, false);
    *reinterpret_cast<Pack<T, E>*>(to) = x;
  }
  // a[] and b[] point at the row; valid(v, i): how many elements of input i there are from column(v) on
  template <class F>
  __device__ __forceinline__ void ask(int stage, F&& valid) {
    if constexpr (STAGES > 0) {
#pragma unroll
      for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int i = 0; i < NA; i++) copy(slot<TA>(stage, i, v), a[i] + Y::column(v), valid(v, i));
#pragma unroll
        for (int i = 0; i < NB; i++) copy(slot<TB>(stage, NA + i, v), b[i] + Y::column(v), valid(v, NA + i));
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  template <class F>
  __device__ __forceinline__ void take(int stage, F&& valid) {
    if constexpr (STAGES > 0) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
#pragma unroll
      for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int i = 0; i < NA; i++) pa[i][v] = *reinterpret_cast<const Pack<TA, E>*>(slot<TA>(stage, i, v));
#pragma unroll
        for (int i = 0; i < NB; i++) pb[i][v] = *reinterpret_cast<const Pack<TB, E>*>(slot<TB>(stage, NA + i, v));
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int i = 0; i < NA; i++) load_some<TA, E>(pa[i][v], a[i] + Y::column(v), valid(v, i), wide);
#pragma unroll
        for (int i = 0; i < NB; i++) load_some<TB, E>(pb[i][v], b[i] + Y::column(v), valid(v, NA + i), wide);
      }
    }
  }
};

// Calls work(r, real, parity) for each row of this thread's, its elements in `in`; point(r) sets the inputs' addresses, with(i)
// says whether there is an input i at all.
template <int TPR, int NV, class In, class Point, class With, class Work>
__device__ __forceinline__ void for_rows(In& in, long long rows, int D, Point&& point, With&& with, Work&& work) {
  using Y = Layout<TPR, NV>;
  const long long stride = (long long)gridDim.x * Y::ROWS, first = (long long)blockIdx.x * Y::ROWS;
  const int mine = threadIdx.x / TPR;
  auto ask = [&](long long base, int stage) {
    const long long r = base + mine;
    const bool real = r < rows;
    point(real ? r : 0);
    in.ask(stage, [&](int v, int i) { return real && with(i) ? D - Y::column(v) : 0; });
  };
  if constexpr (In::STAGES > 0)
#pragma unroll
    for (int k = 0; k < In::STAGES - 1; k++) ask(first + k * stride, k);
  int stage = 0, parity = 0;
  for (long long base = first; base < rows; base += stride, parity ^= 1) {
    const long long r = base + mine;
    const bool real = r < rows;
    if constexpr (In::STAGES > 0) {
      const int ahead = stage == 0 ? In::STAGES - 1 : stage - 1;
      ask(base + (In::STAGES - 1) * stride, ahead);
    } else {
      point(real ? r : 0);
    }
    in.take(stage, [&](int v, int i) { return real && with(i) ? D - Y::column(v) : 0; });
    work(r, real, parity);
    if constexpr (In::STAGES > 0) stage = stage == In::STAGES - 1 ? 0 : stage + 1;
  }
  if constexpr (In::STAGES > 0) asm volatile("cp.async.wait_all;" ::: "memory");
}

// The CTA's sums per column: over its rows' threads in shared memory, then to `to`.
template <int TPR, int NV>
__device__ __forceinline__ void store_column_sums(float (&x)[NV][E], float* sums, float* to, int D) {
  using Y = Layout<TPR, NV>;
  if constexpr (Y::ROWS == 1) {
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < E; e++)
        if (Y::column(v) + e < D) to[Y::column(v) + e] = x[v][e];
  } else {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < E; e++) sums[threadIdx.x / TPR * Y::COLS + Y::column(v) + e] = x[v][e];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += Y::THREADS) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < Y::ROWS; r++) s += sums[r * Y::COLS + c];
      to[c] = s;
    }
  }
}
// A parameter per column as FP32 in shared memory
template <int TPR, int NV>
__device__ __forceinline__ void load_params(float* w, const void* p, int dtype, int D, float otherwise) {
  for (int c = threadIdx.x; c < Layout<TPR, NV>::COLS; c += Layout<TPR, NV>::THREADS) w[c] = c >= D ? 0.f : p == nullptr ? otherwise : param_at(p, dtype, c);
}
__device__ __forceinline__ void read8(float (&x)[E], const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
// act(g) and, if asked for, act'(g)
template <bool SILU, bool SLOPE>
__device__ __forceinline__ float act_of(float g, float& slope) {
  const float sig = sigmoid_fast(g);
  if constexpr (SLOPE) slope = SILU ? sig * fmaf(g, 1.f - sig, 1.f) : sig * (1.f - sig);
  return SILU ? g * sig : sig;
}
// f(SiLU?, gate first?) with both as types: what is asked once stands outside the loops over elements
template <class F>
__device__ __forceinline__ void with_gate(const RewyNormArgs& a, F&& f) {
  if (a.activation == 0) {
    if (a.gate_first) f(std::true_type(), std::true_type());
    else f(std::true_type(), std::false_type());
  } else {
    if (a.gate_first) f(std::false_type(), std::true_type());
    else f(std::false_type(), std::false_type());
  }
}

// CTAs on an SM that the registers are cut for
template <class T, int TPR, int NV, bool BACKWARD>
constexpr int resident() {
  constexpr int threads = Layout<TPR, NV>::THREADS, most = sizeof(T) == 4 ? 512 : BACKWARD ? 768 : 1024;
  return most > threads ? most / threads : 1;
}
template <class T, int TPR, int NV>
using GatedFwd = Stream<T, 2, T, 0, TPR, NV>;
template <class T, int TPR, int NV>
using GatedBwd = Stream<T, 3, T, 0, TPR, NV>;
template <class T, class TR, int TPR, int NV>
using ResidualFwd = Stream<T, 1, TR, 1, TPR, NV>;
template <class T, class TR, int TPR, int NV>
using ResidualBwd = Stream<T, 2, TR, 2, TPR, NV>;

template <class T, int TPR, int NV>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS, resident<T, TPR, NV, false>()) gated_fwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[Y::RED];
  const RewyNormArgs& a = p.a;
  float* const w = reinterpret_cast<float*>(smem + GatedFwd<T, TPR, NV>::BYTES);
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  __syncthreads();
  GatedFwd<T, TPR, NV> in;
  in.smem = smem; in.wide = p.wide;
  auto point = [&](long long r) {
    in.a[0] = static_cast<const T*>(a.x) + row_start(r, a.x_inner, a.rows, a.x_stride);
    in.a[1] = static_cast<const T*>(a.gate) + row_start(r, a.other_inner, a.rows, a.other_stride);
  };
  with_gate(a, [&](auto silu, auto gate_first) {
    for_rows<TPR, NV>(in, a.rows, a.D, point, [](int) { return true; }, [&](long long r, bool real, int parity) {
      float t[NV][E], sum[1] = {0.f}, slope;   // what is normalised, times what stands behind the norm
#pragma unroll
      for (int v = 0; v < NV; v++) {
        float g[E];
        to_floats(t[v], in.pa[0][v]);
        to_floats(g, in.pa[1][v]);
#pragma unroll
        for (int e = 0; e < E; e++) {            // elements that do not exist are zero
          const float x = t[v][e];
          t[v][e] = x * act_of<silu.value, false>(g[e], slope);
          const float n = gate_first.value ? t[v][e] : x;
          sum[0] = fmaf(n, n, sum[0]);
        }
      }
      row_sums<TPR>(sum, red, parity);
      const float rs = rsqrtf(fmaf(sum[0], p.inv_D, a.eps));
      if (!real) return;
      T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int c = Y::column(v);
        if (c >= a.D) continue;
        float wv[E];
        read8(wv, w + c);
        Pack<T, E> out;
#pragma unroll
        for (int e = 0; e < E; e++) wv[e] *= t[v][e] * rs;
        from_floats(out, wv);
        store_some<T, E>(y + c, out, a.D - c, p.wide);
      }
    });
  });
}

template <class T, int TPR, int NV>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS, resident<T, TPR, NV, true>()) gated_bwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[Y::RED];
  const RewyNormArgs& a = p.a;
  float* const w = reinterpret_cast<float*>(smem + GatedBwd<T, TPR, NV>::BYTES);
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  __syncthreads();
  float dw[NV][E] = {};
  GatedBwd<T, TPR, NV> in;
  in.smem = smem; in.wide = p.wide;
  auto point = [&](long long r) {
    in.a[0] = static_cast<const T*>(a.x) + row_start(r, a.x_inner, a.rows, a.x_stride);
    in.a[1] = static_cast<const T*>(a.gate) + row_start(r, a.other_inner, a.rows, a.other_stride);
    in.a[2] = static_cast<const T*>(a.dy) + r * a.D;
  };
  with_gate(a, [&](auto silu, auto gate_first) {
    for_rows<TPR, NV>(in, a.rows, a.D, point, [](int) { return true; }, [&](long long r, bool real, int parity) {
      float sum[2] = {0.f, 0.f}, slope;
#pragma unroll
      for (int v = 0; v < NV; v++) {
        float wv[E], x[E], g[E], d[E];
        read8(wv, w + Y::column(v));
        to_floats(x, in.pa[0][v]);
        to_floats(g, in.pa[1][v]);
        to_floats(d, in.pa[2][v]);
#pragma unroll
        for (int e = 0; e < E; e++) {
          const float act = act_of<silu.value, false>(g[e], slope), dn = d[e] * wv[e], t = gate_first.value ? x[e] * act : x[e];
          sum[0] = fmaf(t, t, sum[0]);
          sum[1] = fmaf(dn * act, x[e], sum[1]);    // dn t either way
        }
      }
      row_sums<TPR>(sum, red, parity);
      if (!real) return;
      const float rs = rsqrtf(fmaf(sum[0], p.inv_D, a.eps)), mean = rs * (sum[1] * p.inv_D);   // of dn n: as large as dn however small the row
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int c = Y::column(v);
        if (c >= a.D) continue;
        float wv[E], x[E], g[E], d[E];
        read8(wv, w + c);
        to_floats(x, in.pa[0][v]);
        to_floats(g, in.pa[1][v]);
        to_floats(d, in.pa[2][v]);
#pragma unroll
        for (int e = 0; e < E; e++) {
          const float act = act_of<silu.value, true>(g[e], slope), xv = x[e], dn = d[e] * wv[e];
          // gate first: v = x act, dx = dv act, dgate = dv x act'.  Else dgate = dn n act', dx = r (dn act - n mean)
          const float n = (gate_first.value ? xv * act : xv) * rs;
          if constexpr (gate_first.value) {
            const float dv = rs * fmaf(-mean, n, dn);
            x[e] = dv * act;
            g[e] = dv * xv * slope;
          } else {
            x[e] = rs * fmaf(-mean, n, dn * act);
            g[e] = dn * n * slope;
          }
          dw[v][e] = fmaf(d[e], gate_first.value ? n : n * act, dw[v][e]);
        }
        Pack<T, E> ox, og;
        from_floats(ox, x);
        from_floats(og, g);
        store_some<T, E>(static_cast<T*>(a.dx) + r * a.D + c, ox, a.D - c, p.wide);
        store_some<T, E>(static_cast<T*>(a.dgate) + r * a.D + c, og, a.D - c, p.wide);
      }
    });
  });
  store_column_sums<TPR, NV>(dw, reinterpret_cast<float*>(smem), p.partial + (long long)blockIdx.x * 2 * a.D, a.D);
}

template <class T, class TR, int TPR, int NV>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS, resident<TR, TPR, NV, false>()) residual_fwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[Y::RED];
  const RewyNormArgs& a = p.a;
  float* const w = reinterpret_cast<float*>(smem + ResidualFwd<T, TR, TPR, NV>::BYTES);
  float* const s = w + Y::COLS;
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  load_params<TPR, NV>(s, a.scale_vector, a.scale_dtype, a.D, a.scale);
  __syncthreads();
  ResidualFwd<T, TR, TPR, NV> in;
  in.smem = smem; in.wide = p.wide;
  const bool has = a.residual != nullptr;
  auto point = [&](long long r) {
    in.a[0] = static_cast<const T*>(a.x) + row_start(r, a.x_inner, a.rows, a.x_stride);
    in.b[0] = static_cast<const TR*>(a.residual) + (has ? row_start(r, a.other_inner, a.rows, a.other_stride) : 0);
  };
  for_rows<TPR, NV>(in, a.rows, a.D, point, [&](int i) { return i == 0 || has; }, [&](long long r, bool real, int parity) {
    float t[NV][E], sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; v++) {
      float sv[E], x[E], res[E];
      read8(sv, s + Y::column(v));
      to_floats(x, in.pa[0][v]);
      to_floats(res, in.pb[0][v]);
#pragma unroll
      for (int e = 0; e < E; e++) {
        t[v][e] = fmaf(sv[e], x[e], res[e]);
        sum[0] = fmaf(t[v][e], t[v][e], sum[0]);
      }
    }
    row_sums<TPR>(sum, red, parity);
    if (!real) return;
    const float rs = rsqrtf(fmaf(sum[0], p.inv_D, a.eps));
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v);
      if (c >= a.D) continue;
      float wv[E];
      read8(wv, w + c);
      Pack<T, E> oy;
      Pack<TR, E> orr;
#pragma unroll
      for (int e = 0; e < E; e++) wv[e] *= t[v][e] * rs;
      from_floats(oy, wv);
      from_floats(orr, t[v]);
      store_some<T, E>(static_cast<T*>(a.y) + r * a.D + c, oy, a.D - c, p.wide);
      store_some<TR, E>(static_cast<TR*>(a.residual_out) + r * a.D + c, orr, a.D - c, p.wide);
    }
  });
}

// SCALE: the scale is a vector that has a gradient
template <class T, class TR, int TPR, int NV, bool SCALE>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS, resident<TR, TPR, NV, true>()) residual_bwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  using In = ResidualBwd<T, TR, TPR, NV>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[Y::RED];
  const RewyNormArgs& a = p.a;
  float* const w = reinterpret_cast<float*>(smem + In::BYTES);
  float* const s = w + Y::COLS;
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  if (SCALE) load_params<TPR, NV>(s, a.scale_vector, a.scale_dtype, a.D, a.scale);
  __syncthreads();
  float dw[NV][E] = {}, ds[SCALE ? NV : 1][E] = {};
  In in;
  in.smem = smem; in.wide = p.wide;
  const bool has = a.residual != nullptr, back_too = a.dresidual_out != nullptr;
  auto point = [&](long long r) {
    in.a[0] = static_cast<const T*>(a.x) + row_start(r, a.x_inner, a.rows, a.x_stride);
    in.a[1] = static_cast<const T*>(a.dy) + r * a.D;
    in.b[0] = static_cast<const TR*>(a.residual) + (has ? row_start(r, a.other_inner, a.rows, a.other_stride) : 0);
    in.b[1] = static_cast<const TR*>(a.dresidual_out) + (back_too ? r * a.D : 0);
  };
  auto scales = [&](float(&sv)[E], int v) {
    if constexpr (SCALE) read8(sv, s + Y::column(v));
    else
#pragma unroll
      for (int e = 0; e < E; e++) sv[e] = a.scale;
  };
  for_rows<TPR, NV>(in, a.rows, a.D, point, [&](int i) { return i < 2 || (i == 2 ? has : back_too); }, [&](long long r, bool real, int parity) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; v++) {
      float wv[E], sv[E], x[E], res[E], d[E];
      read8(wv, w + Y::column(v));
      scales(sv, v);
      to_floats(x, in.pa[0][v]);
      to_floats(res, in.pb[0][v]);
      to_floats(d, in.pa[1][v]);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float t = fmaf(sv[e], x[e], res[e]);
        sum[0] = fmaf(t, t, sum[0]);
        sum[1] = fmaf(d[e] * wv[e], t, sum[1]);
      }
    }
    row_sums<TPR>(sum, red, parity);
    if (!real) return;
    const float rs = rsqrtf(fmaf(sum[0], p.inv_D, a.eps)), mean = rs * (sum[1] * p.inv_D);   // of dn n: as large as dn however small the row
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v);
      if (c >= a.D) continue;
      float wv[E], sv[E], x[E], res[E], d[E], dro[E];
      read8(wv, w + c);
      scales(sv, v);
      to_floats(x, in.pa[0][v]);
      to_floats(res, in.pb[0][v]);
      to_floats(d, in.pa[1][v]);
      to_floats(dro, in.pb[1][v]);
      Pack<T, E> ox;
      Pack<TR, E> orr;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float xv = x[e], n = fmaf(sv[e], xv, res[e]) * rs;
        const float dt = fmaf(rs, fmaf(-mean, n, d[e] * wv[e]), dro[e]);
        x[e] = sv[e] * dt;
        res[e] = dt;
        dw[v][e] = fmaf(d[e], n, dw[v][e]);
        if constexpr (SCALE) ds[v][e] = fmaf(xv, dt, ds[v][e]);
      }
      from_floats(ox, x);
      from_floats(orr, res);
      store_some<T, E>(static_cast<T*>(a.dx) + r * a.D + c, ox, a.D - c, p.wide);
      if (has) store_some<TR, E>(static_cast<TR*>(a.dresidual) + r * a.D + c, orr, a.D - c, p.wide);
    }
  });
  float* to = p.partial + (long long)blockIdx.x * 2 * a.D;
  store_column_sums<TPR, NV>(dw, reinterpret_cast<float*>(smem), to, a.D);
  if constexpr (SCALE) store_column_sums<TPR, NV>(ds, reinterpret_cast<float*>(smem), to + a.D, a.D);
}

// Gradients per column from the CTAs' sums [parts][2][D]: 32 threads per column, blockIdx.y chooses the first or second sum.
__global__ void __launch_bounds__(1024) norm_sums_kernel(const float* __restrict__ partial, int parts, int D, void* first, int first_dtype, void* second,
                                                         int second_dtype) {
  __shared__ float sums[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  const float* from = partial + (blockIdx.y ? D : 0) + c;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int k = y; k < parts; k += 32) s += from[(long long)k * 2 * D];
  }
  sums[y][x] = s;
  __syncthreads();
  if (y == 0 && c < D) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; k++) s += sums[k][x];
    if (blockIdx.y) param_store(second, second_dtype, c, s);
    else param_store(first, first_dtype, c, s);
  }
}

// f(threads per row, accesses per thread)
template <class F>
void with_layout(int D, F&& f) {
  using std::integral_constant;
  if (D <= 128) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (D <= 256) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (D <= 1024) f(integral_constant<int, 128>(), integral_constant<int, 1>());
  else if (D <= 2048) f(integral_constant<int, 256>(), integral_constant<int, 1>());
  else if (D <= 4096) f(integral_constant<int, 512>(), integral_constant<int, 1>());
  else if (D <= 8192) f(integral_constant<int, 1024>(), integral_constant<int, 1>());
  else f(integral_constant<int, 1024>(), integral_constant<int, 2>());
}
template <class F>
void with_residual_type(int dtype, int residual_dtype, F&& f) {
  with_type(dtype, [&](auto t) {
    if (residual_dtype == dtype) f(t, t);
    else f(t, float());
  });
}
int rows_per_cta(int D) { return D <= 128 ? 16 : D <= 256 ? 8 : D <= 1024 ? 2 : 1; }  // as with_layout chooses
int threads_per_cta(int D) { return D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }
int grid_of(int64_t rows, int D, int threads_per_sm) {
  const int64_t ctas = (rows + rows_per_cta(D) - 1) / rows_per_cta(D), each = threads_per_sm / threads_per_cta(D), most = 148 * (each > 0 ? each : 1);
  return (int)(ctas < most ? ctas : most);
}
constexpr int FWD_PER_SM = 1024, BWD_PER_SM = 768;  // threads

int check_norm(const RewyNormArgs* a) {
  LAYER_REQUIRE(a != nullptr, REWY_ERR_NULL, "args is NULL");
  LAYER_REQUIRE(known_dtype(a->dtype) && known_dtype(a->param_dtype) && known_dtype(a->scale_dtype) && known_dtype(a->residual_dtype), REWY_ERR_UNSUPPORTED,
                "unknown element type");
  LAYER_REQUIRE(a->residual_dtype == a->dtype || a->residual_dtype == REWY_F32, REWY_ERR_UNSUPPORTED, "the residual has the type of x or FP32");
  LAYER_REQUIRE(a->D >= 1 && a->D <= 16384, REWY_ERR_UNSUPPORTED, "the norm takes rows of 1 to 16384 values");
  LAYER_REQUIRE(a->rows > 0 && a->x_inner > 0 && a->other_inner > 0, REWY_ERR_SHAPE, "rows and inner counts must be positive");
  LAYER_REQUIRE(a->x != nullptr && a->weight != nullptr, REWY_ERR_NULL, "x or weight is NULL");
  LAYER_REQUIRE(a->activation == 0 || a->activation == 1, REWY_ERR_UNSUPPORTED, "unknown activation");
  return REWY_OK;
}
NormParams norm_params(const RewyNormArgs& a) {
  NormParams p{a, false, static_cast<float*>(a.workspace), 1.f / (float)a.D};
  bool w = a.D % E == 0;
  for (const void* q : {a.x, a.gate, a.residual, (const void*)a.y, (const void*)a.residual_out, a.dy, a.dresidual_out, (const void*)a.dx, (const void*)a.dgate,
                        (const void*)a.dresidual})
    w = w && !unaligned16(q);
  const int per16 = 16 / element_bytes(a.dtype), other16 = 16 / element_bytes(a.gate != nullptr ? a.dtype : a.residual_dtype);
  for (int i = 0; i < 2; i++) w = w && a.x_stride[i] % per16 == 0 && a.other_stride[i] % other16 == 0;
  p.wide = w;
  return p;
}
template <auto Kern>
cudaError_t launch(const NormParams& p, int grid, int threads, int smem, rewy_stream_t st) {
  const cudaError_t e = ensure_dynamic_smem<Kern>(smem);
  if (e == cudaSuccess) Kern<<<grid, threads, smem, (cudaStream_t)st>>>(p);
  return e;
}
int done(cudaError_t e, const char* what, int launches) { return e == cudaSuccess ? launched(what, launches) : report_error(REWY_ERR_LAUNCH, cudaGetErrorString(e)); }
int check_backward(const RewyNormArgs* a) {
  LAYER_REQUIRE(a->dy != nullptr && a->dx != nullptr && a->dweight != nullptr, REWY_ERR_NULL, "dy, dx or dweight is NULL");
  LAYER_REQUIRE(a->workspace != nullptr && a->workspace_bytes >= rewy_norm_bwd_workspace_bytes(a->rows, a->D), REWY_ERR_WORKSPACE,
                "the workspace of the norm backward is too small");
  return REWY_OK;
}
void sum_columns(const NormParams& p, int parts, bool scale, cudaStream_t s) {
  const RewyNormArgs& a = p.a;
  norm_sums_kernel<<<dim3((a.D + 31) / 32, scale ? 2 : 1), 1024, 0, s>>>(p.partial, parts, a.D, a.dweight, a.param_dtype, a.dscale, a.scale_dtype);
}

}  // namespace
}  // namespace rewy

using namespace rewy;

extern "C" size_t rewy_norm_bwd_workspace_bytes(int64_t rows, int32_t D) {
  if (rows <= 0 || D <= 0 || D > 16384) return 0;
  return (size_t)grid_of(rows, D, BWD_PER_SM) * 2 * D * sizeof(float);
}

extern "C" int rewy_gated_norm_fwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE(a->gate != nullptr && a->y != nullptr, REWY_ERR_NULL, "gate or y is NULL");
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, FWD_PER_SM);
  cudaError_t e = cudaSuccess;
  with_type(a->dtype, [&](auto t) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using T = decltype(t);
      using Y = Layout<tpr.value, nv.value>;
      e = launch<gated_fwd_kernel<T, tpr.value, nv.value>>(p, grid, Y::THREADS, GatedFwd<T, tpr.value, nv.value>::BYTES + Y::COLS * 4, st);
    });
  });
  return done(e, "gated norm forward", 1);
}

extern "C" int rewy_gated_norm_bwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE(a->gate != nullptr && a->dgate != nullptr, REWY_ERR_NULL, "gate or dgate is NULL");
  if (const int rc = check_backward(a)) return rc;
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, BWD_PER_SM);
  cudaError_t e = cudaSuccess;
  with_type(a->dtype, [&](auto t) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using T = decltype(t);
      using Y = Layout<tpr.value, nv.value>;
      e = launch<gated_bwd_kernel<T, tpr.value, nv.value>>(p, grid, Y::THREADS, GatedBwd<T, tpr.value, nv.value>::BYTES + Y::COLS * 4, st);
    });
  });
  if (e == cudaSuccess) sum_columns(p, grid, false, (cudaStream_t)st);
  return done(e, "gated norm backward", 2);
}

extern "C" int rewy_residual_norm_fwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE(a->residual_out != nullptr && a->y != nullptr, REWY_ERR_NULL, "residual_out or y is NULL");
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, FWD_PER_SM);
  cudaError_t e = cudaSuccess;
  with_residual_type(a->dtype, a->residual_dtype, [&](auto t, auto tr) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using T = decltype(t);
      using TR = decltype(tr);
      using Y = Layout<tpr.value, nv.value>;
      e = launch<residual_fwd_kernel<T, TR, tpr.value, nv.value>>(p, grid, Y::THREADS, ResidualFwd<T, TR, tpr.value, nv.value>::BYTES + Y::COLS * 8, st);
    });
  });
  return done(e, "residual norm forward", 1);
}

extern "C" int rewy_residual_norm_bwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE((a->scale_vector == nullptr) == (a->dscale == nullptr), REWY_ERR_NULL, "dscale goes with scale_vector");
  LAYER_REQUIRE((a->residual == nullptr) == (a->dresidual == nullptr), REWY_ERR_NULL, "dresidual goes with residual");
  if (const int rc = check_backward(a)) return rc;
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, BWD_PER_SM);
  cudaError_t e = cudaSuccess;
  with_residual_type(a->dtype, a->residual_dtype, [&](auto t, auto tr) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using T = decltype(t);
      using TR = decltype(tr);
      using Y = Layout<tpr.value, nv.value>;
      constexpr int bytes = ResidualBwd<T, TR, tpr.value, nv.value>::BYTES + Y::COLS * 8;
      if (a->scale_vector != nullptr) e = launch<residual_bwd_kernel<T, TR, tpr.value, nv.value, true>>(p, grid, Y::THREADS, bytes, st);
      else e = launch<residual_bwd_kernel<T, TR, tpr.value, nv.value, false>>(p, grid, Y::THREADS, bytes, st);
    });
  });
  if (e == cudaSuccess) sum_columns(p, grid, a->scale_vector != nullptr, (cudaStream_t)st);
  return done(e, "residual norm backward", 2);
}
