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
#include "layer.cuh"

namespace rewy {
namespace {

constexpr int E = 8;  // elements per access

struct NormParams {
  RewyNormArgs a;
  bool wide;
  float* partial;  // [CTAs][2][D]
};

__device__ __forceinline__ long long row_start(long long r, long long inner, const int64_t (&stride)[2]) {
  const long long o = r / inner;
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
    for (int i = 0; i < N; i++) {
      x[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) x[i] += to[(first + w) * N + i];
    }
  }
}

template <int TPR, int NV>
struct Layout {
  static constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR, RED = TPR > 32 ? 2 * THREADS / 32 * 2 : 1;
  __device__ static __forceinline__ int column(int v) { return (v * TPR + threadIdx.x % TPR) * E; }
};
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
      for (int e = 0; e < E; e++) sums[threadIdx.x / TPR * (TPR * NV * E) + Y::column(v) + e] = x[v][e];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += Y::THREADS) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < Y::ROWS; r++) s += sums[r * (TPR * NV * E) + c];
      to[c] = s;
    }
  }
}
template <int TPR, int NV>
__device__ __forceinline__ void load_params(float (&w)[NV][E], const void* p, int dtype, int D, float otherwise) {
#pragma unroll
  for (int v = 0; v < NV; v++)
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int c = Layout<TPR, NV>::column(v) + e;
      w[v][e] = c >= D ? 0.f : p == nullptr ? otherwise : param_at(p, dtype, c);
    }
}

template <class T, int TPR, int NV>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS) gated_fwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  __shared__ float red[Y::RED];
  const RewyNormArgs& a = p.a;
  float w[NV][E];
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  int parity = 0;
  for (long long base = (long long)blockIdx.x * Y::ROWS; base < a.rows; base += (long long)gridDim.x * Y::ROWS, parity ^= 1) {
    const long long r = base + threadIdx.x / TPR;
    const bool real = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + (real ? row_start(r, a.x_inner, a.x_stride) : 0);
    const T* g = static_cast<const T*>(a.gate) + (real ? row_start(r, a.other_inner, a.other_stride) : 0);
    Pack<T, E> px[NV], pg[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v), valid = real ? a.D - c : 0;
      load_some<T, E>(px[v], x + c, valid, p.wide);
      load_some<T, E>(pg[v], g + c, valid, p.wide);
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        float t = to_f32(px[v].v[e]);
        if (a.gate_first && Y::column(v) + e < a.D) {
          const float gv = to_f32(pg[v].v[e]), sig = sigmoid_fast(gv);
          t *= a.activation == 0 ? gv * sig : sig;
        }
        sum[0] = fmaf(t, t, sum[0]);
      }
    row_sums<TPR>(sum, red, parity);
    const float rs = rsqrtf(sum[0] / a.D + a.eps);
    if (!real) continue;
    T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v);
      Pack<T, E> out;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float gv = to_f32(pg[v].v[e]), sig = sigmoid_fast(gv);
        out.v[e] = from_f32<T>(to_f32(px[v].v[e]) * rs * w[v][e] * (a.activation == 0 ? gv * sig : sig));
      }
      if (c < a.D) store_some<T, E>(y + c, out, a.D - c, p.wide);
    }
  }
}

template <class T, int TPR, int NV>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS) gated_bwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  __shared__ float red[Y::RED], sums[Y::ROWS > 1 ? Y::ROWS * TPR * NV * E : 1];
  const RewyNormArgs& a = p.a;
  float w[NV][E], dw[NV][E] = {};
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  int parity = 0;
  for (long long base = (long long)blockIdx.x * Y::ROWS; base < a.rows; base += (long long)gridDim.x * Y::ROWS, parity ^= 1) {
    const long long r = base + threadIdx.x / TPR;
    const bool real = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + (real ? row_start(r, a.x_inner, a.x_stride) : 0);
    const T* g = static_cast<const T*>(a.gate) + (real ? row_start(r, a.other_inner, a.other_stride) : 0);
    const T* dy = static_cast<const T*>(a.dy) + (real ? r * a.D : 0);
    Pack<T, E> px[NV], pg[NV], pd[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v), valid = real ? a.D - c : 0;
      load_some<T, E>(px[v], x + c, valid, p.wide);
      load_some<T, E>(pg[v], g + c, valid, p.wide);
      load_some<T, E>(pd[v], dy + c, valid, p.wide);
    }
    auto gate = [&](int v, int e, float& act, float& slope) {
      const float gv = to_f32(pg[v].v[e]), sig = sigmoid_fast(gv);
      act = a.activation == 0 ? gv * sig : sig;
      slope = a.activation == 0 ? sig * fmaf(gv, 1.f - sig, 1.f) : sig * (1.f - sig);
    };
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (Y::column(v) + e >= a.D) continue;
        float act, slope;
        gate(v, e, act, slope);
        const float xv = to_f32(px[v].v[e]), t = a.gate_first ? xv * act : xv;
        const float dn = to_f32(pd[v].v[e]) * w[v][e] * (a.gate_first ? 1.f : act);
        sum[0] = fmaf(t, t, sum[0]);
        sum[1] = fmaf(dn, t, sum[1]);
      }
    row_sums<TPR>(sum, red, parity);
    if (!real) continue;
    const float rs = rsqrtf(sum[0] / a.D + a.eps), back = rs * rs * rs * (sum[1] / a.D);
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v);
      if (c >= a.D) continue;
      Pack<T, E> ox, og;
#pragma unroll
      for (int e = 0; e < E; e++) {
        float act, slope;
        gate(v, e, act, slope);
        const float xv = to_f32(px[v].v[e]), d = to_f32(pd[v].v[e]);
        if (c + e >= a.D) continue;
        if (a.gate_first) {
          const float t = xv * act, dv = fmaf(rs, d * w[v][e], -back * t);
          ox.v[e] = from_f32<T>(dv * act);
          og.v[e] = from_f32<T>(dv * xv * slope);
          dw[v][e] = fmaf(d, t * rs, dw[v][e]);
        } else {
          const float n = xv * rs, dn = d * w[v][e];
          ox.v[e] = from_f32<T>(fmaf(rs, dn * act, -back * xv));
          og.v[e] = from_f32<T>(dn * n * slope);
          dw[v][e] = fmaf(d, n * act, dw[v][e]);
        }
      }
      store_some<T, E>(static_cast<T*>(a.dx) + r * a.D + c, ox, a.D - c, p.wide);
      store_some<T, E>(static_cast<T*>(a.dgate) + r * a.D + c, og, a.D - c, p.wide);
    }
  }
  store_column_sums<TPR, NV>(dw, sums, p.partial + (long long)blockIdx.x * 2 * a.D, a.D);
}

template <class T, class TR, int TPR, int NV>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS) residual_fwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  __shared__ float red[Y::RED];
  const RewyNormArgs& a = p.a;
  float w[NV][E], s[NV][E];
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  load_params<TPR, NV>(s, a.scale_vector, a.scale_dtype, a.D, a.scale);
  int parity = 0;
  for (long long base = (long long)blockIdx.x * Y::ROWS; base < a.rows; base += (long long)gridDim.x * Y::ROWS, parity ^= 1) {
    const long long r = base + threadIdx.x / TPR;
    const bool real = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + (real ? row_start(r, a.x_inner, a.x_stride) : 0);
    const TR* res = static_cast<const TR*>(a.residual) + (real && a.residual != nullptr ? row_start(r, a.other_inner, a.other_stride) : 0);
    float t[NV][E], sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v), valid = real ? a.D - c : 0;
      Pack<T, E> px;
      Pack<TR, E> pr;
      load_some<T, E>(px, x + c, valid, p.wide);
      load_some<TR, E>(pr, res + c, a.residual != nullptr ? valid : 0, p.wide);
#pragma unroll
      for (int e = 0; e < E; e++) {
        t[v][e] = fmaf(s[v][e], to_f32(px.v[e]), to_f32(pr.v[e]));
        if (c + e < a.D) sum[0] = fmaf(t[v][e], t[v][e], sum[0]);
      }
    }
    row_sums<TPR>(sum, red, parity);
    if (!real) continue;
    const float rs = rsqrtf(sum[0] / a.D + a.eps);
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v);
      if (c >= a.D) continue;
      Pack<T, E> oy;
      Pack<TR, E> orr;
#pragma unroll
      for (int e = 0; e < E; e++) {
        oy.v[e] = from_f32<T>(t[v][e] * rs * w[v][e]);
        orr.v[e] = from_f32<TR>(t[v][e]);
      }
      store_some<T, E>(static_cast<T*>(a.y) + r * a.D + c, oy, a.D - c, p.wide);
      store_some<TR, E>(static_cast<TR*>(a.residual_out) + r * a.D + c, orr, a.D - c, p.wide);
    }
  }
}

// SCALE: the scale is a vector that has a gradient
template <class T, class TR, int TPR, int NV, bool SCALE>
__global__ void __launch_bounds__(Layout<TPR, NV>::THREADS) residual_bwd_kernel(const __grid_constant__ NormParams p) {
  using Y = Layout<TPR, NV>;
  __shared__ float red[Y::RED], sums[Y::ROWS > 1 ? Y::ROWS * TPR * NV * E : 1];
  const RewyNormArgs& a = p.a;
  float w[NV][E], s[SCALE ? NV : 1][E], dw[NV][E] = {}, ds[SCALE ? NV : 1][E] = {};
  load_params<TPR, NV>(w, a.weight, a.param_dtype, a.D, 1.f);
  if constexpr (SCALE) load_params<TPR, NV>(s, a.scale_vector, a.scale_dtype, a.D, a.scale);
  int parity = 0;
  for (long long base = (long long)blockIdx.x * Y::ROWS; base < a.rows; base += (long long)gridDim.x * Y::ROWS, parity ^= 1) {
    const long long r = base + threadIdx.x / TPR;
    const bool real = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + (real ? row_start(r, a.x_inner, a.x_stride) : 0);
    const TR* res = static_cast<const TR*>(a.residual) + (real && a.residual != nullptr ? row_start(r, a.other_inner, a.other_stride) : 0);
    const T* dy = static_cast<const T*>(a.dy) + (real ? r * a.D : 0);
    const TR* dro = static_cast<const TR*>(a.dresidual_out) + (real && a.dresidual_out != nullptr ? r * a.D : 0);
    Pack<T, E> px[NV], pd[NV];
    Pack<TR, E> pr[NV], po[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v), valid = real ? a.D - c : 0;
      load_some<T, E>(px[v], x + c, valid, p.wide);
      load_some<TR, E>(pr[v], res + c, a.residual != nullptr ? valid : 0, p.wide);
      load_some<T, E>(pd[v], dy + c, valid, p.wide);
      load_some<TR, E>(po[v], dro + c, a.dresidual_out != nullptr ? valid : 0, p.wide);
    }
    auto scale = [&](int v, int e) { return SCALE ? s[SCALE ? v : 0][e] : a.scale; };
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (Y::column(v) + e >= a.D) continue;
        const float t = fmaf(scale(v, e), to_f32(px[v].v[e]), to_f32(pr[v].v[e]));
        sum[0] = fmaf(t, t, sum[0]);
        sum[1] = fmaf(to_f32(pd[v].v[e]) * w[v][e], t, sum[1]);
      }
    row_sums<TPR>(sum, red, parity);
    if (!real) continue;
    const float rs = rsqrtf(sum[0] / a.D + a.eps), back = rs * rs * rs * (sum[1] / a.D);
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = Y::column(v);
      if (c >= a.D) continue;
      Pack<T, E> ox;
      Pack<TR, E> orr;
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (c + e >= a.D) continue;
        const float xv = to_f32(px[v].v[e]), t = fmaf(scale(v, e), xv, to_f32(pr[v].v[e])), d = to_f32(pd[v].v[e]);
        const float dt = to_f32(po[v].v[e]) + fmaf(rs, d * w[v][e], -back * t);
        ox.v[e] = from_f32<T>(scale(v, e) * dt);
        orr.v[e] = from_f32<TR>(dt);
        dw[v][e] = fmaf(d, t * rs, dw[v][e]);
        if constexpr (SCALE) ds[v][e] = fmaf(xv, dt, ds[v][e]);
      }
      store_some<T, E>(static_cast<T*>(a.dx) + r * a.D + c, ox, a.D - c, p.wide);
      if (a.dresidual != nullptr) store_some<TR, E>(static_cast<TR*>(a.dresidual) + r * a.D + c, orr, a.D - c, p.wide);
    }
  }
  float* to = p.partial + (long long)blockIdx.x * 2 * a.D;
  store_column_sums<TPR, NV>(dw, sums, to, a.D);
  if constexpr (SCALE) store_column_sums<TPR, NV>(ds, sums, to + a.D, a.D);
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
  else if (D <= 4096) f(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (D <= 8192) f(integral_constant<int, 512>(), integral_constant<int, 2>());
  else f(integral_constant<int, 1024>(), integral_constant<int, 2>());
}
template <class F>
void with_residual_type(int dtype, int residual_dtype, F&& f) {
  with_type(dtype, [&](auto t) {
    if (residual_dtype == dtype) f(t, t);
    else f(t, float());
  });
}
int rows_per_cta(int D) { return D <= 128 ? 16 : D <= 256 ? 8 : D <= 1024 ? 2 : 1; }
int grid_of(int64_t rows, int D, int per_sm) {
  const int64_t ctas = (rows + rows_per_cta(D) - 1) / rows_per_cta(D), most = 148ll * per_sm;
  return (int)(ctas < most ? ctas : most);
}
constexpr int FWD_PER_SM = 8, BWD_PER_SM = 3;

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
  NormParams p{a, false, static_cast<float*>(a.workspace)};
  bool w = a.D % E == 0;
  for (const void* q : {a.x, a.gate, a.residual, (const void*)a.y, (const void*)a.residual_out, a.dy, a.dresidual_out, (const void*)a.dx, (const void*)a.dgate,
                        (const void*)a.dresidual})
    w = w && !unaligned16(q);
  const int per16 = 16 / element_bytes(a.dtype), other16 = 16 / element_bytes(a.gate != nullptr ? a.dtype : a.residual_dtype);
  for (int i = 0; i < 2; i++) w = w && a.x_stride[i] % per16 == 0 && a.other_stride[i] % other16 == 0;
  p.wide = w;
  return p;
}
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
  with_type(a->dtype, [&](auto t) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using Y = Layout<tpr.value, nv.value>;
      gated_fwd_kernel<decltype(t), tpr.value, nv.value><<<grid, Y::THREADS, 0, (cudaStream_t)st>>>(p);
    });
  });
  return launched("gated norm forward");
}

extern "C" int rewy_gated_norm_bwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE(a->gate != nullptr && a->dgate != nullptr, REWY_ERR_NULL, "gate or dgate is NULL");
  if (const int rc = check_backward(a)) return rc;
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, BWD_PER_SM);
  with_type(a->dtype, [&](auto t) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using Y = Layout<tpr.value, nv.value>;
      gated_bwd_kernel<decltype(t), tpr.value, nv.value><<<grid, Y::THREADS, 0, (cudaStream_t)st>>>(p);
    });
  });
  sum_columns(p, grid, false, (cudaStream_t)st);
  return launched("gated norm backward", 2);
}

extern "C" int rewy_residual_norm_fwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE(a->residual_out != nullptr && a->y != nullptr, REWY_ERR_NULL, "residual_out or y is NULL");
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, FWD_PER_SM);
  with_residual_type(a->dtype, a->residual_dtype, [&](auto t, auto tr) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using Y = Layout<tpr.value, nv.value>;
      residual_fwd_kernel<decltype(t), decltype(tr), tpr.value, nv.value><<<grid, Y::THREADS, 0, (cudaStream_t)st>>>(p);
    });
  });
  return launched("residual norm forward");
}

extern "C" int rewy_residual_norm_bwd(const RewyNormArgs* a, rewy_stream_t st) {
  if (const int rc = check_norm(a)) return rc;
  LAYER_REQUIRE((a->scale_vector == nullptr) == (a->dscale == nullptr), REWY_ERR_NULL, "dscale goes with scale_vector");
  LAYER_REQUIRE((a->residual == nullptr) == (a->dresidual == nullptr), REWY_ERR_NULL, "dresidual goes with residual");
  if (const int rc = check_backward(a)) return rc;
  const NormParams p = norm_params(*a);
  const int grid = grid_of(a->rows, a->D, BWD_PER_SM);
  with_residual_type(a->dtype, a->residual_dtype, [&](auto t, auto tr) {
    with_layout(a->D, [&](auto tpr, auto nv) {
      using Y = Layout<tpr.value, nv.value>;
      if (a->scale_vector != nullptr)
        residual_bwd_kernel<decltype(t), decltype(tr), tpr.value, nv.value, true><<<grid, Y::THREADS, 0, (cudaStream_t)st>>>(p);
      else
        residual_bwd_kernel<decltype(t), decltype(tr), tpr.value, nv.value, false><<<grid, Y::THREADS, 0, (cudaStream_t)st>>>(p);
    });
  });
  sum_columns(p, grid, a->scale_vector != nullptr, (cudaStream_t)st);
  return launched("residual norm backward", 2);
}
