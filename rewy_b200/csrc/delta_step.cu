// One token of a delta rule for every row of a decoding batch, the state of its slot updated in place:
//
//   S <- diag(exp g) S;  r = beta (v - k^T S)  (GDN2: w v - (b k)^T S);  S <- S + k r^T;  o = scale q^T S
//
// Bound by HBM: the FP32 state of a (row, value head) is 64 KB, read and written once; everything else is a few hundred
// bytes.  A CTA takes 32 value channels of one state (16 KB, eight 16-byte loads per thread in flight before anything is
// waited for), so that even one sequence with few heads fills the SMs.  The state stays in registers between load and store.
// Both products over the key channels come from one exchange: q^T (S + k r^T) = q^T S + (q k) r.  q, k and the gates are
// read, normalised and activated by every CTA for itself.  All arithmetic is FP32.
// Measured, KDA, 64 sequences of 32 heads of 128 x 128, everything fused: 53 us (5.2 TB/s; the same loads and stores alone take 45);
// one sequence of 16 value heads 4 us.  Before: gates and targets asked for when they were used, single FP32 values, 73 us.
#include "layer.cuh"

namespace rewy {
namespace {

constexpr int NT = 128, SLICE = 32, ROWS = 8;  // threads, value channels per CTA, state vectors per thread

template <bool WIDE>
__device__ __forceinline__ float4 load_state(const float* p, int valid) {
  if constexpr (WIDE) return valid > 0 ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(valid > 0 ? p[0] : 0.f, valid > 1 ? p[1] : 0.f, valid > 2 ? p[2] : 0.f, valid > 3 ? p[3] : 0.f);
}
template <bool WIDE>
__device__ __forceinline__ void store_state(float* p, float4 x, int valid) {
  if constexpr (WIDE) {
    if (valid > 0) __stcs(reinterpret_cast<float4*>(p), x);   // not read again before the next token: 62 -> 56 us
    return;
  }
  if (valid > 0) p[0] = x.x;
  if (valid > 1) p[1] = x.y;
  if (valid > 2) p[2] = x.z;
  if (valid > 3) p[3] = x.w;
}

// WIDE: every row of the state starts on 16 bytes and holds whole groups of four
template <class T, bool V_FIRST, bool WIDE>
__global__ void __launch_bounds__(NT, 8) delta_step_kernel(const __grid_constant__ RewyDeltaStepArgs a, int slices) {
  __shared__ __align__(16) float sk[NT], sq[NT], serase[NT], sdecay[NT], red[3][4];
  __shared__ __align__(16) float part[4][2][SLICE];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slice = blockIdx.x % slices;
  const unsigned rest = blockIdx.x / slices;
  const int hv = rest % a.HV, b = rest / a.HV, v0 = slice * SLICE;
  const long long slot = pool_row(a.slots, a.slots_i64, b, a.pool), head = (long long)b * a.HV + hv;
  T* o = static_cast<T*>(a.o) + head * a.V;
  float* state = a.state + ((slot < 0 ? 0 : slot) * a.HV + hv) * ((long long)a.K * a.V);
  // this thread's state vectors: [K,V] four value channels of key rows kr + 16 i; [V,K] four key channels of value rows vr + 4 i
  const int c4 = V_FIRST ? lane * 4 : (tid & 7) * 4, r0 = V_FIRST ? warp : tid >> 3;
  float4 S[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int r = V_FIRST ? v0 + r0 + 4 * i : r0 + 16 * i, c = V_FIRST ? c4 : v0 + c4;
    const int rows = V_FIRST ? a.V : a.K, cols = V_FIRST ? a.K : a.V;
    S[i] = load_state<WIDE>(state + (long long)r * cols + c, r < rows && slot >= 0 ? cols - c : 0);
  }
  // Everything is asked for before anything is used: what the state should give for k (before the part that is erased is taken
  // off), the gates of this thread's key channel, the write strength.
  constexpr int TARGETS = V_FIRST ? ROWS : 4;
  T value[TARGETS], write[TARGETS];
#pragma unroll
  for (int i = 0; i < TARGETS; i++) {
    const int v = v0 + (V_FIRST ? r0 + 4 * i : c4 + i);
    value[i] = v < a.V ? static_cast<const T*>(a.v)[head * a.V + v] : from_f32<T>(0.f);
    write[i] = a.family == REWY_GDN2 && v < a.V ? static_cast<const T*>(a.w_gate)[head * a.V + v] : from_f32<T>(1.f);
  }
  const long long qk = ((long long)b * a.H + hv / (a.HV / a.H)) * a.K;
  const bool key = tid < a.K, fused = a.A_log != nullptr;
  const T raw_q = key ? static_cast<const T*>(a.q)[qk + tid] : from_f32<T>(0.f), raw_k = key ? static_cast<const T*>(a.k)[qk + tid] : from_f32<T>(0.f);
  const T raw_erase = key && a.family == REWY_GDN2 ? static_cast<const T*>(a.b_gate)[head * a.K + tid] : from_f32<T>(1.f);
  float beta = a.family != REWY_GDN2 ? param_at(a.beta, a.beta_dtype, head) : 1.f;
  float g = a.family == REWY_DELTA || !key ? 0.f : param_at(a.g, a.gate_dtype, a.family == REWY_GDN ? head : head * a.K + tid);
  const float rate = fused ? a.A_log[hv] : 0.f, shift = fused && key && a.dt_bias != nullptr ? a.dt_bias[(long long)hv * a.K + tid] : 0.f;
  if (row_repeats(a.slots, a.slots_i64, b, slot) || slot < 0) {
    if (tid < SLICE && v0 + tid < a.V) o[v0 + tid] = from_f32<T>(0.f);
    return;
  }
  const float q = to_f32(raw_q), k = to_f32(raw_k), erase = to_f32(raw_erase);
  if (fused && key) {
    float sig;
    g = -ex2(LOG2E * rate) * softplus_fast(g + shift, sig);
  }
  const float decay = ex2(LOG2E * g);
  if (a.beta_scale != 0.f) beta = a.beta_scale * sigmoid_fast(beta);
  float qq = q * q, kk = k * k, dot = q * k;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    qq += __shfl_xor_sync(0xffffffffu, qq, m);
    kk += __shfl_xor_sync(0xffffffffu, kk, m);
    dot += __shfl_xor_sync(0xffffffffu, dot, m);
  }
  if (lane == 0) { red[0][warp] = qq; red[1][warp] = kk; red[2][warp] = dot; }
  __syncthreads();
  auto total = [&](int i) {
    const float4 x = *reinterpret_cast<const float4*>(red[i]);
    return (x.x + x.y) + (x.z + x.w);
  };
  qq = total(0); kk = total(1); dot = total(2);
  const float qn = a.qk_norm ? rsqrtf(qq + 1e-6f) : 1.f, kn = a.qk_norm ? rsqrtf(kk + 1e-6f) : 1.f;
  dot *= qn * kn;
  sq[tid] = q * qn;
  sk[tid] = k * kn;
  serase[tid] = k * kn * erase;
  sdecay[tid] = decay;
  __syncthreads();
  if constexpr (!V_FIRST) {
    F2 x[ROWS][2], e[2] = {both(0.f), both(0.f)}, p[2] = {both(0.f), both(0.f)};
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int r = r0 + 16 * i;
      const F2 d = both(sdecay[r]), er = both(serase[r]), qr = both(sq[r]);
      x[i][0] = mul2(pair(S[i].x, S[i].y), d);
      x[i][1] = mul2(pair(S[i].z, S[i].w), d);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        e[k] = fma2(er, x[i][k], e[k]);
        p[k] = fma2(qr, x[i][k], p[k]);
      }
    }
    float sums[8];   // e, then p
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const float2 a2 = halves(e[k]), b2 = halves(p[k]);
      sums[2 * k] = a2.x; sums[2 * k + 1] = a2.y; sums[4 + 2 * k] = b2.x; sums[5 + 2 * k] = b2.y;
    }
#pragma unroll
    for (int m = 16; m >= 8; m >>= 1)
#pragma unroll
      for (int i = 0; i < 8; i++) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], m);
    if (lane < 8) {
      *reinterpret_cast<float4*>(&part[warp][0][c4]) = make_float4(sums[0], sums[1], sums[2], sums[3]);
      *reinterpret_cast<float4*>(&part[warp][1][c4]) = make_float4(sums[4], sums[5], sums[6], sums[7]);
    }
    __syncthreads();
    float erased[4] = {}, seen[4] = {}, r4[4];
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float4 a4 = *reinterpret_cast<const float4*>(&part[w][0][c4]), b4 = *reinterpret_cast<const float4*>(&part[w][1][c4]);
      erased[0] += a4.x; erased[1] += a4.y; erased[2] += a4.z; erased[3] += a4.w;
      seen[0] += b4.x; seen[1] += b4.y; seen[2] += b4.z; seen[3] += b4.w;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      r4[i] = beta * (to_f32(value[i]) * to_f32(write[i]) - erased[i]);
      if (tid < 8 && v0 + c4 + i < a.V) o[v0 + c4 + i] = from_f32<T>(a.scale * fmaf(dot, r4[i], seen[i]));
    }
    const F2 r2[2] = {pair(r4[0], r4[1]), pair(r4[2], r4[3])};
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int r = r0 + 16 * i;
      const F2 kr = both(sk[r]);
      const float2 a2 = halves(fma2(kr, r2[0], x[i][0])), b2 = halves(fma2(kr, r2[1], x[i][1]));
      store_state<WIDE>(state + (long long)r * a.V + v0 + c4, make_float4(a2.x, a2.y, b2.x, b2.y), r < a.K ? a.V - v0 - c4 : 0);
    }
  } else {
    const float4 d = *reinterpret_cast<const float4*>(sdecay + c4), x = *reinterpret_cast<const float4*>(serase + c4),
                 y = *reinterpret_cast<const float4*>(sq + c4), kx = *reinterpret_cast<const float4*>(sk + c4);
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int v = v0 + r0 + 4 * i;
      S[i].x *= d.x; S[i].y *= d.y; S[i].z *= d.z; S[i].w *= d.w;
      float e = fmaf(x.x, S[i].x, x.y * S[i].y) + fmaf(x.z, S[i].z, x.w * S[i].w);
      float p = fmaf(y.x, S[i].x, y.y * S[i].y) + fmaf(y.z, S[i].z, y.w * S[i].w);
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) {
        e += __shfl_xor_sync(0xffffffffu, e, m);
        p += __shfl_xor_sync(0xffffffffu, p, m);
      }
      const float r = beta * (to_f32(value[i]) * to_f32(write[i]) - e);
      if (lane == 0 && v < a.V) o[v] = from_f32<T>(a.scale * fmaf(dot, r, p));
      S[i].x = fmaf(kx.x, r, S[i].x); S[i].y = fmaf(kx.y, r, S[i].y); S[i].z = fmaf(kx.z, r, S[i].z); S[i].w = fmaf(kx.w, r, S[i].w);
      store_state<WIDE>(state + (long long)v * a.K + c4, S[i], v < a.V ? a.K - c4 : 0);
    }
  }
}

}  // namespace
}  // namespace rewy

using namespace rewy;

extern "C" int rewy_delta_step(const RewyDeltaStepArgs* a, rewy_stream_t st) {
  LAYER_REQUIRE(a != nullptr, REWY_ERR_NULL, "args is NULL");
  LAYER_REQUIRE(a->family >= REWY_DELTA && a->family <= REWY_GDN2, REWY_ERR_UNSUPPORTED, "unknown family");
  LAYER_REQUIRE(known_dtype(a->dtype) && known_dtype(a->gate_dtype) && known_dtype(a->beta_dtype), REWY_ERR_UNSUPPORTED, "unknown element type");
  LAYER_REQUIRE(a->B > 0 && a->H > 0 && a->HV > 0 && a->pool > 0 && a->HV % a->H == 0, REWY_ERR_SHAPE, "bad B, H, HV or pool");
  LAYER_REQUIRE(a->K >= 1 && a->K <= 128 && a->V >= 1 && a->V <= 128, REWY_ERR_UNSUPPORTED, "the step takes head dimensions of 1 to 128");
  LAYER_REQUIRE(a->slots != nullptr || a->pool >= a->B, REWY_ERR_SHAPE, "fewer states than rows");
  const int slices = (a->V + SLICE - 1) / SLICE;
  LAYER_REQUIRE((long long)a->B * a->HV * slices < (1LL << 31), REWY_ERR_SHAPE, "more rows and heads than one grid holds");
  LAYER_REQUIRE(a->q != nullptr && a->k != nullptr && a->v != nullptr && a->state != nullptr && a->o != nullptr, REWY_ERR_NULL, "q, k, v, state or o is NULL");
  LAYER_REQUIRE(a->family == REWY_DELTA || a->g != nullptr, REWY_ERR_NULL, "g is NULL");
  LAYER_REQUIRE(a->family == REWY_GDN2 ? a->b_gate != nullptr && a->w_gate != nullptr : a->beta != nullptr, REWY_ERR_NULL, "beta, or b_gate and w_gate, are NULL");
  LAYER_REQUIRE(a->A_log == nullptr || a->family == REWY_KDA, REWY_ERR_UNSUPPORTED, "the fused gate belongs to KDA");
  const bool wide = (a->state_v_first ? a->K : a->V) % 4 == 0 && !unaligned16(a->state);
  const unsigned grid = (unsigned)((long long)a->B * a->HV * slices);
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    const cudaStream_t s = (cudaStream_t)st;
    if (a->state_v_first && wide) delta_step_kernel<T, true, true><<<grid, NT, 0, s>>>(*a, slices);
    else if (a->state_v_first) delta_step_kernel<T, true, false><<<grid, NT, 0, s>>>(*a, slices);
    else if (wide) delta_step_kernel<T, false, true><<<grid, NT, 0, s>>>(*a, slices);
    else delta_step_kernel<T, false, false><<<grid, NT, 0, s>>>(*a, slices);
  });
  return launched("delta-rule step");
}
