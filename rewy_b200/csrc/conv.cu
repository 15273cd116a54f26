// Short causal convolution per channel in front of a recurrence, with its activation, its state between calls and its gradients.
//
//   y_t = act(bias + sum_w weight[w] x_(t-W+1+w))       x before a sequence: its initial state (W-1 rows, the oldest first) or 0
//   g_t = dy_t act'(pre_t),  dx_t = sum_w weight[w] g_(t+W-1-w),  dweight[w] = sum_t g_t x_(t-W+1+w),  dbias = sum_t g_t
//
// Bound by HBM in the forward (reads x, writes y), by HBM and instruction issue in the backward (reads x and dy, writes dx, some 25
// operations per element).  A warp owns neighbouring channels (8 bytes per lane) and a block of tokens, and slides the W-1 last
// inputs (backward: and the W-1 last g) through registers, so that an element is loaded once but for the W-1 rows between blocks
// of tokens, which come from the caches; the rows ahead are on their way through shared memory (Ring), which takes no registers.
// The pre-activation is computed again in the backward rather than kept.  All sums are FP32, on two channels at a time; an output
// is rounded once.  dweight and dbias: FP32 sums in registers over the warp's tokens, over the CTA's warps in shared memory, and
// over the CTAs in a second kernel, always in the same order.
// Measured, B=2 T=4096 D=8192 W=4 in BF16 with SiLU: forward 62 us (4.3 TB/s), backward 105 (3.8 TB/s).  Before: rows loaded
// into registers, conditions on every token, 157 and 400; the same without conditions 75 and 192; copies ahead 67 and 158;
// conversions in pairs 67 and 112; FP32 pairs and one access for a channel's taps, now.
#include "layer.cuh"

namespace rewy {
namespace {

constexpr int WARPS = 8;
template <class T>
constexpr int lane_channels() { return 8 / sizeof(T); }
constexpr int U = 4, RING = 4;  // tokens per group of copies; groups that a thread's ring holds

struct ConvParams {
  RewyConvArgs a;
  int token_block, token_blocks, channel_blocks;  // tokens per warp; CTAs per sequence row; CTAs per token
  bool wide;                                      // every row of x starts on a whole access
};

struct Span {  // the sequence a token lies in
  int s, begin, end;
};
__device__ __forceinline__ Span span_at(const RewyConvArgs& a, int b, int t) {
  if (a.cu_seqlens == nullptr) return {b, 0, a.T};
  const int s = packed_sequence(a.cu_seqlens, a.num_seqs, t);
  return {s, min(max(a.cu_seqlens[s], 0), t), s + 1 < a.num_seqs ? min(max(a.cu_seqlens[s + 1], t + 1), a.T) : a.T};
}
__device__ __forceinline__ Span span_after(const RewyConvArgs& a, const Span& p) {  // p is not the last one
  const int s = p.s + 1;
  return {s, p.end, s + 1 < a.num_seqs ? min(max(a.cu_seqlens[s + 1], p.end + 1), a.T) : a.T};
}

// The W taps of a channel
template <int W>
__device__ __forceinline__ void load_taps(float (&w)[W], const void* weight, int dtype, long long channel) {
  if (W == 4 && dtype == REWY_F32 && (reinterpret_cast<uintptr_t>(weight) & 15) == 0) {
    const float4 v = __ldg(static_cast<const float4*>(weight) + channel);
    w[0] = v.x; w[1] = v.y; w[W > 2 ? 2 : 0] = v.z; w[W - 1] = v.w;
    return;
  }
#pragma unroll
  for (int j = 0; j < W; j++) w[j] = param_at(weight, dtype, channel * W + j);
}

template <class T, int W, int V, bool WIDE>
struct Columns {  // a warp's channels
  const RewyConvArgs& a;
  const T* x;
  long long state_row;  // elements of one sequence's state
  int c0, valid;
  static constexpr bool wide = WIDE;
  static constexpr int P = V / 2;   // arithmetic on two channels at a time
  F2 weight[W][P], bias[P];

  __device__ __forceinline__ Columns(const ConvParams& p, int b, int channel)
      : a(p.a), x(static_cast<const T*>(p.a.x) + b * p.a.x_batch_stride), state_row((long long)(W - 1) * p.a.D), c0(channel),
        valid(WIDE ? V : p.a.D - channel) {
#pragma unroll
    for (int i = 0; i < P; i++) {
      float taps[2][W] = {}, both_bias[2] = {};
#pragma unroll
      for (int k = 0; k < 2; k++)
        if (2 * i + k < valid) {
          load_taps(taps[k], a.weight, a.param_dtype, c0 + 2 * i + k);
          if (a.bias != nullptr) both_bias[k] = param_at(a.bias, a.param_dtype, c0 + 2 * i + k);
        }
#pragma unroll
      for (int w = 0; w < W; w++) weight[w][i] = pair(taps[0][w], taps[1][w]);
      bias[i] = pair(both_bias[0], both_bias[1]);
    }
  }
  __device__ __forceinline__ void load_x(Pack<T, V>& d, int t) const { load_some<T, V>(d, x + t * a.x_token_stride + c0, valid, wide); }
  // the W-1 inputs before token t of sequence s
  __device__ __forceinline__ void window(F2 (&win)[W - 1][P], const Span& s, int t) const {
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
      const int pos = t - (W - 1) + j;
      Pack<T, V> v;
      if (pos >= s.begin) load_x(v, pos);
      else if (a.initial_state != nullptr)
        load_some<T, V>(v, static_cast<const T*>(a.initial_state) + s.s * state_row + (long long)(W - 1 + pos - s.begin) * a.D + c0, valid, wide);
      else zero_pack(v);
      to_pairs(win[j], v);
    }
  }
};

// A thread's inputs on their way through shared memory, N tensors, U tokens at a time: three groups are under way while one is
// worked on, without registers that hold them.  A thread reads only what it has copied itself.
template <class T, int V, int N>
struct Ring {
  using P = Pack<T, V>;
  static constexpr int BYTES = RING * U * N * WARPS * 32 * (int)sizeof(P);
  P* own;      // of this thread; its slots are a CTA's width apart
  __device__ __forceinline__ explicit Ring(unsigned char* smem) : own(reinterpret_cast<P*>(smem) + threadIdx.x) {}
  __device__ __forceinline__ P& slot(int group, int u, int i) const { return own[(((group & (RING - 1)) * U + u) * N + i) * WARPS * 32]; }
  __device__ __forceinline__ void copy(int group, int u, int i, const T* from, int valid, bool wide) const {
    P& to = slot(group, u, i);
    if (wide && valid >= V) {
      const unsigned dst = (unsigned)__cvta_generic_to_shared(&to);
      static_assert(sizeof(P) == 8, "one copy is eight bytes");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(from) : "memory");
    } else {
      load_some<T, V>(to, from, valid, false);
    }
  }
  __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory"); }
  __device__ __forceinline__ static void wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
};

// WIDE: whole accesses only
template <class T, int W, int V, bool WIDE>
__global__ void __launch_bounds__(WARPS * 32, 4) conv_fwd_kernel(const __grid_constant__ ConvParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const Ring<T, V, 1> ring(smem);
  constexpr int P = V / 2;
  const int channel = (blockIdx.x % p.channel_blocks * 32 + (threadIdx.x & 31)) * V;
  const unsigned rest = blockIdx.x / p.channel_blocks;
  const int b = rest / p.token_blocks;
  const long long first = ((long long)(rest % p.token_blocks) * WARPS + (threadIdx.x >> 5)) * p.token_block;
  if (channel >= p.a.D || first >= p.a.T) return;
  const int t0 = (int)first, t1 = (int)min(first + p.token_block, (long long)p.a.T);
  const Columns<T, W, V, WIDE> c(p, b, channel);
  T* y = static_cast<T*>(p.a.y) + (long long)b * p.a.T * p.a.D + channel;
  Span s = span_at(p.a, b, t0);
  for (int from = t0; from < t1;) {   // the part of one sequence that lies in the block
    const int to = min(t1, s.end);
    F2 win[W - 1][P];
    c.window(win, s, from);
    auto token = [&](int t, const Pack<T, V>& in) {
      F2 now[P];
      float pre[V];
      to_pairs(now, in);
#pragma unroll
      for (int i = 0; i < P; i++) {
        F2 sum = fma2(c.weight[W - 1][i], now[i], c.bias[i]);
#pragma unroll
        for (int w = 0; w < W - 1; w++) sum = fma2(c.weight[w][i], win[w][i], sum);
        const float2 h = halves(sum);
        pre[2 * i] = h.x; pre[2 * i + 1] = h.y;
#pragma unroll
        for (int j = 0; j < W - 2; j++) win[j][i] = win[j + 1][i];
        win[W - 2][i] = now[i];
      }
      if (p.a.activation)
#pragma unroll
        for (int i = 0; i < V; i++) pre[i] *= sigmoid_fast(pre[i]);
      Pack<T, V> out;
      from_floats(out, pre);
      store_some<T, V>(y + (long long)t * p.a.D, out, c.valid, c.wide);
    };
    auto ask = [&](int group) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int t = from + group * U + u;
        if (t < to) ring.copy(group, u, 0, c.x + t * p.a.x_token_stride + channel, c.valid, c.wide);
      }
      ring.commit();
    };
#pragma unroll
    for (int k = 0; k < RING - 1; k++) ask(k);
    for (int k = 0; from + k * U < to; k++) {
      ask(k + RING - 1);
      ring.wait();
      if (from + k * U + U <= to) {
#pragma unroll
        for (int u = 0; u < U; u++) token(from + k * U + u, ring.slot(k, u, 0));
      } else {
#pragma unroll 1
        for (int u = 0; from + k * U + u < to; u++) token(from + k * U + u, ring.slot(k, u, 0));
      }
    }
    ring.wait_all();
    if (p.a.final_state != nullptr && to == s.end) {
#pragma unroll
      for (int j = 0; j < W - 1; j++) {
        Pack<T, V> v;
        from_pairs(v, win[j]);
        store_some<T, V>(static_cast<T*>(p.a.final_state) + s.s * c.state_row + (long long)j * p.a.D + channel, v, c.valid, c.wide);
      }
    }
    from = to;
    if (from < t1) s = span_after(p.a, s);
  }
}

template <class T, int W, int V, bool WIDE>
__global__ void __launch_bounds__(WARPS * 32, 2) conv_bwd_kernel(const __grid_constant__ ConvParams p, float* __restrict__ partial) {
  extern __shared__ __align__(16) unsigned char smem[];
  const Ring<T, V, 2> ring(smem);
  const RewyConvArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int channel = (blockIdx.x % p.channel_blocks * 32 + lane) * V;
  const unsigned rest = blockIdx.x / p.channel_blocks;
  const int b = rest / p.token_blocks;
  const long long first = ((long long)(rest % p.token_blocks) * WARPS + warp) * p.token_block;
  constexpr int P = V / 2;
  F2 dw[W][P], db[P];
#pragma unroll
  for (int i = 0; i < P; i++) {
    db[i] = both(0.f);
#pragma unroll
    for (int w = 0; w < W; w++) dw[w][i] = both(0.f);
  }
  if (channel < a.D && first < a.T) {
    const int t0 = (int)first, t1 = (int)min(first + p.token_block, (long long)a.T);
    const Columns<T, W, V, WIDE> c(p, b, channel);
    const long long row = (long long)b * a.T;
    const T* dy = static_cast<const T*>(a.dy) + row * a.D + channel;
    T* dx = static_cast<T*>(a.dx) + row * a.D + channel;
    Span s = span_at(a, b, t0);
    for (int from = t0; from < t1;) {        // the part of one sequence that lies in the block
      const int to = min(t1, s.end);
      F2 win[W - 1][P], g[W - 1][P];
      c.window(win, s, from);
#pragma unroll
      for (int j = 0; j < W - 1; j++)
#pragma unroll
        for (int i = 0; i < P; i++) g[j][i] = both(0.f);
      const int stop = to + W - 1, real = min(stop, s.end);   // tokens of the next block too; beyond the sequence there is no g
      auto ask = [&](int group) {
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int t = from + group * U + u;
          if (t < real) {
            ring.copy(group, u, 0, c.x + t * a.x_token_stride + channel, c.valid, c.wide);
            ring.copy(group, u, 1, dy + (long long)t * a.D, c.valid, c.wide);
          }
        }
        ring.commit();
      };
      // Token t of the sequence: its g, and out, the complete gradient W-1 tokens before it.  OWN: it counts for dweight.
      auto step = [&](auto own, const Pack<T, V>& in, const Pack<T, V>& d, float (&out)[V]) {
        F2 x[P], gi[P];
        to_pairs(x, in);
        to_pairs(gi, d);
        if (a.activation)
#pragma unroll
          for (int i = 0; i < P; i++) {
            F2 pre = fma2(c.weight[W - 1][i], x[i], c.bias[i]);
#pragma unroll
            for (int w = 0; w < W - 1; w++) pre = fma2(c.weight[w][i], win[w][i], pre);
            const float2 h = halves(pre);
            const F2 sig = pair(sigmoid_fast(h.x), sigmoid_fast(h.y));
            gi[i] = mul2(mul2(gi[i], sig), fma2(pre, fma2(sig, both(-1.f), both(1.f)), both(1.f)));
          }
#pragma unroll
        for (int i = 0; i < P; i++) {
          if (own.value) {
#pragma unroll
            for (int w = 0; w < W - 1; w++) dw[w][i] = fma2(gi[i], win[w][i], dw[w][i]);
            dw[W - 1][i] = fma2(gi[i], x[i], dw[W - 1][i]);
            db[i] = add2(db[i], gi[i]);
          }
#pragma unroll
          for (int j = 0; j < W - 2; j++) win[j][i] = win[j + 1][i];
          win[W - 2][i] = x[i];
          F2 sum = mul2(c.weight[0][i], gi[i]);
#pragma unroll
          for (int w = 1; w < W; w++) sum = fma2(c.weight[w][i], g[W - 1 - w][i], sum);
          const float2 h = halves(sum);
          out[2 * i] = h.x; out[2 * i + 1] = h.y;
#pragma unroll
          for (int j = 0; j < W - 2; j++) g[j][i] = g[j + 1][i];
          g[W - 2][i] = gi[i];
        }
      };
      auto put = [&](int pos, float (&out)[V]) {
        Pack<T, V> v;
        from_floats(v, out);
        store_some<T, V>(dx + (long long)pos * a.D, v, c.valid, c.wide);
      };
      // At the edges: rows before the sequence are its initial state's, the last ones get the final state's gradient too.
      auto put_edge = [&](int pos, float (&out)[V]) {
        const bool before = pos < from;
        if (before && (from != s.begin || a.dinitial_state == nullptr)) return;
        if (a.dfinal_state != nullptr && pos >= s.end - (W - 1)) {
          Pack<T, V> v;
          load_some<T, V>(v, static_cast<const T*>(a.dfinal_state) + s.s * c.state_row + (long long)(pos - (s.end - (W - 1))) * a.D + channel,
                          c.valid, c.wide);
#pragma unroll
          for (int i = 0; i < V; i++) out[i] += to_f32(v.v[i]);
        }
        if (!before) {
          put(pos, out);
          return;
        }
        Pack<T, V> v;
        from_floats(v, out);
        store_some<T, V>(static_cast<T*>(a.dinitial_state) + s.s * c.state_row + (long long)(W - 1 + pos - s.begin) * a.D + channel, v, c.valid, c.wide);
      };
      float out[V];
#pragma unroll
      for (int k = 0; k < RING - 1; k++) ask(k);
      for (int k = 0; from + k * U < stop; k++) {
        const int t = from + k * U;
        ask(k + RING - 1);
        ring.wait();
        if (t >= from + W - 1 && t + U <= to) {
#pragma unroll
          for (int u = 0; u < U; u++) {
            step(std::true_type(), ring.slot(k, u, 0), ring.slot(k, u, 1), out);
            put(t + u - (W - 1), out);
          }
        } else {       // the first tokens, the last ones and those of the next block
#pragma unroll 1
          for (int u = 0; u < U && t + u < stop; u++) {
            Pack<T, V> in, d;
            zero_pack(in);
            zero_pack(d);
            if (t + u < real) {
              in = ring.slot(k, u, 0);
              d = ring.slot(k, u, 1);
            }
            if (t + u < to) step(std::true_type(), in, d, out);
            else step(std::false_type(), in, d, out);
            put_edge(t + u - (W - 1), out);
          }
        }
      }
      ring.wait_all();
      from = to;
      if (from < t1) s = span_after(a, s);
    }
  }
  __syncthreads();   // the rings have been read: their room takes the sums
  float(*const sums)[W + 1][32 * V] = reinterpret_cast<float(*)[W + 1][32 * V]>(smem);
  static_assert(sizeof(float) * WARPS * (W + 1) * 32 * V <= Ring<T, V, 2>::BYTES, "the sums fit the rings");
#pragma unroll
  for (int i = 0; i < P; i++) {
#pragma unroll
    for (int w = 0; w <= W; w++) *reinterpret_cast<unsigned long long*>(&sums[warp][w][lane * V + 2 * i]) = (w < W ? dw[w < W ? w : 0][i] : db[i]).v;
  }
  __syncthreads();
  const int c0 = blockIdx.x % p.channel_blocks * 32 * V;
  for (int i = threadIdx.x; i < (W + 1) * 32 * V; i += blockDim.x) {
    const int w = i / (32 * V), col = i % (32 * V);
    if (c0 + col >= a.D) continue;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; k++) sum += sums[k][w][col];
    partial[((long long)rest * (W + 1) + w) * a.D + c0 + col] = sum;
  }
}

// dweight [D,W] and dbias [D] from the CTAs' sums [parts][W+1][D]
__global__ void __launch_bounds__(256) conv_sums_kernel(const float* __restrict__ partial, int parts, int D, int W, void* dweight, void* dbias,
                                                        int param_dtype) {
  const long long n = (long long)(W + 1) * D, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
#pragma unroll 8
  for (int k = 0; k < parts; k++) sum += partial[k * n + i];
  const int w = (int)(i / D), c = (int)(i % D);
  if (w < W) param_store(dweight, param_dtype, (long long)c * W + w, sum);
  else if (dbias != nullptr) param_store(dbias, param_dtype, c, sum);
}

// One token per row, the state of its slot shifted by it.
template <class T, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const __grid_constant__ RewyConvStepArgs a, int channel_blocks, bool wide) {
  const int b = blockIdx.x / channel_blocks, c0 = (blockIdx.x % channel_blocks * 128 + threadIdx.x) * V;
  const long long slot = pool_row(a.slots, a.slots_i64, b, a.pool);
  const int valid = a.D - c0, W = a.W;
  T* state = static_cast<T*>(a.state) + (slot < 0 ? 0 : slot) * (W - 1) * a.D + c0;
  Pack<T, V> now, old[3];
#pragma unroll
  for (int j = 0; j < 3; j++)
    if (j < W - 1 && slot >= 0 && valid > 0) {   // (written in this kernel: not through the read-only path)
      if (wide && valid >= V) old[j] = *reinterpret_cast<const Pack<T, V>*>(state + (long long)j * a.D);
      else
        for (int i = 0; i < V; i++) old[j].v[i] = i < valid ? state[(long long)j * a.D + i] : from_f32<T>(0.f);
    } else {
      zero_pack(old[j]);
    }
  load_some<T, V>(now, static_cast<const T*>(a.x) + b * a.x_stride + c0, valid, wide);
  float weight[V][4], pre[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    pre[i] = a.bias != nullptr && i < valid ? param_at(a.bias, a.param_dtype, c0 + i) : 0.f;
    if (W == 4 && i < valid) {
      load_taps<4>(weight[i], a.weight, a.param_dtype, c0 + i);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) weight[i][j] = j < W && i < valid ? param_at(a.weight, a.param_dtype, (long long)(c0 + i) * W + j) : 0.f;
    }
  }
  const bool skip = row_repeats(a.slots, a.slots_i64, b, slot) || slot < 0;
  if (valid <= 0) return;
  T* y = static_cast<T*>(a.y) + (long long)b * a.D + c0;
  Pack<T, V> out;
  if (skip) {
    zero_pack(out);
    store_some<T, V>(y, out, valid, wide);
    return;
  }
  float x[V];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (j >= W) continue;
    if (j == W - 1) to_floats(x, now);
    else to_floats(x, old[j < 3 ? j : 2]);
#pragma unroll
    for (int i = 0; i < V; i++) pre[i] = fmaf(weight[i][j], x[i], pre[i]);
  }
  if (a.activation)
#pragma unroll
    for (int i = 0; i < V; i++) pre[i] *= sigmoid_fast(pre[i]);
  from_floats(out, pre);
  store_some<T, V>(y, out, valid, wide);
#pragma unroll
  for (int j = 0; j < 3; j++)
    if (j < W - 1) store_some<T, V>(state + (long long)j * a.D, j + 1 < W - 1 ? old[j + 1 < 3 ? j + 1 : 2] : now, valid, wide);
}

// What 32-bit counts of tokens and channels hold
bool conv_fits(int B, int T, int D) { return (long long)B * T <= (1LL << 30) && D <= (1 << 24); }

int check_conv(const RewyConvArgs* a) {
  LAYER_REQUIRE(a != nullptr, REWY_ERR_NULL, "args is NULL");
  LAYER_REQUIRE(known_dtype(a->dtype) && known_dtype(a->param_dtype), REWY_ERR_UNSUPPORTED, "unknown element type");
  LAYER_REQUIRE(a->W >= 2 && a->W <= 4, REWY_ERR_UNSUPPORTED, "the convolution takes 2 to 4 taps");
  LAYER_REQUIRE(a->B > 0 && a->T > 0 && a->D > 0, REWY_ERR_SHAPE, "B, T and D must be positive");
  LAYER_REQUIRE(conv_fits(a->B, a->T, a->D), REWY_ERR_SHAPE, "B*T exceeds 2^30 tokens or D 2^24 channels");
  LAYER_REQUIRE(((long long)a->B * a->T / 64 + a->B) * (a->D / 64 + 1) < (1LL << 31), REWY_ERR_SHAPE, "more tokens and channels than one grid holds");
  LAYER_REQUIRE(a->x != nullptr && a->weight != nullptr, REWY_ERR_NULL, "x or weight is NULL");
  LAYER_REQUIRE(a->cu_seqlens == nullptr || (a->B == 1 && a->num_seqs > 0), REWY_ERR_SHAPE, "packed sequences need B = 1 and num_seqs > 0");
  return REWY_OK;
}

// Tokens per warp.  Long blocks load fewer rows twice (W-1 per block) and leave fewer sums; short ones give a small problem
// enough warps.  Forward / backward with its sums in us, blocks of 8, 16, 32, 64, 128: B=2 T=4096 D=8192 86 / 239, 66 / 161, 62 / 125,
// 62 / 109, 70 / 112 (64 taken); 16001 tokens in 12 documents, D=2048 47 / 144, 37 / 98, 35 / 76, 38 / 68, 40 / 63 (64); B=1 T=2000
// D=1024 5.7 / 13, 6.1 / 12, 9.0 / 15, 15 / 22, 27 / 36 (8); B=8 T=500 D=768 7.0 / 20, 7.7 / 16, 9.1 / 16, 15 / 22, 24 / 29 (8).
// A sequence of a fixed batch shorter than eight blocks leaves warps of its CTA idle: B=64 T=64 D=2048 takes 13 / 37.
int token_block(long long tokens, int warps_per_token) {
  int block = 64;
  while (block > 8 && tokens / block * warps_per_token < 148 * 24) block /= 2;
  return block;
}

ConvParams conv_params(const RewyConvArgs& a, int V) {
  ConvParams p;
  p.a = a;
  const int e = element_bytes(a.dtype), access = V * e;
  p.channel_blocks = (a.D + 32 * V - 1) / (32 * V);
  p.token_block = token_block((long long)a.B * a.T, (a.D + 127) / 128);
  p.token_blocks = (a.T + p.token_block * WARPS - 1) / (p.token_block * WARPS);
  auto row = [&](const void* q) { return (reinterpret_cast<uintptr_t>(q) % access) == 0; };
  p.wide = a.D % V == 0 && a.x_token_stride % V == 0 && a.x_batch_stride % V == 0 && row(a.x) && row(a.y) && row(a.dy) && row(a.dx) &&
           row(a.initial_state) && row(a.final_state) && row(a.dfinal_state) && row(a.dinitial_state);
  return p;
}
template <class F>
void with_taps(int W, F&& f) {
  if (W == 2) f(std::integral_constant<int, 2>());
  else if (W == 3) f(std::integral_constant<int, 3>());
  else f(std::integral_constant<int, 4>());
}

}  // namespace
}  // namespace rewy

using namespace rewy;

extern "C" int rewy_conv_fwd(const RewyConvArgs* a, rewy_stream_t st) {
  if (const int rc = check_conv(a)) return rc;
  LAYER_REQUIRE(a->y != nullptr, REWY_ERR_NULL, "y is NULL");
  cudaError_t e = cudaSuccess;
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = lane_channels<T>(), bytes = Ring<T, V, 1>::BYTES;
    const ConvParams p = conv_params(*a, V);
    const unsigned grid = (unsigned)((long long)p.channel_blocks * p.token_blocks * a->B);
    with_taps(a->W, [&](auto w) {
      auto go = [&](auto wide) {
        e = ensure_dynamic_smem<conv_fwd_kernel<T, w.value, V, wide.value>>(bytes);
        if (e == cudaSuccess) conv_fwd_kernel<T, w.value, V, wide.value><<<grid, WARPS * 32, bytes, (cudaStream_t)st>>>(p);
      };
      p.wide ? go(std::true_type()) : go(std::false_type());
    });
  });
  if (e != cudaSuccess) return report_error(REWY_ERR_LAUNCH, cudaGetErrorString(e));
  return launched("causal convolution forward");
}

extern "C" size_t rewy_conv_bwd_workspace_bytes(int32_t B, int32_t T, int32_t D, int32_t W) {
  if (B <= 0 || T <= 0 || D <= 0 || W < 2 || W > 4 || !conv_fits(B, T, D)) return 0;
  RewyConvArgs a{};
  a.B = B; a.T = T; a.D = D; a.W = W;
  const ConvParams p = conv_params(a, 4);
  return (size_t)p.token_blocks * B * (W + 1) * D * sizeof(float);
}

extern "C" int rewy_conv_bwd(const RewyConvArgs* a, rewy_stream_t st) {
  if (const int rc = check_conv(a)) return rc;
  LAYER_REQUIRE(a->dy != nullptr && a->dx != nullptr && a->dweight != nullptr, REWY_ERR_NULL, "dy, dx or dweight is NULL");
  LAYER_REQUIRE(a->workspace != nullptr && a->workspace_bytes >= rewy_conv_bwd_workspace_bytes(a->B, a->T, a->D, a->W), REWY_ERR_WORKSPACE,
                "the workspace of the convolution backward is too small");
  float* partial = static_cast<float*>(a->workspace);
  int parts = 0;
  cudaError_t e = cudaSuccess;
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = lane_channels<T>(), bytes = Ring<T, V, 2>::BYTES;
    const ConvParams p = conv_params(*a, V);
    parts = p.token_blocks * a->B;
    const unsigned grid = (unsigned)((long long)p.channel_blocks * parts);
    with_taps(a->W, [&](auto w) {
      auto go = [&](auto wide) {
        e = ensure_dynamic_smem<conv_bwd_kernel<T, w.value, V, wide.value>>(bytes);
        if (e == cudaSuccess) conv_bwd_kernel<T, w.value, V, wide.value><<<grid, WARPS * 32, bytes, (cudaStream_t)st>>>(p, partial);
      };
      p.wide ? go(std::true_type()) : go(std::false_type());
    });
  });
  if (e != cudaSuccess) return report_error(REWY_ERR_LAUNCH, cudaGetErrorString(e));
  conv_sums_kernel<<<(unsigned)(((long long)(a->W + 1) * a->D + 255) / 256), 256, 0, (cudaStream_t)st>>>(partial, parts, a->D, a->W, a->dweight, a->dbias,
                                                                                                         a->param_dtype);
  return launched("causal convolution backward", 2);
}

extern "C" int rewy_conv_step(const RewyConvStepArgs* a, rewy_stream_t st) {
  LAYER_REQUIRE(a != nullptr, REWY_ERR_NULL, "args is NULL");
  LAYER_REQUIRE(known_dtype(a->dtype) && known_dtype(a->param_dtype), REWY_ERR_UNSUPPORTED, "unknown element type");
  LAYER_REQUIRE(a->W >= 2 && a->W <= 4, REWY_ERR_UNSUPPORTED, "the convolution takes 2 to 4 taps");
  LAYER_REQUIRE(a->B > 0 && a->D > 0 && a->pool > 0, REWY_ERR_SHAPE, "B, D and the pool must be positive");
  LAYER_REQUIRE(a->D <= (1 << 24) && (long long)a->B * (a->D / 256 + 1) < (1LL << 31), REWY_ERR_SHAPE, "more rows and channels than one grid holds");
  LAYER_REQUIRE(a->slots != nullptr || a->pool >= a->B, REWY_ERR_SHAPE, "fewer states than rows");
  LAYER_REQUIRE(a->x != nullptr && a->weight != nullptr && a->state != nullptr && a->y != nullptr, REWY_ERR_NULL, "x, weight, state or y is NULL");
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 8 / sizeof(T);
    const int access = V * (int)sizeof(T), channel_blocks = (a->D + 128 * V - 1) / (128 * V);
    auto row = [&](const void* q) { return (reinterpret_cast<uintptr_t>(q) % access) == 0; };
    const bool wide = a->D % V == 0 && a->x_stride % V == 0 && row(a->x) && row(a->y) && row(a->state);
    conv_step_kernel<T, V><<<(unsigned)((long long)channel_blocks * a->B), 128, 0, (cudaStream_t)st>>>(*a, channel_blocks, wide);
  });
  return launched("causal convolution step");
}
