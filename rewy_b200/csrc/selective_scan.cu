// Selective state space scan: a diagonal recurrence per channel whose decay and input weights depend on the token.
//
//   dt = softplus(dt_raw + bias);  a_t = exp(dt_t A);  h_t = a_t h_(t-1) + dt_t u_t B_t;  y_t = (C_t h_t + D u_t) silu(z_t)
//   with dy' = dy silu(z):  gh_t = C_t dy'_t + a_(t+1) gh_(t+1);  drive_t = sum_n gh_t B_t;  q_t = gh_t h_(t-1) a_t
//   du = dt drive + D dy';  ddt = sum_n q A + u drive;  dA = sum_t q dt;  dB = sum_m gh dt u;  dC = sum_m dy' h
//
// Everything is FP32 between the element types at both ends; nothing is kept in fewer bits in between.
//
// Recurrence.  A thread holds S states of one channel, L neighbouring lanes the states of a channel (N <= L S), a group of two or four
// warps 8 to 32 channels, which it takes through a segment of the tokens in tiles of 32.  A second group of four warps works beside it:
// it puts the next tile's dt and dt u per channel, its B and its C into shared memory as FP32 (softplus and gate once per
// element, eight elements per thread, loads asked for a tile ahead), and writes what came of the tile before.  One barrier per tile.
// Arithmetic on two states at a time (FP32 pairs).
// The backward needs h_(t-1) in reverse: the forward leaves the state before every 16th token (4 N / 16 bytes per token and
// channel), from which 16 tokens are run forward into registers and walked back.
// Sums over the states of a channel are exchanged for several sets of four values step by step together, those over channels
// (dB, dC) for two tokens; the latter end scattered over the lanes, are added over the CTA's warps in shared memory and over the
// CTAs by a second kernel, all in one order: results repeat bit for bit.
//
// Few channels: the token axis is cut into segments.  A first pass finds each segment's end state from a zero start (backward:
// the gradient that leaves its first token), and the main pass starts every segment from those before it, joined by
// h <- exp(A sum dt) h + end.  That doubles the exponentials and pays only where most SMs would idle.
//
// Measured, B=2 T=4096 M=4096 N=16 in BF16 with softplus, skip and gate: forward 294 us (the exponentials alone, 16 per clock and
// SM, take 117, memory 41), backward 1030 us and 48 for the sums of dB and dC (memory 62 and 41).  Both are bound by latency and
// issue together: two CTAs fit an SM (the backward's 256 threads take 128 registers each), so a scheduler has two warps of recurrence
// in the backward and, with eight states to a thread, one in the forward; issue is 47 and 38 % active, and what a warp waits for are
// its own shuffles, exponentials and multiply-adds.  Before: every warp doing everything in turn, 456 and 1875 us; conditions
// inside the element loops, 340 and 1052.  Tried and not kept (backward): two states per thread and twice the warps 1758 us; eight
// tokens in registers, half the code, 1031; registers moved from the second group to the first by setmaxnreg 1010; 64 channels
// per CTA 994 with its sums, but half the CTAs for narrow layers; two warps in the second group 1131.  (Forward): tiles ahead by
// asynchronous copies through shared memory 303; two warps in the second group 562.
// N above 16: CTAs hold 16 (N <= 32) or 8 channels, one CTA fits an SM in the backward (117 and 184 KB of shared memory), and the
// partial sums of dB and dC grow to 16 and 64 bytes per token and channel.  512 channels, 4000 tokens, forward and backward without
// skip and gate: N = 32 286 us, N = 64 638.
#include <climits>
#include "layer.cuh"

namespace rewy {
namespace {

constexpr int TILE = 32;  // segments hold a multiple of so many tokens
constexpr int CK = 16;    // tokens between checkpoints
constexpr float LN2 = 0.6931471805599453f;

// exp(dt A) from dt and A log2 e.  The exponential instruction gives results that are 2 to 3 parts in 10^8 too small on average for
// arguments between -1 and -0.005, and a state that lives for hundreds of tokens would gather that up: 2.0e-6 of dA for 4096
// tokens.  2.8e-8 on the argument, in the multiply-add that forms it, leaves 1e-8 there either way (a step of zero still gives 1),
// and from -1e-9 on no more than the correctly rounded values next to 1 have themselves: 3.7e-8 at most, between -1e-7 and -1e-8,
// 1.4e-8 elsewhere.  Beyond -4 it does not count: the argument's own rounding is larger.  Segments are joined with one exponential
// of a sum, which gathers nothing up and goes without.
constexpr float EX2_LOW = 2.8e-8f;
__device__ __forceinline__ float decay_of(float d, float A2) { return ex2(fmaf(d, A2, EX2_LOW)); }
__device__ __forceinline__ F2 decay_of(F2 d, F2 A2) { return ex2_2(fma2(d, A2, both(EX2_LOW))); }

// N <= L S states of a channel: S to a thread, L neighbouring threads.  NS threads run the recurrence of CH channels in tiles of
// TT tokens, NH threads do what stands around it.
template <int L_, int S_, int NS_, int NH_, int TT_>
struct Shape {
  static constexpr int L = L_, S = S_, P = S_ / 2, NS = NS_, NH = NH_, TT = TT_, CH = NS_ / L_, NP = L_ * S_, YS = CH + 8, THREADS = NS_ + NH_, WARPS = NS_ / 32;
};

struct ScanParams {
  RewyScanArgs a;
  int Mg, blocks, segments, seg_len;   // channels per group, CTAs per group, segments of seg_len tokens
  float *seg_state, *seg_dt;           // [B][segments][M][N], [B][segments][M]
  float *part_bc, *part_m;             // [blocks][B*T][G][2][N]; [B*segments][M*N + 2 M]
  bool wide, wide_bc, wide_state;      // whole accesses possible for u, dt, z, y; B, C; the FP32 states
};

// Where a CTA works.
template <class C>
struct Place {
  static constexpr int CH = C::CH;
  int b, seg, g, cb, m0, valid;        // first channel and how many exist
  int t0, t1;                          // tokens of the segment
  __device__ __forceinline__ Place(const ScanParams& p, int seg_offset, int seg_count) {
    unsigned i = blockIdx.x;
    cb = i % p.blocks; i /= p.blocks;
    g = i % p.a.G; i /= p.a.G;
    seg = i % seg_count + seg_offset;
    b = i / seg_count;
    m0 = g * p.Mg + cb * CH;
    valid = min(CH, p.Mg - cb * CH);
    t0 = seg * p.seg_len;
    t1 = min(p.a.T, t0 + p.seg_len);
  }
};

// Sequence bookkeeping of a CTA that moves forward through tokens.
struct Sequence {
  int s, begin, next;  // sequence, its first token, the first token of the one behind it (INT_MAX: none)
  __device__ __forceinline__ void at(const RewyScanArgs& a, int b, int t) {
    if (a.cu_seqlens == nullptr) { s = b; begin = 0; next = INT_MAX; return; }
    s = packed_sequence(a.cu_seqlens, a.num_seqs, t);
    begin = min(max(a.cu_seqlens[s], 0), t);
    next = s + 1 < a.num_seqs ? max(a.cu_seqlens[s + 1], t + 1) : INT_MAX;
  }
  __device__ __forceinline__ void advance(const RewyScanArgs& a) {
    s++;
    begin = next;
    next = s + 1 < a.num_seqs ? max(a.cu_seqlens[s + 1], begin + 1) : INT_MAX;
  }
};

template <int S>
__device__ __forceinline__ void load_states(float (&x)[S], const float* p, int n0, int N, bool ok, bool wide) {
  if (ok && wide && n0 < N) {
    if constexpr (S >= 4) {
#pragma unroll
      for (int i = 0; i < S; i += 4) {
        const float4 v = n0 + i < N ? *reinterpret_cast<const float4*>(p + n0 + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
      }
    } else {
      const float2 v = *reinterpret_cast<const float2*>(p + n0);
      x[0] = v.x; x[1] = v.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < S; i++) x[i] = ok && n0 + i < N ? p[n0 + i] : 0.f;
}
template <int S>
__device__ __forceinline__ void store_states(float* p, const float (&x)[S], int n0, int N, bool ok, bool wide) {
  if (!ok) return;
  if (wide) {
    if (n0 >= N) return;
    if constexpr (S >= 4) {
#pragma unroll
      for (int i = 0; i < S; i += 4)
        if (n0 + i < N) *reinterpret_cast<float4*>(p + n0 + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else *reinterpret_cast<float2*>(p + n0) = make_float2(x[0], x[1]);
    return;
  }
#pragma unroll
  for (int i = 0; i < S; i++)
    if (n0 + i < N) p[n0 + i] = x[i];
}
// The same as pairs
template <int P>
__device__ __forceinline__ void load_pairs(F2 (&x)[P], const float* p, int n0, int N, bool ok, bool wide) {
  float v[2 * P];
  load_states(v, p, n0, N, ok, wide);
#pragma unroll
  for (int i = 0; i < P; i++) x[i] = pair(v[2 * i], v[2 * i + 1]);
}
template <int P>
__device__ __forceinline__ void store_pairs(float* p, const F2 (&x)[P], int n0, int N, bool ok, bool wide) {
  float v[2 * P];
#pragma unroll
  for (int i = 0; i < P; i++) {
    const float2 h = halves(x[i]);
    v[2 * i] = h.x; v[2 * i + 1] = h.y;
  }
  store_states(p, v, n0, N, ok, wide);
}
// P pairs from shared memory
template <int P>
__device__ __forceinline__ void shared_pairs(F2 (&x)[P], const float* p) {
  if constexpr (P >= 2) {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p + 2 * i);
      x[i].v = v.x; x[i + 1].v = v.y;
    }
  } else {
    x[0].v = *reinterpret_cast<const unsigned long long*>(p);
  }
}

// Sums over the L lanes of a channel, for G sets of four values.  Afterwards lane l of them holds in x[.][0] (L = 2: x[.][0], x[.][1])
// the sum of the value that put_sums writes.  Exchanges keep the order in which they are written, so all sets take a step
// together: one latency per step instead of one per set.
template <int L, int G>
__device__ __forceinline__ void sum_states(float (&x)[G][4], int l) {
#pragma unroll
  for (int m = L / 2; m >= 4; m >>= 1)
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int i = 0; i < 4; i++) x[g][i] += __shfl_xor_sync(0xffffffffu, x[g][i], m);
  const bool odd = l & 1, up = l & 2;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float keep = odd ? x[g][2 + i] : x[g][i], give = odd ? x[g][i] : x[g][2 + i];
      x[g][i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
    }
  if constexpr (L >= 4) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      const float keep = up ? x[g][1] : x[g][0], give = up ? x[g][0] : x[g][1];
      x[g][0] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
    }
  }
}
template <int L>
__device__ __forceinline__ void put_sums(float* at, int stride, const float (&x)[4], int l) {  // at: row of the first of four tokens
  const int first = (l & 1) * 2;
  if constexpr (L == 2) {
    at[first * stride] = x[0];
    at[(first + 1) * stride] = x[1];
  } else {
    if (L == 4 || l < 4) at[(first + ((l >> 1) & 1)) * stride] = x[0];
  }
}

// Sums of v (dB and dC of a thread's S states) over the warp's 32 / L channels, the lanes that differ in the bits from L up.
// Each exchange halves the values that a lane is left with; it puts them at places i of a row of [dB | dC] counted from
// sum_place, where `put` gets them.
template <class C>
__device__ __forceinline__ int sum_place(int lane, int n0) {
  int base = 0, n = 2 * C::S;
#pragma unroll
  for (int m = 16; m >= C::L && n > 1; m >>= 1) {
    n >>= 1;
    base += lane & m ? n : 0;
  }
  return (base / C::S) * C::NP + n0 + base % C::S;
}
template <class C, int G, class F>
__device__ __forceinline__ void sum_channels(float (&v)[G][2 * C::S], int lane, F&& put) {  // G tokens step by step together
  int n = 2 * C::S;
#pragma unroll
  for (int m = 16; m >= C::L; m >>= 1) {
    const bool up = lane & m;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < C::S; i++)
          if (i < n) {
            const float keep = up ? v[g][i + n] : v[g][i], give = up ? v[g][i] : v[g][i + n];
            v[g][i] = keep + __shfl_xor_sync(0xffffffffu, give, m);
          }
    } else {
#pragma unroll
      for (int g = 0; g < G; g++) v[g][0] += __shfl_xor_sync(0xffffffffu, v[g][0], m);
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < C::S; i++)   // the values lie in one half of the row: the first exchange has chosen it
      if (i < n) put(g, i, v[g][i]);
}

__device__ __forceinline__ void read8(float (&x)[8], const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void write8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// A tile's rows of one [B,T,M] tensor: 8 channels per access.
template <class C>
struct Rows {
  static constexpr int PER_TOKEN = C::CH / 8, COUNT = C::TT * PER_TOKEN, EACH = (COUNT + C::NH - 1) / C::NH;
  __device__ static __forceinline__ bool mine(int k, int& tok, int& c) {
    const int i = (int)threadIdx.x - C::NS + k * C::NH;
    tok = i / PER_TOKEN;
    c = i % PER_TOKEN * 8;
    return i < COUNT;
  }
};
template <class T>
__device__ __forceinline__ void fetch8(Pack<T, 8>& d, const T* base, long long token_stride, int t, int t1, int c, int valid, bool wide) {
  load_some<T, 8>(d, base + t * token_stride + c, t < t1 ? valid - c : 0, wide);
}
// B and C of a tile as FP32 [TT][NP]; WHICH: 1 B, 2 C, 3 both
template <class T, class C, int WHICH>
struct Shared {
  static constexpr int PER_TOKEN = C::NP / 8, TENSORS = WHICH == 3 ? 2 : 1, COUNT = C::TT * PER_TOKEN * TENSORS, EACH = (COUNT + C::NH - 1) / C::NH;
  Pack<T, 8> v[EACH];
  __device__ __forceinline__ void fetch(const ScanParams& p, const T* Bm, const T* Cm, int t0, int t1) {
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int i = (int)threadIdx.x - C::NS + k * C::NH, which = WHICH == 3 ? i / (C::TT * PER_TOKEN) : WHICH - 1, j = i % (C::TT * PER_TOKEN);
      const int t = t0 + j / PER_TOKEN, n = j % PER_TOKEN * 8;
      if (i < COUNT)
        load_some<T, 8>(v[k], (which ? Cm + t * p.a.C_stride[1] : Bm + t * p.a.B_stride[1]) + n, t < t1 ? p.a.N - n : 0, p.wide_bc);
    }
  }
  __device__ __forceinline__ void publish(float* sB, float* sC) const {
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int i = (int)threadIdx.x - C::NS + k * C::NH, which = WHICH == 3 ? i / (C::TT * PER_TOKEN) : WHICH - 1, j = i % (C::TT * PER_TOKEN);
      if (i < COUNT) {
        float* to = (which ? sC : sB) + j * 8;
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4*>(to + e) = make_float4(to_f32(v[k].v[e]), to_f32(v[k].v[e + 1]), to_f32(v[k].v[e + 2]), to_f32(v[k].v[e + 3]));
      }
    }
  }
};

// Eight elements at a time: what is asked once stands outside the loops, whose chains then run side by side.
// dt of raw inputs, and what a gradient of dt is multiplied by for them
template <bool SLOPE>
__device__ __forceinline__ void steps_of(float (&d)[8], float (&slope)[8], bool softplus) {
  if (softplus) {
#pragma unroll
    for (int e = 0; e < 8; e++) d[e] = softplus_fast(d[e], slope[e]);
  } else if (SLOPE) {
#pragma unroll
    for (int e = 0; e < 8; e++) slope[e] = 1.f;
  }
}

// State at the first token of segment `seg` of a sequence that began before it, from the ends of the segments between.
template <int S>
__device__ __forceinline__ void join_forward(float (&h)[S], const ScanParams& p, int b, int seg, int begin, long long m, const float (&A2)[S], int n0, bool ok) {
  const int first = begin / p.seg_len;
  for (int j = first; j < seg; j++) {
    const long long row = ((long long)b * p.segments + j) * p.a.M + m;
    float end[S];
    load_states(end, p.seg_state + row * p.a.N, n0, p.a.N, ok, p.wide_state);
    const float d = ok ? p.seg_dt[row] : 0.f;
#pragma unroll
    for (int i = 0; i < S; i++) h[i] = j == first ? end[i] : fmaf(ex2(A2[i] * d), h[i], end[i]);
  }
}

template <class C>
struct FwdShared {
  static constexpr int CH = C::CH, NP = C::NP, YS = C::YS, TT = C::TT;
  float dt[2][TT * CH], du[2][TT * CH], B[2][TT * NP], Cm[2][TT * NP], y[2][TT * YS];  // du: dt u
};

// STATE_ONLY: the first pass of a scan in segments (all but the last one).
// Two groups of warps (two or four, and four): the first runs the recurrence of a tile, the second meanwhile writes what came of the
// tile before and prepares the tile behind.
template <class T, class C, bool STATE_ONLY>
__global__ void __launch_bounds__(C::THREADS, 2) scan_fwd_kernel(const __grid_constant__ ScanParams p) {
  constexpr int CH = C::CH, NP = C::NP, YS = C::YS, L = C::L, S = C::S, P = C::P, TT = C::TT;
  using R = Rows<C>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  FwdShared<C>& sm = *reinterpret_cast<FwdShared<C>*>(raw_smem);
  const RewyScanArgs& a = p.a;
  const Place<C> at(p, 0, STATE_ONLY ? p.segments - 1 : p.segments);
  const int tiles = (at.t1 - at.t0 + TT - 1) / TT;
  const bool gated = !STATE_ONLY && a.z != nullptr;
  if (threadIdx.x >= C::NS) {
    const T* u = static_cast<const T*>(a.u) + at.b * a.u_stride[0] + at.m0;
    const T* dt = static_cast<const T*>(a.dt) + at.b * a.dt_stride[0] + at.m0;
    const T* z = static_cast<const T*>(a.z) + (a.z != nullptr ? at.b * a.z_stride[0] + at.m0 : 0);
    const T* Bm = static_cast<const T*>(a.Bm) + at.b * a.B_stride[0] + at.g * a.B_stride[2];
    const T* Cm = static_cast<const T*>(a.C) + at.b * a.C_stride[0] + at.g * a.C_stride[2];
    float bias[R::EACH][8], Dv[R::EACH][8];
#pragma unroll
    for (int k = 0; k < R::EACH; k++) {
      int tok, c;
      R::mine(k, tok, c);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        bias[k][e] = a.dt_bias != nullptr && c + e < at.valid ? a.dt_bias[at.m0 + c + e] : 0.f;
        Dv[k][e] = !STATE_ONLY && a.D != nullptr && c + e < at.valid ? a.D[at.m0 + c + e] : 0.f;
      }
    }
    Pack<T, 8> ru[R::EACH], rd[R::EACH], xu[R::EACH], xz[R::EACH];
    Shared<T, C, STATE_ONLY ? 1 : 3> bc;
    auto fetch = [&](int t) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        fetch8(ru[k], u, a.u_stride[1], t + tok, at.t1, c, at.valid, p.wide);
        fetch8(rd[k], dt, a.dt_stride[1], t + tok, at.t1, c, at.valid, p.wide);
      }
      bc.fetch(p, Bm, Cm, t, at.t1);
    };
    auto publish = [&](int t, int buf) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        float d[8], w[8], x[8];
        to_floats(d, rd[k]);
        to_floats(x, ru[k]);
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] += bias[k][e];
        steps_of<false>(d, w, a.softplus);
        const int real = t + tok < at.t1 ? at.valid - c : 0;   // a token that does not exist: no decay, no input
#pragma unroll
        for (int e = 0; e < 8; e++) {
          d[e] = e < real ? d[e] : 0.f;
          w[e] = d[e] * x[e];
        }
        write8(&sm.dt[buf][tok * CH + c], d);
        write8(&sm.du[buf][tok * CH + c], w);
      }
      bc.publish(sm.B[buf], sm.Cm[buf]);
    };
    auto fetch_again = [&](int t0) {   // u and z of the tile whose recurrence has been run
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        if (a.D != nullptr) fetch8(xu[k], u, a.u_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
        else zero_pack(xu[k]);
        if (gated) fetch8(xz[k], z, a.z_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
      }
    };
    auto finish_tile = [&](int t0, int buf) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c) || t0 + tok >= at.t1 || c >= at.valid) continue;
        float y[8], x[8];
        read8(y, &sm.y[buf][tok * YS + c]);
        to_floats(x, xu[k]);
        Pack<T, 8> out;
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = fmaf(Dv[k][e], x[e], y[e]);
        if (gated) {
          to_floats(x, xz[k]);
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] *= x[e] * sigmoid_fast(x[e]);
        }
        from_floats(out, y);
        store_some<T, 8>(static_cast<T*>(a.y) + ((long long)at.b * a.T + t0 + tok) * a.M + at.m0 + c, out, at.valid - c, p.wide);
      }
    };
    // What a step reads has been asked for a step before.
    fetch(at.t0);
    publish(at.t0, 0);
    if (tiles > 1) fetch(at.t0 + TT);
    if (!STATE_ONLY) fetch_again(at.t0);
    __syncthreads();
    for (int i = 0; i < tiles; i++) {
      const int t0 = at.t0 + i * TT;
      if (i + 1 < tiles) publish(t0 + TT, (i + 1) & 1);
      if (i + 2 < tiles) fetch(t0 + 2 * TT);
      if (!STATE_ONLY && i > 0) {
        finish_tile(t0 - TT, (i - 1) & 1);
        fetch_again(t0);
      }
      __syncthreads();
    }
    if (!STATE_ONLY) finish_tile(at.t0 + (tiles - 1) * TT, (tiles - 1) & 1);
    return;
  }

  const int ch = threadIdx.x / L, sl = threadIdx.x % L, n0 = sl * S;
  const bool ok = ch < at.valid;
  const long long m = at.m0 + ch;
  float A2[S], h[S] = {};
  load_states(A2, a.A + m * a.N, n0, a.N, ok, p.wide_state);
#pragma unroll
  for (int i = 0; i < S; i++) A2[i] *= LOG2E;
  F2 A2p[P];
#pragma unroll
  for (int i = 0; i < P; i++) A2p[i] = pair(A2[2 * i], A2[2 * i + 1]);

  Sequence q;
  q.at(a, at.b, at.t0);
  auto start = [&](int s) { load_states(h, a.initial_state + ((long long)s * a.M + m) * a.N, n0, a.N, ok && a.initial_state != nullptr, p.wide_state); };
  auto finish = [&](int s) {
    if (!STATE_ONLY && a.final_state != nullptr) store_states(a.final_state + ((long long)s * a.M + m) * a.N, h, n0, a.N, ok, p.wide_state);
  };
  if (q.begin == at.t0) start(q.s);
  else if (!STATE_ONLY) join_forward(h, p, at.b, at.seg, q.begin, m, A2, n0, ok);

  float total = 0.f;
  __syncthreads();
  for (int i = 0; i < tiles; i++) {
    const int t0 = at.t0 + i * TT, buf = i & 1;
    const float *__restrict__ const sdt = sm.dt[buf] + ch, *__restrict__ const sdu = sm.du[buf] + ch;
    const float *__restrict__ const sB = sm.B[buf] + n0, *__restrict__ const sC = sm.Cm[buf] + n0;
    float* __restrict__ const sy = sm.y[buf] + ch;
    // Eight tokens; check: a sequence may begin inside the tile
    auto tokens = [&](auto check, int k) {
      [[maybe_unused]] float y[2][4];
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int kh = k + 4 * half;
        if (!STATE_ONLY && kh % CK == 0 && a.checkpoints != nullptr && t0 + kh < a.T)
          store_states(a.checkpoints + (((long long)at.b * ((a.T + CK - 1) / CK) + (t0 + kh) / CK) * a.M + m) * a.N, h, n0, a.N, ok, p.wide_state);
        F2 dec[4][P], in[4][P], Cv[4][P];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float dj = sdt[(kh + j) * CH];
          const F2 d = both(dj), w = both(sdu[(kh + j) * CH]);
          F2 Bv[P];
          shared_pairs(Bv, sB + (kh + j) * NP);
          if (!STATE_ONLY) shared_pairs(Cv[j], sC + (kh + j) * NP);
          else total += dj;
#pragma unroll
          for (int i = 0; i < P; i++) {
            dec[j][i] = decay_of(d, A2p[i]);
            in[j][i] = mul2(w, Bv[i]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (check.value && t0 + kh + j == q.next && t0 + kh + j < at.t1) {
            finish(q.s);
            q.advance(a);
            start(q.s);
          }
          F2 sum;
#pragma unroll
          for (int i = 0; i < P; i++) {
            const F2 x = fma2(dec[j][i], pair(h[2 * i], h[2 * i + 1]), in[j][i]);
            const float2 hx = halves(x);
            h[2 * i] = hx.x; h[2 * i + 1] = hx.y;
            if (!STATE_ONLY) sum = i ? fma2(Cv[j][i], x, sum) : mul2(Cv[j][i], x);
          }
          if constexpr (!STATE_ONLY) y[half][j] = sum_halves(sum);
        }
      }
      if constexpr (!STATE_ONLY) {
        sum_states<L>(y, sl);
        put_sums<L>(sy + k * YS, YS, y[0], sl);
        put_sums<L>(sy + (k + 4) * YS, YS, y[1], sl);
      }
    };
    if (t0 + TT <= q.next) {
#pragma unroll
      for (int k = 0; k < TT; k += 8) tokens(std::false_type(), k);
    } else {
#pragma unroll 1
      for (int k = 0; k < TT; k += 8) tokens(std::true_type(), k);
    }
    __syncthreads();
  }
  if constexpr (STATE_ONLY) {
    const long long row = ((long long)at.b * p.segments + at.seg) * a.M + m;
    store_states(p.seg_state + row * a.N, h, n0, a.N, ok, p.wide_state);
    if (ok && sl == 0) p.seg_dt[row] = total;
  } else {
    if (at.t1 == a.T || at.t1 == q.next) finish(q.s);
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------

// Gradient of the state that token t1 - 1 hands on: from the segments behind, or from the final state's gradient.
template <class C, int S>
__device__ __forceinline__ void join_backward(float (&carry)[S], const ScanParams& p, const Place<C>& at, long long m, const float (&A2)[S], int n0, bool ok) {
  const RewyScanArgs& a = p.a;
  Sequence q;
  q.at(a, at.b, at.t1 - 1);
  const int end = min(q.next, a.T);
  if (end <= at.t1) {   // the sequence ends with this segment
    load_states(carry, a.dfinal_state + ((long long)q.s * a.M + m) * a.N, n0, a.N, ok && a.dfinal_state != nullptr, p.wide_state);
    return;
  }
  const int last = (end - 1) / p.seg_len;
  for (int j = last; j > at.seg; j--) {
    const long long row = ((long long)at.b * p.segments + j) * a.M + m;
    float out[S];
    load_states(out, p.seg_state + row * a.N, n0, a.N, ok, p.wide_state);
    const float d = ok ? p.seg_dt[row] : 0.f;
#pragma unroll
    for (int i = 0; i < S; i++) carry[i] = j == last ? out[i] : fmaf(ex2(A2[i] * d), carry[i], out[i]);
  }
}

// First pass over the segments but the first: the gradient that leaves each one's first token for the state before it.
template <class T, class C>
__global__ void __launch_bounds__(C::THREADS) scan_bwd_state_kernel(const __grid_constant__ ScanParams p) {
  constexpr int CH = C::CH, NP = C::NP, L = C::L, S = C::S, TT = C::TT;
  using R = Rows<C>;
  __shared__ __align__(16) float sdt[2][TT * CH], sdy[2][TT * CH], sC[2][TT * NP];
  const RewyScanArgs& a = p.a;
  const Place<C> at(p, 1, p.segments - 1);
  const int tiles = (at.t1 - at.t0 + TT - 1) / TT;
  if (threadIdx.x >= C::NS) {
    const T* dt = static_cast<const T*>(a.dt) + at.b * a.dt_stride[0] + at.m0;
    const T* z = static_cast<const T*>(a.z) + (a.z != nullptr ? at.b * a.z_stride[0] + at.m0 : 0);
    const T* dy = static_cast<const T*>(a.dy) + (long long)at.b * a.T * a.M + at.m0;
    const T* Cm = static_cast<const T*>(a.C) + at.b * a.C_stride[0] + at.g * a.C_stride[2];
    Pack<T, 8> xd[R::EACH], xy[R::EACH], xz[R::EACH];
    Shared<T, C, 2> cc;
    float bias[R::EACH][8];
#pragma unroll
    for (int k = 0; k < R::EACH; k++) {
      int tok, c;
      R::mine(k, tok, c);
#pragma unroll
      for (int e = 0; e < 8; e++) bias[k][e] = a.dt_bias != nullptr && c + e < at.valid ? a.dt_bias[at.m0 + c + e] : 0.f;
    }
    auto fetch = [&](int t0) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        fetch8(xd[k], dt, a.dt_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
        fetch8(xy[k], dy, (long long)a.M, t0 + tok, at.t1, c, at.valid, p.wide);
        if (a.z != nullptr) fetch8(xz[k], z, a.z_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
      }
      cc.fetch(p, nullptr, Cm, t0, at.t1);
    };
    auto publish = [&](int t0, int buf) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        float d[8], g[8], v[8];
        to_floats(d, xd[k]);
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] += bias[k][e];
        steps_of<false>(d, g, a.softplus);
        to_floats(g, xy[k]);
        if (a.z != nullptr) {
          to_floats(v, xz[k]);
#pragma unroll
          for (int e = 0; e < 8; e++) g[e] *= v[e] * sigmoid_fast(v[e]);
        }
        const int real = t0 + tok < at.t1 ? at.valid - c : 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          d[e] = e < real ? d[e] : 0.f;
          g[e] = e < real ? g[e] : 0.f;
        }
        write8(&sdt[buf][tok * CH + c], d);
        write8(&sdy[buf][tok * CH + c], g);
      }
      cc.publish(nullptr, sC[buf]);
    };
    fetch(at.t0 + (tiles - 1) * TT);
    publish(at.t0 + (tiles - 1) * TT, (tiles - 1) & 1);
    if (tiles > 1) fetch(at.t0 + (tiles - 2) * TT);
    __syncthreads();
    for (int tile = tiles - 1; tile >= 0; tile--) {
      if (tile > 0) publish(at.t0 + (tile - 1) * TT, (tile - 1) & 1);
      if (tile > 1) fetch(at.t0 + (tile - 2) * TT);
      __syncthreads();
    }
    return;
  }
  const int ch = threadIdx.x / L, sl = threadIdx.x % L, n0 = sl * S;
  const bool ok = ch < at.valid;
  const long long m = at.m0 + ch;
  float A2[S], gh[S] = {}, step[S], total = 0.f;   // as in the main pass
  load_states(A2, a.A + m * a.N, n0, a.N, ok, p.wide_state);
#pragma unroll
  for (int i = 0; i < S; i++) {
    A2[i] *= LOG2E;
    step[i] = 1.f;
  }
  Sequence q;
  q.at(a, at.b, at.t1 - 1);
  auto last_of = [&](int s) {
    load_states(gh, a.dfinal_state + ((long long)s * a.M + m) * a.N, n0, a.N, ok && a.dfinal_state != nullptr, p.wide_state);
#pragma unroll
    for (int i = 0; i < S; i++) step[i] = 1.f;
  };
  if (min(q.next, a.T) <= at.t1) last_of(q.s);
  __syncthreads();
  for (int tile = tiles - 1; tile >= 0; tile--) {
    const int t0 = at.t0 + tile * TT, buf = tile & 1;
    auto token = [&](int k) {
      const float d = sdt[buf][k * CH + ch], g = sdy[buf][k * CH + ch];
      const float* const c = &sC[buf][k * NP + n0];
#pragma unroll
      for (int i = 0; i < S; i++) {
        gh[i] = fmaf(step[i], gh[i], c[i] * g);
        step[i] = decay_of(d, A2[i]);
      }
      total += d;
    };
    if (a.cu_seqlens == nullptr || q.begin < t0 || q.s == 0) {     // (the first sequence begins with the first segment)
#pragma unroll 4
      for (int k = TT - 1; k >= 0; k--) token(k);
    } else {
#pragma unroll 1
      for (int k = TT - 1; k >= 0; k--) {
        token(k);
        if (t0 + k == q.begin && q.s > 0 && t0 + k > at.t0) {   // what flows on belongs to the sequence before
          q.at(a, at.b, t0 + k - 1);
          last_of(q.s);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < S; i++) gh[i] *= step[i];
  const long long row = ((long long)at.b * p.segments + at.seg) * a.M + m;
  store_states(p.seg_state + row * a.N, gh, n0, a.N, ok, p.wide_state);
  if (ok && sl == 0) p.seg_dt[row] = total;
}

template <class C>
struct BwdShared {
  static constexpr int CH = C::CH, NP = C::NP, YS = C::YS, TT = C::TT;
  float4 x[2][TT * CH];                                       // dt, dt u, dy' and the slope of dt, at place(token, channel)
  float B[2][TT * NP], Cm[2][TT * NP];
  float drive[2][TT * YS], decay[2][TT * YS], y[2][TT * YS];  // per token and channel: sum gh B, sum q A2, sum C h
  float bc[2][C::WARPS][TT][2 * NP];                           // each warp's sums over its channels
  float bias[CH], D[CH];
  // A thread writes the entries of eight neighbouring channels: turned by what keeps the threads of a quarter warp apart
  __device__ static __forceinline__ int place(int tok, int c) { return tok * CH + (c & ~7) + ((c ^ ((c >> 3) + CH / 8 * tok)) & 7); }
};

// Two groups of four warps: the recurrence of a tile beside what stands around the tiles next to it.
template <class T, class C>
__global__ void __launch_bounds__(C::THREADS, 2) scan_bwd_kernel(const __grid_constant__ ScanParams p) {
  constexpr int CH = C::CH, NP = C::NP, YS = C::YS, L = C::L, S = C::S, P = C::P, TT = C::TT;
  using R = Rows<C>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  BwdShared<C>& sm = *reinterpret_cast<BwdShared<C>*>(raw_smem);
  const RewyScanArgs& a = p.a;
  const Place<C> at(p, 0, p.segments);
  const bool gated = a.z != nullptr;
  const int tiles = (at.t1 - at.t0 + TT - 1) / TT;
  float* const part = p.part_m + ((long long)at.b * p.segments + at.seg) * ((long long)a.M * (a.N + 2));
  if (threadIdx.x >= C::NS) {
    const T* u = static_cast<const T*>(a.u) + at.b * a.u_stride[0] + at.m0;
    const T* dt = static_cast<const T*>(a.dt) + at.b * a.dt_stride[0] + at.m0;
    const T* z = static_cast<const T*>(a.z) + (gated ? at.b * a.z_stride[0] + at.m0 : 0);
    const T* dy = static_cast<const T*>(a.dy) + (long long)at.b * a.T * a.M + at.m0;
    const T* Bm = static_cast<const T*>(a.Bm) + at.b * a.B_stride[0] + at.g * a.B_stride[2];
    const T* Cm = static_cast<const T*>(a.C) + at.b * a.C_stride[0] + at.g * a.C_stride[2];
    const int me = threadIdx.x - C::NS;
    struct Inputs {
      Pack<T, 8> u[R::EACH], dt[R::EACH], dy[R::EACH], z[R::EACH];
    };
    auto fetch = [&](Inputs& x, int t0, bool all) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        fetch8(x.u[k], u, a.u_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
        if (all) fetch8(x.dt[k], dt, a.dt_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
        if (all || gated) fetch8(x.dy[k], dy, (long long)a.M, t0 + tok, at.t1, c, at.valid, p.wide);
        if (gated) fetch8(x.z[k], z, a.z_stride[1], t0 + tok, at.t1, c, at.valid, p.wide);
      }
    };
    Inputs ahead, behind;      // of the tile that is prepared next, of the one that is finished next
    Shared<T, C, 3> bc;
    auto prepare = [&](int t0, int buf) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c)) continue;
        float d[8], g[8], slope[8], x[8];
        read8(d, sm.bias + c);
        to_floats(x, ahead.dt[k]);
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] += x[e];
        steps_of<true>(d, slope, a.softplus);
        to_floats(g, ahead.dy[k]);
        if (gated) {
          to_floats(x, ahead.z[k]);
#pragma unroll
          for (int e = 0; e < 8; e++) g[e] *= x[e] * sigmoid_fast(x[e]);
        }
        to_floats(x, ahead.u[k]);
        const int real = t0 + tok < at.t1 ? at.valid - c : 0;
#pragma unroll
        for (int e = 0; e < 8; e++)
          sm.x[buf][BwdShared<C>::place(tok, c + e)] =
              e < real ? make_float4(d[e], d[e] * x[e], g[e], slope[e]) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      bc.publish(sm.B[buf], sm.Cm[buf]);
    };
    float sD[R::EACH][8] = {}, sbias[R::EACH][8] = {};   // sums over the tokens that this thread sees
    auto finish_tile = [&](int t0, int buf) {
#pragma unroll
      for (int k = 0; k < R::EACH; k++) {
        int tok, c;
        if (!R::mine(k, tok, c) || t0 + tok >= at.t1 || c >= at.valid) continue;
        Pack<T, 8> ou, od, oz;
        float drive[8], decay[8], uv[8], z8[8];
        const float* const Dv = sm.D + c;
        to_floats(uv, behind.u[k]);
        if (gated) {
          float y[8], dy8[8];
          read8(y, &sm.y[buf][tok * YS + c]);
          to_floats(z8, behind.z[k]);
          to_floats(dy8, behind.dy[k]);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float s = sigmoid_fast(z8[e]);
            z8[e] = dy8[e] * fmaf(Dv[e], uv[e], y[e]) * s * fmaf(z8[e], 1.f - s, 1.f);
          }
          from_floats(oz, z8);
        }
        read8(drive, &sm.drive[buf][tok * YS + c]);
        read8(decay, &sm.decay[buf][tok * YS + c]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float4 x = sm.x[buf][BwdShared<C>::place(tok, c + e)];   // as this thread left it
          const float dd = fmaf(uv[e], drive[e], LN2 * decay[e]) * x.w;
          drive[e] = fmaf(Dv[e], x.z, drive[e] * x.x);
          decay[e] = dd;
          sD[k][e] = fmaf(x.z, uv[e], sD[k][e]);     // (channels that do not exist are not read)
          sbias[k][e] += dd;
        }
        from_floats(ou, drive);
        from_floats(od, decay);
        const long long to = ((long long)at.b * a.T + t0 + tok) * a.M + at.m0 + c;
        store_some<T, 8>(static_cast<T*>(a.du) + to, ou, at.valid - c, p.wide);
        store_some<T, 8>(static_cast<T*>(a.ddt) + to, od, at.valid - c, p.wide);
        if (gated) store_some<T, 8>(static_cast<T*>(a.dz) + to, oz, at.valid - c, p.wide);
      }
      // the warps' sums over their channels, a place of the row after the other
      constexpr int SPAN = C::NH < 2 * NP ? C::NH : 2 * NP, EVERY = C::NH / SPAN;   // a group of SPAN threads takes every EVERY-th token
#pragma unroll
      for (int v = me % SPAN; v < 2 * NP; v += SPAN) {
        const int n = v % NP;
        if (n >= a.N) continue;
        float* to = p.part_bc + ((((long long)at.cb * a.B + at.b) * a.T + t0) * a.G + at.g) * 2 * a.N + v / NP * a.N + n;
        const int row = a.G * 2 * a.N;
#pragma unroll 4
        for (int tok = me / SPAN; tok < TT; tok += EVERY) {
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < C::WARPS; w++) sum += sm.bc[buf][w][tok][v];
          if (t0 + tok < at.t1) to[(long long)tok * row] = sum;
        }
      }
    };
    for (int c = me; c < CH; c += C::NH) {
      sm.bias[c] = a.dt_bias != nullptr && c < at.valid ? a.dt_bias[at.m0 + c] : 0.f;
      sm.D[c] = a.D != nullptr && c < at.valid ? a.D[at.m0 + c] : 0.f;
    }
    __syncthreads();
    // What a step reads has been asked for a step before.
    {
      const int t0 = at.t0 + (tiles - 1) * TT;
      fetch(ahead, t0, true);
      bc.fetch(p, Bm, Cm, t0, at.t1);
      prepare(t0, (tiles - 1) & 1);
      behind = ahead;
      if (tiles > 1) {
        fetch(ahead, t0 - TT, true);
        bc.fetch(p, Bm, Cm, t0 - TT, at.t1);
      }
    }
    __syncthreads();
    for (int tile = tiles - 1; tile >= 0; tile--) {
      const int t0 = at.t0 + tile * TT;
      if (tile + 1 < tiles) {      // before the operands of the next tile take the place of its own: a thread reads what it wrote
        finish_tile(t0 + TT, (tile + 1) & 1);
        fetch(behind, t0, false);
      }
      if (tile > 0) prepare(t0 - TT, (tile - 1) & 1);
      if (tile > 1) {
        fetch(ahead, t0 - 2 * TT, true);
        bc.fetch(p, Bm, Cm, t0 - 2 * TT, at.t1);
      }
      __syncthreads();
    }
    finish_tile(at.t0, 0);
    // over the tokens of a tile, in the room of the operands of the tile behind, which nothing reads any more
    float *const all_D = reinterpret_cast<float*>(sm.x[1]), *const all_bias = all_D + TT * CH;
#pragma unroll
    for (int k = 0; k < R::EACH; k++) {
      int tok, c;
      if (!R::mine(k, tok, c)) continue;
      write8(all_D + tok * CH + c, sD[k]);
      write8(all_bias + tok * CH + c, sbias[k]);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(C::NH) : "memory");   // this group only
    for (int c = me; c < at.valid; c += C::NH) {
      float x = 0.f, y = 0.f;
#pragma unroll 4
      for (int k = 0; k < TT; k++) { x += all_D[k * CH + c]; y += all_bias[k * CH + c]; }
      part[(long long)a.M * a.N + at.m0 + c] = x;
      part[(long long)a.M * (a.N + 1) + at.m0 + c] = y;
    }
    return;
  }

  const int ch = threadIdx.x / L, sl = threadIdx.x % L, n0 = sl * S, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool ok = ch < at.valid;
  const long long m = at.m0 + ch;
  float A2[S], carry4[S] = {};
  load_states(A2, a.A + m * a.N, n0, a.N, ok, p.wide_state);
#pragma unroll
  for (int i = 0; i < S; i++) A2[i] *= LOG2E;
  join_backward(carry4, p, at, m, A2, n0, ok);
  // gh of the token behind and its decay, whose product flows to this one: kept apart, so that the chain over the tokens rounds
  // once per token, in one multiply-add
  F2 A2p[P], gh[P], step[P], dA[P], dA_lost[P];
#pragma unroll
  for (int i = 0; i < P; i++) {
    A2p[i] = pair(A2[2 * i], A2[2 * i + 1]);
    gh[i] = pair(carry4[2 * i], carry4[2 * i + 1]);
    step[i] = both(1.f);
    dA[i] = dA_lost[i] = both(0.f);
  }
  const int place = sum_place<C>(lane, n0);
  auto initial = [&](F2(&x)[P], int s) {
    load_pairs(x, a.initial_state + ((long long)s * a.M + m) * a.N, n0, a.N, ok && a.initial_state != nullptr, p.wide_state);
  };
  // The gradient that leaves a sequence's first token is its initial state's; the token before belongs to another one.
  auto leave = [&](int s) {
    if (a.dinitial_state != nullptr) {
      F2 out[P];
#pragma unroll
      for (int i = 0; i < P; i++) out[i] = mul2(step[i], gh[i]);
      store_pairs(a.dinitial_state + ((long long)s * a.M + m) * a.N, out, n0, a.N, ok, p.wide_state);
    }
    const bool has = a.dfinal_state != nullptr && a.cu_seqlens != nullptr && s > 0;
    load_pairs(gh, a.dfinal_state + (has ? ((long long)(s - 1) * a.M + m) * a.N : 0), n0, a.N, ok && has, p.wide_state);
#pragma unroll
    for (int i = 0; i < P; i++) step[i] = both(1.f);
  };
  const float* const kept = a.checkpoints + ((long long)at.b * ((a.T + CK - 1) / CK) * a.M + m) * a.N;
  F2 next[P];   // the state before the 16 tokens that come next
  load_pairs(next, kept + (long long)((at.t1 - 1) / CK) * a.M * a.N, n0, a.N, ok, p.wide_state);
  __syncthreads();
  __syncthreads();
  for (int tile = tiles - 1; tile >= 0; tile--) {
    const int t0 = at.t0 + tile * TT, buf = tile & 1;
    const float4* __restrict__ const sx = sm.x[buf];
    const float *__restrict__ const sB = sm.B[buf] + n0, *__restrict__ const sC = sm.Cm[buf] + n0;
    float *__restrict__ const to_drive = sm.drive[buf] + ch, *__restrict__ const to_decay = sm.decay[buf] + ch, *__restrict__ const to_y = sm.y[buf] + ch;
    float* __restrict__ const to_bc = &sm.bc[buf][warp][0][place];
#pragma unroll 1
    for (int sub = TT / CK - 1; sub >= 0; sub--) {
      const int k0 = sub * CK, ts = t0 + k0;
      if (ts >= at.t1) continue;
      // bit j: a sequence starts at token ts + j; s_low: the sequence of token ts
      unsigned starts = ts == 0 ? 1u : 0u;
      int s_low = at.b;
      if (a.cu_seqlens != nullptr) {
        Sequence q;
        q.at(a, at.b, ts);
        starts = q.begin == ts ? 1u : 0u;
        s_low = q.s;
        while (q.next < min(ts + CK, at.t1)) {
          q.advance(a);
          starts |= 1u << (q.begin - ts);
        }
      }
      F2 before[P], local[P];
#pragma unroll
      for (int i = 0; i < P; i++) {
        before[i] = next[i];
        local[i] = both(0.f);
      }
      if (ts > at.t0) load_pairs(next, kept + (long long)(ts / CK - 1) * a.M * a.N, n0, a.N, ok, p.wide_state);
      if (starts & 1u) initial(before, s_low);
      // inside: sequences begin behind the first of the 16 tokens
      auto walk = [&](auto inside) {
        F2 h[CK][P], x[P];
#pragma unroll
        for (int i = 0; i < P; i++) x[i] = before[i];
        int s = s_low;
#pragma unroll
        for (int j = 0; j < CK; j++) {
          if (inside.value && j > 0 && (starts >> j & 1u)) initial(x, ++s);
          const float2 v = *reinterpret_cast<const float2*>(sx + k0 * CH + BwdShared<C>::place(j, ch));
          const F2 d = both(v.x), w = both(v.y);
          F2 Bv[P];
          shared_pairs(Bv, sB + (k0 + j) * NP);
#pragma unroll
          for (int i = 0; i < P; i++) h[j][i] = x[i] = fma2(decay_of(d, A2p[i]), x[i], mul2(w, Bv[i]));
        }
#pragma unroll
        for (int j4 = CK - 4; j4 >= 0; j4 -= 4) {
          float sums[3][4], v[2][2 * S];   // drive, decay, y of four tokens; dB and dC of this channel of two
#pragma unroll
          for (int jj = 3; jj >= 0; jj--) {
            const int j = j4 + jj;
            const float4 xv = sx[k0 * CH + BwdShared<C>::place(j, ch)];
            const F2 d = both(xv.x), w = both(xv.y), g = both(xv.z);
            F2 Bv[P], Cv[P], old[P];
            shared_pairs(Bv, sB + (k0 + j) * NP);
            shared_pairs(Cv, sC + (k0 + j) * NP);
#pragma unroll
            for (int i = 0; i < P; i++) old[i] = j == 0 ? before[i] : h[j > 0 ? j - 1 : 0][i];
            const bool first = inside.value && j > 0 && (starts >> j & 1u);
            if (first) initial(old, s);
            F2 dr, de, yy;
#pragma unroll
            for (int i = 0; i < P; i++) {
              gh[i] = fma2(step[i], gh[i], mul2(Cv[i], g));
              step[i] = decay_of(d, A2p[i]);
              const F2 qv = mul2(mul2(step[i], gh[i]), old[i]);
              dr = i ? fma2(gh[i], Bv[i], dr) : mul2(gh[i], Bv[i]);
              de = i ? fma2(qv, A2p[i], de) : mul2(qv, A2p[i]);
              yy = i ? fma2(Cv[i], h[j][i], yy) : mul2(Cv[i], h[j][i]);
              local[i] = fma2(qv, d, local[i]);
              const float2 vb = halves(mul2(gh[i], w)), vc = halves(mul2(g, h[j][i]));
              v[jj & 1][2 * i] = vb.x; v[jj & 1][2 * i + 1] = vb.y; v[jj & 1][S + 2 * i] = vc.x; v[jj & 1][S + 2 * i + 1] = vc.y;
            }
            sums[0][jj] = sum_halves(dr); sums[1][jj] = sum_halves(de); sums[2][jj] = sum_halves(yy);
            if (first) leave(s--);
            if (jj % 2 == 0) sum_channels<C>(v, lane, [&](int odd, int i, float e) { to_bc[(k0 + j + odd) * 2 * NP + i] = e; });
          }
          sum_states<L>(sums, sl);
          put_sums<L>(to_drive + (k0 + j4) * YS, YS, sums[0], sl);
          put_sums<L>(to_decay + (k0 + j4) * YS, YS, sums[1], sl);
          if (gated) put_sums<L>(to_y + (k0 + j4) * YS, YS, sums[2], sl);
        }
      };
      if (starts >> 1) walk(std::true_type());
      else walk(std::false_type());
      if (starts & 1u) leave(s_low);
      // dA over thousands of tokens: sums of 16, joined with what each addition rounds off
#pragma unroll
      for (int i = 0; i < P; i++) {
        const F2 add = add2(local[i], dA_lost[i]), sum = add2(dA[i], add);
        dA_lost[i] = add2(add, neg2(add2(sum, neg2(dA[i]))));
        dA[i] = sum;
      }
    }
    __syncthreads();
  }
  store_pairs(part + m * a.N, dA, n0, a.N, ok, false);
}

// dB, dC [B*T][G][N] from the CTAs' sums [blocks][B*T][G][2][N], E neighbouring states per thread
template <class T, int E>
__global__ void __launch_bounds__(256) scan_sum_bc_kernel(const float* __restrict__ part, int blocks, long long rows, int N, T* __restrict__ dB, T* __restrict__ dC) {
  const long long n = rows * 2 * N, i = ((long long)blockIdx.x * 256 + threadIdx.x) * E;
  if (i >= n) return;
  float sum[E] = {};
#pragma unroll 8
  for (int k = 0; k < blocks; k++) {
    Pack<float, E> x;
    load_pack<float, E>(x, part + k * n + i);
#pragma unroll
    for (int e = 0; e < E; e++) sum[e] += x.v[e];
  }
  const long long row = i / (2 * N);
  const int v = (int)(i - row * 2 * N);
  T* to = v < N ? dB + row * N + v : dC + row * N + v - N;
#pragma unroll
  for (int e = 0; e < E; e++) to[e] = from_f32<T>(sum[e]);
}
// dA [M,N], dD and ddt_bias [M] from the sums [parts][M N + 2 M]
__global__ void __launch_bounds__(256) scan_sum_m_kernel(const float* __restrict__ part, int parts, long long MN, int M, float* dA, float* dD, float* dbias) {
  const long long n = MN + 2 * M, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
#pragma unroll 4
  for (int k = 0; k < parts; k++) sum += part[k * n + i];
  float* to = i < MN ? dA + i : i < MN + M ? (dD != nullptr ? dD + (i - MN) : nullptr) : (dbias != nullptr ? dbias + (i - MN - M) : nullptr);
  if (to != nullptr) *to = sum;
}

// One token per row: a channel's states over L lanes as above, two channels per thread.
template <class T, int L>
__global__ void __launch_bounds__(128) scan_step_kernel(const __grid_constant__ RewyScanStepArgs a, int blocks, bool wide, bool wide_bc) {
  constexpr int S = 4, CH = 128 / L, U = 2;
  const int b = blockIdx.x / blocks, sl = threadIdx.x % L, n0 = sl * S;
  const long long first = (long long)(blockIdx.x % blocks) * CH * U + threadIdx.x / L;
  const long long slot = pool_row(a.slots, a.slots_i64, b, a.pool);
  float A2[U][S], u[U], d[U], z[U], D[U], h[U][S], out[U];
  Pack<T, S> Bv[U], Cv[U];
#pragma unroll
  for (int i = 0; i < U; i++) {
    const long long m = first + i * CH;
    const bool ok = m < a.M;
    const int g = ok && a.G > 1 ? (int)m / (a.M / a.G) : 0;
    load_states(A2[i], a.A + m * a.N, n0, a.N, ok, wide);
    load_some<T, S>(Bv[i], static_cast<const T*>(a.Bm) + b * a.B_stride[0] + g * a.B_stride[1] + n0, ok ? a.N - n0 : 0, wide_bc);
    load_some<T, S>(Cv[i], static_cast<const T*>(a.C) + b * a.C_stride[0] + g * a.C_stride[1] + n0, ok ? a.N - n0 : 0, wide_bc);
    u[i] = ok ? to_f32(static_cast<const T*>(a.u)[b * a.u_stride + m]) : 0.f;
    d[i] = ok ? to_f32(static_cast<const T*>(a.dt)[b * a.dt_stride + m]) + (a.dt_bias != nullptr ? a.dt_bias[m] : 0.f) : 0.f;
    z[i] = ok && a.z != nullptr ? to_f32(static_cast<const T*>(a.z)[b * a.z_stride + m]) : 0.f;
    D[i] = ok && a.D != nullptr ? a.D[m] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < U; i++) load_states(h[i], a.state + (slot * a.M + first + i * CH) * a.N, n0, a.N, slot >= 0 && first + i * CH < a.M, wide);
  T* y = static_cast<T*>(a.y) + (long long)b * a.M;
  if (row_repeats(a.slots, a.slots_i64, b, slot) || slot < 0) {
#pragma unroll
    for (int i = 0; i < U; i++)
      if (first + i * CH < a.M && sl == 0) y[first + i * CH] = from_f32<T>(0.f);
    return;
  }
#pragma unroll
  for (int i = 0; i < U; i++) {
    float sig;
    if (a.softplus) d[i] = softplus_fast(d[i], sig);
    out[i] = 0.f;
#pragma unroll
    for (int k = 0; k < S; k++) {
      h[i][k] = fmaf(decay_of(d[i], A2[i][k] * LOG2E), h[i][k], d[i] * u[i] * to_f32(Bv[i].v[k]));
      out[i] = fmaf(to_f32(Cv[i].v[k]), h[i][k], out[i]);
    }
    store_states(a.state + (slot * a.M + first + i * CH) * a.N, h[i], n0, a.N, first + i * CH < a.M, wide);
  }
#pragma unroll
  for (int k = L / 2; k > 0; k >>= 1)
#pragma unroll
    for (int i = 0; i < U; i++) out[i] += __shfl_xor_sync(0xffffffffu, out[i], k);
#pragma unroll
  for (int i = 0; i < U; i++) {
    out[i] = fmaf(D[i], u[i], out[i]);
    if (a.z != nullptr) out[i] *= z[i] * sigmoid_fast(z[i]);
    if (first + i * CH < a.M && sl == 0) y[first + i * CH] = from_f32<T>(out[i]);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------

// f(Shape()) for N states
template <class F>
void with_shape(int N, F&& f) {
  if (N <= 8) f(Shape<4, 2, 128, 128, 32>());
  else if (N <= 16) f(Shape<4, 4, 128, 128, 32>());
  else if (N <= 32) f(Shape<8, 4, 128, 128, 32>());
  else f(Shape<16, 4, 128, 128, 32>());
}
// The forward keeps no 16 tokens of states in registers, so that eight of them fit a thread, with half the threads for the same
// channels.  Eight / four per thread, B=2 T=4096 M=4096 without checkpoints: N = 16 273 / 298 us, N = 32 669 / 680, N = 64 1745 /
// 1699; 4000 tokens of 512 channels: N = 32 61 / 63, N = 64 152 / 124.  Taken where it gains most.
template <class F>
void with_forward_shape(int N, F&& f) {
  if (N > 8 && N <= 16) f(Shape<2, 8, 64, 128, 32>());
  else with_shape(N, f);
}
int channels_of(int N) { return N <= 16 ? 32 : N <= 32 ? 16 : 8; }   // per CTA, as above
template <class F>
void with_step_lanes(int N, F&& f) {
  if (N <= 8) f(std::integral_constant<int, 2>());
  else if (N <= 16) f(std::integral_constant<int, 4>());
  else if (N <= 32) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

struct Plan {
  int blocks, segments, seg_len;
  long long ctas;                                     // per segment
  size_t seg_state, seg_dt, bc, m;                    // floats
};
Plan make_plan(int B, int T, int M, int N, int G, bool backward) {
  Plan p{};
  const int CH = channels_of(N), Mg = M / G;
  p.blocks = (Mg + CH - 1) / CH;
  p.ctas = (long long)p.blocks * G * B;
  const int tiles = (T + TILE - 1) / TILE;
  // Two CTAs fit an SM (one in the backward with N above 16, where the same counts still measure best: 512 channels, 4000 tokens,
  // forward and backward, 4 / 9 / 13 segments: N = 32 343 / 284 / 316 us, N = 64 690 / 636 / 670).  Segments cost a first pass (0.6 of
  // the forward, 0.25 of the backward), and a CTA alone on its SM is 1.5 times as fast as one beside another: fewer than three
  // segments do not pay.  As many as fill the GPU once, or twice where that leaves fewer tokens to each place (forward: 64 CTAs,
  // 16001 tokens of 2048 channels, 4 / 9 / 13 segments 451 / 408 / 427 us; 32 CTAs, 2000 tokens of 1024 channels, 6 / 9 / 13 46 / 34 /
  // 48; 16 CTAs, 16000 tokens of 512 channels, 13 / 18 / 26 147 / 113 / 159).
  const long long once = 2 * 148 / p.ctas, twice = 4 * 148 / p.ctas;
  long long want = 2 * once < 0.95 * twice ? twice : once;
  if (once < 3) want = 1;
  if (want > tiles / 4) want = tiles / 4;
  if (want < 3) want = 1;
  const int tiles_per = (int)((tiles + want - 1) / want);
  p.seg_len = tiles_per * TILE;
  p.segments = (T + p.seg_len - 1) / p.seg_len;
  const size_t rows = (size_t)B * p.segments * M;
  p.seg_state = p.segments > 1 ? rows * N : 0;
  p.seg_dt = p.segments > 1 ? rows : 0;
  if (backward) {
    p.bc = (size_t)p.blocks * B * T * G * 2 * N;
    p.m = (size_t)B * p.segments * M * (N + 2);
  }
  auto up = [](size_t x) { return (x + 63) & ~size_t(63); };
  p.seg_state = up(p.seg_state); p.seg_dt = up(p.seg_dt); p.bc = up(p.bc); p.m = up(p.m);
  return p;
}

// What 32-bit counts of tokens and channels hold
bool scan_fits(int B, int T, int M) { return (long long)B * T <= (1LL << 30) && M <= (1 << 24); }

int check_scan(const RewyScanArgs* a, bool backward, Plan& plan) {
  LAYER_REQUIRE(a != nullptr, REWY_ERR_NULL, "args is NULL");
  LAYER_REQUIRE(known_dtype(a->dtype), REWY_ERR_UNSUPPORTED, "unknown element type");
  LAYER_REQUIRE(a->B > 0 && a->T > 0 && a->M > 0 && a->G > 0, REWY_ERR_SHAPE, "B, T, M and G must be positive");
  LAYER_REQUIRE(a->N >= 1 && a->N <= 64, REWY_ERR_UNSUPPORTED, "the scan takes 1 to 64 states per channel");
  LAYER_REQUIRE(a->M % a->G == 0, REWY_ERR_SHAPE, "the channels must divide into the groups of B and C");
  LAYER_REQUIRE(scan_fits(a->B, a->T, a->M), REWY_ERR_SHAPE, "B*T exceeds 2^30 tokens or M 2^24 channels");
  LAYER_REQUIRE(a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->C != nullptr && a->A != nullptr, REWY_ERR_NULL, "u, dt, B, C or A is NULL");
  LAYER_REQUIRE(a->cu_seqlens == nullptr || (a->B == 1 && a->num_seqs > 0), REWY_ERR_SHAPE, "packed sequences need B = 1 and num_seqs > 0");
  plan = make_plan(a->B, a->T, a->M, a->N, a->G, backward);
  LAYER_REQUIRE(plan.ctas * plan.segments < (1LL << 31), REWY_ERR_SHAPE, "more rows and channels than one grid holds");
  const size_t need = (plan.seg_state + plan.seg_dt + plan.bc + plan.m) * sizeof(float);
  LAYER_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need), REWY_ERR_WORKSPACE, "the workspace of the scan is too small");
  return REWY_OK;
}

ScanParams scan_params(const RewyScanArgs& a, const Plan& plan) {
  ScanParams p{};
  p.a = a;
  p.Mg = a.M / a.G; p.blocks = plan.blocks; p.segments = plan.segments; p.seg_len = plan.seg_len;
  float* w = static_cast<float*>(a.workspace);
  p.seg_state = w; w += plan.seg_state;
  p.seg_dt = w; w += plan.seg_dt;
  p.part_bc = w; w += plan.bc;
  p.part_m = w;
  const int e = element_bytes(a.dtype), per16 = 16 / e;
  auto row = [&](const void* q) { return !unaligned16(q); };
  auto step = [&](int64_t s) { return s % per16 == 0; };
  p.wide = p.Mg % 8 == 0 && row(a.u) && row(a.dt) && row(a.z) && row(a.y) && row(a.dy) && row(a.du) && row(a.ddt) && row(a.dz);
  for (int i = 0; i < 2; i++) p.wide = p.wide && step(a.u_stride[i]) && step(a.dt_stride[i]) && (a.z == nullptr || step(a.z_stride[i]));
  p.wide_bc = a.N % 8 == 0 && row(a.Bm) && row(a.C);
  for (int i = 0; i < 3; i++) p.wide_bc = p.wide_bc && step(a.B_stride[i]) && step(a.C_stride[i]);
  p.wide_state = a.N % 4 == 0 && row(a.A) && row(a.initial_state) && row(a.final_state) && row(a.checkpoints) && row(a.dfinal_state) &&
                 row(a.dinitial_state) && row(a.workspace);
  return p;
}

}  // namespace
}  // namespace rewy

using namespace rewy;

extern "C" size_t rewy_scan_checkpoint_bytes(int32_t B, int32_t T, int32_t M, int32_t N) {
  if (B <= 0 || T <= 0 || M <= 0 || N <= 0 || N > 64 || !scan_fits(B, T, M)) return 0;
  return (size_t)B * ((T + CK - 1) / CK) * M * N * sizeof(float);
}

extern "C" size_t rewy_scan_workspace_bytes(int32_t B, int32_t T, int32_t M, int32_t N, int32_t G, int32_t backward) {
  if (B <= 0 || T <= 0 || M <= 0 || N <= 0 || N > 64 || G <= 0 || M % G || !scan_fits(B, T, M)) return 0;
  const Plan p = make_plan(B, T, M, N, G, backward != 0);
  return (p.seg_state + p.seg_dt + p.bc + p.m) * sizeof(float);
}

extern "C" int rewy_scan_fwd(const RewyScanArgs* a, rewy_stream_t st) {
  Plan plan;
  if (const int rc = check_scan(a, false, plan)) return rc;
  LAYER_REQUIRE(a->y != nullptr, REWY_ERR_NULL, "y is NULL");
  const ScanParams p = scan_params(*a, plan);
  const cudaStream_t s = (cudaStream_t)st;
  cudaError_t e = cudaSuccess;
  with_type(a->dtype, [&](auto t) {
    with_forward_shape(a->N, [&](auto c) {
      using T = decltype(t);
      using C = decltype(c);
      constexpr int bytes = sizeof(FwdShared<C>);
      if (plan.segments > 1) {
        e = ensure_dynamic_smem<scan_fwd_kernel<T, C, true>>(bytes);
        if (e == cudaSuccess) scan_fwd_kernel<T, C, true><<<(unsigned)(plan.ctas * (plan.segments - 1)), C::THREADS, bytes, s>>>(p);
      }
      if (e == cudaSuccess) e = ensure_dynamic_smem<scan_fwd_kernel<T, C, false>>(bytes);
      if (e == cudaSuccess) scan_fwd_kernel<T, C, false><<<(unsigned)(plan.ctas * plan.segments), C::THREADS, bytes, s>>>(p);
    });
  });
  if (e != cudaSuccess) return report_error(REWY_ERR_LAUNCH, cudaGetErrorString(e));
  return launched("selective scan forward", plan.segments > 1 ? 2 : 1);
}

extern "C" int rewy_scan_bwd(const RewyScanArgs* a, rewy_stream_t st) {
  Plan plan;
  if (const int rc = check_scan(a, true, plan)) return rc;
  LAYER_REQUIRE(a->dy != nullptr && a->checkpoints != nullptr && a->du != nullptr && a->ddt != nullptr && a->dB != nullptr && a->dC != nullptr && a->dA != nullptr,
                REWY_ERR_NULL, "dy, checkpoints or a gradient is NULL");
  LAYER_REQUIRE((a->z == nullptr) == (a->dz == nullptr), REWY_ERR_NULL, "dz goes with z");
  const ScanParams p = scan_params(*a, plan);
  const cudaStream_t s = (cudaStream_t)st;
  cudaError_t e = cudaSuccess;
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    with_shape(a->N, [&](auto c) {
      using C = decltype(c);
      e = ensure_dynamic_smem<scan_bwd_kernel<T, C>>(sizeof(BwdShared<C>));
      if (e != cudaSuccess) return;
      if (plan.segments > 1) scan_bwd_state_kernel<T, C><<<(unsigned)(plan.ctas * (plan.segments - 1)), C::THREADS, 0, s>>>(p);
      scan_bwd_kernel<T, C><<<(unsigned)(plan.ctas * plan.segments), C::THREADS, sizeof(BwdShared<C>), s>>>(p);
    });
    if (e != cudaSuccess) return;
    const long long rows = (long long)a->B * a->T * a->G;
    const long long n = rows * 2 * a->N;
    if (a->N % 4 == 0 && !unaligned16(p.part_bc))
      scan_sum_bc_kernel<T, 4><<<(unsigned)((n / 4 + 255) / 256), 256, 0, s>>>(p.part_bc, plan.blocks, rows, a->N, static_cast<T*>(a->dB), static_cast<T*>(a->dC));
    else
      scan_sum_bc_kernel<T, 1><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p.part_bc, plan.blocks, rows, a->N, static_cast<T*>(a->dB), static_cast<T*>(a->dC));
  });
  if (e != cudaSuccess) return report_error(REWY_ERR_LAUNCH, cudaGetErrorString(e));
  const long long MN = (long long)a->M * a->N;
  scan_sum_m_kernel<<<(unsigned)((MN + 2 * a->M + 255) / 256), 256, 0, s>>>(p.part_m, a->B * plan.segments, MN, a->M, a->dA, a->dD, a->ddt_bias);
  return launched("selective scan backward", plan.segments > 1 ? 4 : 3);
}

extern "C" int rewy_scan_step(const RewyScanStepArgs* a, rewy_stream_t st) {
  LAYER_REQUIRE(a != nullptr, REWY_ERR_NULL, "args is NULL");
  LAYER_REQUIRE(known_dtype(a->dtype), REWY_ERR_UNSUPPORTED, "unknown element type");
  LAYER_REQUIRE(a->N >= 1 && a->N <= 64, REWY_ERR_UNSUPPORTED, "the scan takes 1 to 64 states per channel");
  LAYER_REQUIRE(a->B > 0 && a->M > 0 && a->G > 0 && a->pool > 0 && a->M % a->G == 0, REWY_ERR_SHAPE, "bad B, M, G or pool");
  LAYER_REQUIRE(a->slots != nullptr || a->pool >= a->B, REWY_ERR_SHAPE, "fewer states than rows");
  LAYER_REQUIRE(a->M <= (1 << 24) && (long long)a->B * (a->M / 8 + 1) < (1LL << 31), REWY_ERR_SHAPE, "more rows and channels than one grid holds");
  LAYER_REQUIRE(a->u != nullptr && a->dt != nullptr && a->Bm != nullptr && a->C != nullptr && a->A != nullptr && a->state != nullptr && a->y != nullptr,
                REWY_ERR_NULL, "a required pointer of the scan step is NULL");
  const bool wide = a->N % 4 == 0 && !unaligned16(a->state) && !unaligned16(a->A);
  bool wide_bc = a->N % 4 == 0 && !unaligned16(a->Bm) && !unaligned16(a->C);
  for (int i = 0; i < 2; i++) wide_bc = wide_bc && a->B_stride[i] % 4 == 0 && a->C_stride[i] % 4 == 0;
  with_type(a->dtype, [&](auto t) {
    with_step_lanes(a->N, [&](auto l) {
      const int per = 128 / l.value * 2, blocks = (a->M + per - 1) / per;
      scan_step_kernel<decltype(t), l.value><<<(unsigned)((long long)blocks * a->B), 128, 0, (cudaStream_t)st>>>(*a, blocks, wide, wide_bc);
    });
  });
  return launched("selective scan step");
}
