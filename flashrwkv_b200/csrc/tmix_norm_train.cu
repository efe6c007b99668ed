// Training form of the block-level LayerNorm and of add + LayerNorm, forward and backward, on bf16 rows.
//
//   s    = x + residual                       (rounded to bf16: the tensor the caller keeps; without residual s = x)
//   xhat = (s - mean) * rstd,  y = xhat * w + b            mean, biased variance and rstd of s in fp32, saved per row
//   backward, with h = dy * w:
//   ds   = rstd * (h - mean(h) - xhat * mean(h * xhat)) + dsum         (dsum: the gradient that reaches s directly)
//   dw   = sum over rows of dy * xhat,   db = sum over rows of dy
//
// A row belongs to a group of T threads with V 16-byte pieces each, which stays in registers from its one read to its
// one write: every tensor crosses HBM once, which is the bound of both passes (forward 2 or 4, backward 3 or 4 tensors
// of rows x C).  Groups of one warp need no barrier; small groups share a CTA of 256 threads (backward 512).  Forward: four pieces per
// thread (8192 x 4096 in 25 us; two pieces 33 us, for want of bytes under way; with residual 38 us, its bytes take 42 at
// the rate of a plain copy).  Backward: two pieces per thread; a CTA walks a slab of rows, keeps the column sums of dw and
// db in registers along the walk, requests the next row before it reduces the present one, does its arithmetic on fp32
// pairs (the pass is bound by instruction issue as much as by bytes) and writes one fp32 partial per CTA, one CTA per SM;
// sum_slabs_kernel adds the partials in a fixed order, so the parameter gradients are the same on every run.  8192 x 4096
// in 38 us, with a second gradient into the sum 49 us, where the bytes take 31 and 42, and 4 us for the slabs (two CTAs of
// half the threads per SM: 41, 49 and 7).  A ring of rows in shared memory in place of the row in registers was slower (56
// us): the bytes were not what it waited for.
//
// The reference has the inference forms only (flashrwkv2/tmix/normalization/__init__.py:31-90).

#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "frwkv_common.cuh"

namespace frwkv {
namespace {

using bf16 = __nv_bfloat16;
using IO = Io16<bf16>;

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  float2 t;
  t = IO::unpack(u.x); f[0] = t.x; f[1] = t.y;
  t = IO::unpack(u.y); f[2] = t.x; f[3] = t.y;
  t = IO::unpack(u.z); f[4] = t.x; f[5] = t.y;
  t = IO::unpack(u.w); f[6] = t.x; f[7] = t.y;
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(IO::pack(f[0], f[1]), IO::pack(f[2], f[3]), IO::pack(f[4], f[5]), IO::pack(f[6], f[7]));
}
__device__ __forceinline__ uint4 load16(const bf16* row, int piece) {
  return __ldg(reinterpret_cast<const uint4*>(row) + piece);
}

// Sums over the T threads of a row's group.  `scratch` holds two float2 per warp; `turn` alternates so that one barrier
// per call is enough (a slot is written again only after the barrier of the call in between).
template <int T, int kThreads>
__device__ __forceinline__ float2 group_sum(float2 v, float2* scratch, int turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (T == 32) return v;
  static_assert(T % 32 == 0, "a group is whole warps: its barrier counts them");
  constexpr int kWarps = T / 32, kAllWarps = kThreads / 32;
  static_assert(kThreads / T < 16 || T == 32, "a barrier per group, and barrier 0 is the CTA's");
  const int warp = threadIdx.x >> 5, group = threadIdx.x / T;
  float2* slot = scratch + turn * kAllWarps;
  if ((threadIdx.x & 31) == 0) slot[warp] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");  // the group's own barrier
  v = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const float2 p = slot[group * kWarps + i];
    v.x += p.x;
    v.y += p.y;
  }
  return v;
}

__host__ __device__ constexpr int forward_threads(int T) { return T < 256 ? 256 : T; }

template <int T, int V, bool kAdd>
__global__ __launch_bounds__(forward_threads(T)) void norm_forward_kernel(
    const bf16* __restrict__ x, const bf16* __restrict__ residual, const bf16* __restrict__ weight,
    const bf16* __restrict__ bias, bf16* __restrict__ sum_out, bf16* __restrict__ out, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, long long rows, int channels, float eps) {
  chain_begin();
  __shared__ float2 scratch[2 * (forward_threads(T) / 32)];
  constexpr int kGroups = forward_threads(T) / T;
  const int lane = threadIdx.x % T, pieces = channels >> 3;
  const long long row = (long long)blockIdx.x * kGroups + threadIdx.x / T;
  if (row >= rows) return;  // whole groups leave: the barriers are per group
  const long long at = row * channels;
  float f[V][8];
  float2 part = make_float2(0.f, 0.f);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int p = lane + v * T;
    uint4 u = make_uint4(0u, 0u, 0u, 0u), r = u;
    if (p < pieces) {
      u = load16(x + at, p);
      if (kAdd) r = load16(residual + at, p);
    }
    unpack8(u, f[v]);
    if (kAdd) {
      float g[8];
      unpack8(r, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] += f[v][e];
      u = pack8(g);
      if (p < pieces) reinterpret_cast<uint4*>(sum_out + at)[p] = u;
      unpack8(u, f[v]);  // the statistics are those of the rounded sum, the tensor the caller sees
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part.x += f[v][e];
  }
  const float inv = 1.f / (float)channels;
  const float mean = group_sum<T, forward_threads(T)>(part, scratch, 0).x * inv;
  part.x = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (lane + v * T < pieces) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[v][e] -= mean;
        part.x = fmaf(f[v][e], f[v][e], part.x);
      }
    }
  }
  const float rstd = rsqrtf(group_sum<T, forward_threads(T)>(part, scratch, 1).x * inv + eps);
  if (lane == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int p = lane + v * T;
    if (p < pieces) {
      float w[8], b[8];
      unpack8(load16(weight, p), w);
      unpack8(load16(bias, p), b);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = fmaf(f[v][e] * rstd, w[e], b[e]);
      reinterpret_cast<uint4*>(out + at)[p] = pack8(w);
    }
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------
// fp32 pairs: fma.rn.f32x2 and its kin do two elements per issue slot, each rounded as the scalar instruction rounds
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void unpack_pairs(const uint4& u, f32x2 (&f)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = IO::unpack(w[i]);
    f[i] = pair(t.x, t.y);
  }
}

__host__ __device__ constexpr int backward_threads(int T) { return T < 512 ? 512 : T; }

// One row of the backward pass as it comes from memory.
template <int V>
struct RowPieces {
  uint4 s[V], dy[V];
  float mean, rstd;
};

template <int T, int V>
__device__ __forceinline__ void load_row(RowPieces<V>& r, const bf16* s, const bf16* dy, const float* mean, const float* rstd, long long row, int channels, int lane) {
  const long long at = row * channels;
  const int pieces = channels >> 3;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int p = lane + v * T;
    r.s[v] = r.dy[v] = make_uint4(0u, 0u, 0u, 0u);
    if (p < pieces) {
      r.s[v] = load16(s + at, p);
      r.dy[v] = load16(dy + at, p);
    }
  }
  r.mean = __ldg(mean + row);
  r.rstd = __ldg(rstd + row);
}

// kSum: a gradient reaches s beside the one through the norm.  kParams: dw and db are wanted.
template <int T, int V, bool kSum, bool kParams>
__global__ __launch_bounds__(backward_threads(T), 1) void norm_backward_kernel(
    const bf16* __restrict__ dy, const bf16* __restrict__ dsum, const bf16* __restrict__ s,
    const bf16* __restrict__ weight, const float* __restrict__ mean, const float* __restrict__ rstd,
    bf16* __restrict__ dx, bf16* __restrict__ dw, bf16* __restrict__ db, float* __restrict__ partials, long long rows,
    int channels, long long rows_per_cta) {
  chain_begin();
  constexpr int kThreads = backward_threads(T), kAllWarps = kThreads / 32, kGroups = kThreads / T;
  __shared__ float2 scratch[2 * kAllWarps];
  const int lane = threadIdx.x % T, group = threadIdx.x / T, pieces = channels >> 3;
  const long long begin = blockIdx.x * rows_per_cta;
  const long long end = begin + rows_per_cta < rows ? begin + rows_per_cta : rows;
  const float inv = 1.f / (float)channels;
  f32x2 sw[V][4], sb[V][4];
  uint4 w[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    w[v] = lane + v * T < pieces ? load16(weight, lane + v * T) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) sw[v][i] = sb[v][i] = pair(0.f, 0.f);
  }
  RowPieces<V> now;
  long long row = begin + group;
  if (row < end) load_row<T, V>(now, s, dy, mean, rstd, row, channels, lane);
  for (int turn = 0; row < end; turn ^= 1) {
    const long long next_row = row + kGroups;
    RowPieces<V> next = now;
    if (next_row < end) load_row<T, V>(next, s, dy, mean, rstd, next_row, channels, lane);
    uint4 ds[V];  // wanted after the sums only: it needs no row of lead
    if (kSum) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (lane + v * T < pieces) ds[v] = load16(dsum + row * channels, lane + v * T);
    }
    f32x2 unit[V][4], hw[V][4], p1 = pair(0.f, 0.f), p2 = p1;
    const f32x2 scale = pair(now.rstd, now.rstd), shift = pair(-now.mean * now.rstd, -now.mean * now.rstd);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f32x2 c[4], h[4], g[4];
      unpack_pairs(now.s[v], c);
      unpack_pairs(now.dy[v], h);
      unpack_pairs(w[v], g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unit[v][i] = fma2(c[i], scale, shift);
        if (kParams) {
          sw[v][i] = fma2(h[i], unit[v][i], sw[v][i]);
          sb[v][i] = add2(sb[v][i], h[i]);
        }
        hw[v][i] = mul2(h[i], g[i]);
        p1 = add2(p1, hw[v][i]);
        p2 = fma2(hw[v][i], unit[v][i], p2);
      }
    }
    const float2 q1 = halves(p1), q2 = halves(p2);
    const float2 total = group_sum<T, kThreads>(make_float2(q1.x + q1.y, q2.x + q2.y), scratch, turn);
    // ds = rstd * hw - (rstd * mean(h)) - unit * (rstd * mean(h * xhat))
    const float m1 = -now.rstd * total.x * inv, m2 = -now.rstd * total.y * inv;
    const f32x2 n1 = pair(m1, m1), n2 = pair(m2, m2);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int p = lane + v * T;
      if (p < pieces) {
        f32x2 d[4];
        if (kSum) unpack_pairs(ds[v], d);
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x2 g = fma2(hw[v][i], scale, fma2(unit[v][i], n2, n1));
          if (kSum) g = add2(g, d[i]);
          const float2 t = halves(g);
          out[i] = IO::pack(t.x, t.y);
        }
        reinterpret_cast<uint4*>(dx + row * channels)[p] = make_uint4(out[0], out[1], out[2], out[3]);
      }
    }
    row = next_row;
    now = next;
  }
  if (!kParams) return;
  // the CTA's groups are added in their order, then one partial per CTA leaves (or, of a single CTA, the result)
  if (kGroups > 1) {
    __shared__ f32x2 sums[kGroups > 1 ? (kGroups - 1) * T * 8 : 1];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      __syncthreads();
      if (group > 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sums[((group - 1) * 8 + i) * T + lane] = sw[v][i];
          sums[((group - 1) * 8 + 4 + i) * T + lane] = sb[v][i];
        }
      }
      __syncthreads();
      if (group == 0) {
        for (int g = 0; g < kGroups - 1; ++g) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sw[v][i] = add2(sw[v][i], sums[(g * 8 + i) * T + lane]);
            sb[v][i] = add2(sb[v][i], sums[(g * 8 + 4 + i) * T + lane]);
          }
        }
      }
    }
  }
  if (group > 0) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int p = lane + v * T;
    if (p >= pieces) continue;
    uint32_t ow[4], ob[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = halves(sw[v][i]), b = halves(sb[v][i]);
      if (gridDim.x > 1) {
        float* q = partials + (long long)blockIdx.x * 2 * channels + 8 * p + 2 * i;
        *reinterpret_cast<float2*>(q) = a;
        *reinterpret_cast<float2*>(q + channels) = b;
      }
      ow[i] = IO::pack(a.x, a.y);
      ob[i] = IO::pack(b.x, b.y);
    }
    if (gridDim.x == 1) {
      reinterpret_cast<uint4*>(dw)[p] = make_uint4(ow[0], ow[1], ow[2], ow[3]);
      reinterpret_cast<uint4*>(db)[p] = make_uint4(ob[0], ob[1], ob[2], ob[3]);
    }
  }
}

// dw and db of rows too wide for one CTA's registers to hold the column sums beside the row (above 8192 channels): a pass of
// its own over s and dy (2048 x 16384: 89 us in all, 132 with sums that spill).  A warp takes 256 channels, a CTA's four warps a quarter of its slab each.
__global__ __launch_bounds__(128) void norm_columns_kernel(const bf16* __restrict__ dy, const bf16* __restrict__ s,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           float* __restrict__ partials, long long rows, int channels,
                                                           long long rows_per_cta) {
  chain_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, p = blockIdx.x * 32 + lane;
  const long long begin = blockIdx.y * rows_per_cta;
  const long long end = begin + rows_per_cta < rows ? begin + rows_per_cta : rows;
  const bool mine = p < (channels >> 3);
  f32x2 sw[4], sb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sw[i] = sb[i] = pair(0.f, 0.f);
  if (mine) {
#pragma unroll 4
    for (long long row = begin + warp; row < end; row += 4) {
      f32x2 c[4], h[4];
      unpack_pairs(load16(s + row * channels, p), c);
      unpack_pairs(load16(dy + row * channels, p), h);
      const float r = __ldg(rstd + row), m = -__ldg(mean + row) * r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sw[i] = fma2(h[i], fma2(c[i], pair(r, r), pair(m, m)), sw[i]);
        sb[i] = add2(sb[i], h[i]);
      }
    }
  }
  __shared__ f32x2 sums[3][8][32];
  if (warp > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[warp - 1][i][lane] = sw[i];
      sums[warp - 1][4 + i][lane] = sb[i];
    }
  }
  __syncthreads();
  if (warp > 0 || !mine) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      sw[i] = add2(sw[i], sums[j][i][lane]);
      sb[i] = add2(sb[i], sums[j][4 + i][lane]);
    }
    float* q = partials + (long long)blockIdx.y * 2 * channels + 8 * p + 2 * i;
    *reinterpret_cast<float2*>(q) = halves(sw[i]);
    *reinterpret_cast<float2*>(q + channels) = halves(sb[i]);
  }
}

// dw[c], db[c] = sum over the slabs of partials[slab][2][C].  A CTA takes 32 of the 2C columns; each of its sixteen warps
// walks every sixteenth slab with eight requests in flight, and the warps' sums are added in their order.
constexpr int kSumWarps = 16;
__global__ __launch_bounds__(kSumWarps * 32) void sum_slabs_kernel(const float* __restrict__ partials, bf16* __restrict__ dw,
                                                        bf16* __restrict__ db, int slabs, int channels) {
  chain_begin();
  __shared__ float sums[kSumWarps][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int column = blockIdx.x * 32 + lane, columns = 2 * channels;
  float acc = 0.f;
  if (column < columns) {
    for (int s = warp; s < slabs; s += kSumWarps * 8) {
      float v[8];  // the eight requests leave together: the row is clamped rather than the load skipped
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = s + j * kSumWarps;
        v[j] = __ldg(partials + (long long)(at < slabs ? at : s) * columns + column);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc += s + j * kSumWarps < slabs ? v[j] : 0.f;
    }
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || column >= columns) return;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kSumWarps; ++w) total += sums[w][lane];
  (column < channels ? dw[column] : db[column - channels]) = IO::store(total);
}

// ---- host side -----------------------------------------------------------------------------------------------------
constexpr int kMaxChannels = 512 * 4 * 8;
constexpr int kForwardPieces = 4, kBackwardPieces = 2;

constexpr int kKnownDevices = 64;  // what a device answered once is kept: the queries cost as much as a launch

int sm_count() {
  static std::atomic<int> known[kKnownDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < kKnownDevices && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  if (dev < kKnownDevices) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

struct NormPlan {
  int slabs;
  long long rows_per_cta;
};
// Slabs of at least four rows, and no more of them than one wave of CTAs: fewer slabs mean fewer partials.
NormPlan plan_backward(long long rows) {
  const long long most = sm_count();
  long long slabs = (rows + 3) / 4;
  if (slabs > most) slabs = most;
  const long long per = (rows + slabs - 1) / slabs;
  return {(int)((rows + per - 1) / per), per};
}

// Calls f with the group size and the pieces per thread that cover the channels; kMost pieces per thread at most.
template <int kMost, typename F>
int by_width(int channels, F&& f) {
  const int pieces = channels / 8;
  using std::integral_constant;
#define WIDTH(T, V) f(integral_constant<int, T>{}, integral_constant<int, V>{})
  if (pieces <= 32) return WIDTH(32, 1);
  if (pieces <= 64) return WIDTH(32, 2);
  if (pieces <= 128) return WIDTH(128 / kMost, kMost);
  if (pieces <= 256) return WIDTH(256 / kMost, kMost);
  if (pieces <= 512) return WIDTH(512 / kMost, kMost);
  if (pieces <= 1024) return WIDTH(1024 / kMost, kMost);
  return WIDTH(2048 / kMost, kMost);
#undef WIDTH
}

bool aligned16(std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  return true;
}

int check_sizes(const char* what, long long rows, int channels) {
  FRWKV_REQUIRE(rows > 0 && rows <= 0x7fffffffLL && channels > 0, "%s: sizes must be positive", what);
  FRWKV_REQUIRE(channels % 8 == 0 && channels <= kMaxChannels, "%s: channel count must be a multiple of 8 up to %d", what,
                kMaxChannels);
  return FRWKV_OK;
}

}  // namespace
}  // namespace frwkv

extern "C" int frwkv_pretrain_layer_norm_forward(const void* x, const void* residual, const void* weight,
                                                 const void* bias, void* sum_out, void* out, float* mean, float* rstd,
                                                 long long rows, int channels, float eps, frwkv_stream_t stream) {
  using namespace frwkv;
  clear_error();
  FRWKV_REQUIRE(x && weight && bias && out && mean && rstd, "pretrain_layer_norm: null pointer argument");
  FRWKV_REQUIRE((residual == nullptr) == (sum_out == nullptr), "pretrain_layer_norm: residual and sum_out go together");
  if (int rc = check_sizes("pretrain_layer_norm", rows, channels)) return rc;
  FRWKV_REQUIRE(eps > 0.f && eps - eps == 0.f, "pretrain_layer_norm: eps must be finite and positive");
  FRWKV_REQUIRE(aligned16({x, residual, weight, bias, sum_out, out}),
                "pretrain_layer_norm: tensors must be 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return by_width<kForwardPieces>(channels, [&](auto t, auto v) {
    constexpr int T = decltype(t)::value, V = decltype(v)::value, kGroups = forward_threads(T) / T;
    const dim3 grid((unsigned)((rows + kGroups - 1) / kGroups)), block(forward_threads(T));
    const auto kernel = residual != nullptr ? norm_forward_kernel<T, V, true> : norm_forward_kernel<T, V, false>;
    launch_chained(kernel, grid, block, 0, s, static_cast<const bf16*>(x), static_cast<const bf16*>(residual),
                   static_cast<const bf16*>(weight), static_cast<const bf16*>(bias), static_cast<bf16*>(sum_out),
                   static_cast<bf16*>(out), mean, rstd, rows, channels, eps);
    return check_launch("norm_forward_kernel");
  });
}

extern "C" long long frwkv_pretrain_layer_norm_workspace_floats(long long rows, int channels) {
  if (rows <= 0 || channels <= 0) return 0;
  const long long slabs = frwkv::plan_backward(rows).slabs;
  return slabs * 2 * channels;
}

extern "C" int frwkv_pretrain_layer_norm_backward(const void* grad_out, const void* grad_sum, const void* sum,
                                                  const void* weight, const float* mean, const float* rstd,
                                                  void* grad_x, void* grad_weight, void* grad_bias, float* workspace,
                                                  long long workspace_floats, long long rows, int channels,
                                                  frwkv_stream_t stream) {
  using namespace frwkv;
  clear_error();
  FRWKV_REQUIRE(grad_out && sum && weight && mean && rstd && grad_x, "pretrain_layer_norm_backward: null pointer argument");
  FRWKV_REQUIRE((grad_weight == nullptr) == (grad_bias == nullptr),
                "pretrain_layer_norm_backward: grad_weight and grad_bias go together");
  FRWKV_REQUIRE(grad_weight == nullptr || workspace != nullptr, "pretrain_layer_norm_backward: null workspace");
  if (int rc = check_sizes("pretrain_layer_norm_backward", rows, channels)) return rc;
  FRWKV_REQUIRE(grad_weight == nullptr || workspace_floats >= frwkv_pretrain_layer_norm_workspace_floats(rows, channels),
                "pretrain_layer_norm_backward: workspace is smaller than frwkv_pretrain_layer_norm_workspace_floats");
  FRWKV_REQUIRE(aligned16({grad_out, grad_sum, sum, weight, grad_x, grad_weight, grad_bias, workspace}),
                "pretrain_layer_norm_backward: tensors must be 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return by_width<kBackwardPieces>(channels, [&](auto t, auto v) {
    constexpr int T = decltype(t)::value, V = decltype(v)::value;
    constexpr bool kApart = T > 512;  // the column sums take a pass of their own
    const bool parameters = grad_weight != nullptr;
    const NormPlan plan = plan_backward(rows);
    const auto run = [&](auto sum_known, auto params) {
      constexpr auto kernel = norm_backward_kernel<T, V, decltype(sum_known)::value, decltype(params)::value>;
      launch_chained(kernel, dim3(plan.slabs), dim3(backward_threads(T)), 0, s, static_cast<const bf16*>(grad_out),
                     static_cast<const bf16*>(grad_sum), static_cast<const bf16*>(sum), static_cast<const bf16*>(weight), mean,
                     rstd, static_cast<bf16*>(grad_x), static_cast<bf16*>(grad_weight), static_cast<bf16*>(grad_bias),
                     workspace, rows, channels, plan.rows_per_cta);
      return check_launch("norm_backward_kernel");
    };
    constexpr std::bool_constant<true> yes{};
    constexpr std::bool_constant<false> no{};
    constexpr std::bool_constant<!kApart> here{};
    const int launched = parameters ? (grad_sum != nullptr ? run(yes, here) : run(no, here))
                                    : (grad_sum != nullptr ? run(yes, no) : run(no, no));
    if (launched != FRWKV_OK) return launched;
    if (!parameters || (plan.slabs == 1 && !kApart)) return (int)FRWKV_OK;
    if (kApart) {
      launch_chained(norm_columns_kernel, dim3((channels + 255) / 256, plan.slabs), dim3(128), 0, s,
                     static_cast<const bf16*>(grad_out), static_cast<const bf16*>(sum), mean, rstd, workspace, rows, channels,
                     plan.rows_per_cta);
      if (int rc = check_launch("norm_columns_kernel")) return rc;
    }
    launch_chained(sum_slabs_kernel, dim3((2 * channels + 31) / 32), dim3(kSumWarps * 32), 0, s,
                   static_cast<const float*>(workspace),
                   static_cast<bf16*>(grad_weight), static_cast<bf16*>(grad_bias), plan.slabs, channels);
    return check_launch("sum_slabs_kernel");
  });
}
