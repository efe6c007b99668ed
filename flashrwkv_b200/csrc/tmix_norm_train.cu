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
// of rows x C).  A group is a warp up to 512 channels (no barrier at all), 2 to 16 warps above; small groups share a
// CTA of 256 threads.  The backward pass walks a slab of rows per CTA, keeps the column sums of dw and db in registers
// along the walk, requests the next row before it reduces the present one, and writes one fp32 partial per CTA;
// sum_slabs_kernel adds the partials in a fixed order, so the parameter gradients are the same on every run.
//
// The reference has the inference forms only (flashrwkv2/tmix/normalization/__init__.py:31-90).

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

__host__ __device__ constexpr int cta_threads(int T) { return T < 256 ? 256 : T; }

// Sums over the T threads of a row's group.  `scratch` holds two float2 per warp; `turn` alternates so that one barrier
// per call is enough (a slot is written again only after the barrier of the call in between).
template <int T>
__device__ __forceinline__ float2 group_sum(float2 v, float2* scratch, int turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (T == 32) return v;
  constexpr int kWarps = T / 32, kAllWarps = cta_threads(T) / 32;
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

template <int T, int V, bool kAdd>
__global__ __launch_bounds__(cta_threads(T)) void norm_forward_kernel(
    const bf16* __restrict__ x, const bf16* __restrict__ residual, const bf16* __restrict__ weight,
    const bf16* __restrict__ bias, bf16* __restrict__ sum_out, bf16* __restrict__ out, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, long long rows, int channels, float eps) {
  chain_begin();
  __shared__ float2 scratch[2 * (cta_threads(T) / 32)];
  constexpr int kGroups = cta_threads(T) / T;
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
  const float mean = group_sum<T>(part, scratch, 0).x * inv;
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
  const float rstd = rsqrtf(group_sum<T>(part, scratch, 1).x * inv + eps);
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

// One row of the backward pass as it comes from memory.
template <int V>
struct RowPieces {
  uint4 s[V], dy[V], ds[V];
  float mean, rstd;
};

template <int T, int V, bool kSum>
__device__ __forceinline__ void load_row(RowPieces<V>& r, const bf16* s, const bf16* dy, const bf16* dsum,
                                         const float* mean, const float* rstd, long long row, int channels, int lane) {
  const long long at = row * channels;
  const int pieces = channels >> 3;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int p = lane + v * T;
    r.s[v] = r.dy[v] = r.ds[v] = make_uint4(0u, 0u, 0u, 0u);
    if (p < pieces) {
      r.s[v] = load16(s + at, p);
      r.dy[v] = load16(dy + at, p);
      if (kSum) r.ds[v] = load16(dsum + at, p);
    }
  }
  r.mean = __ldg(mean + row);
  r.rstd = __ldg(rstd + row);
}

// kSum: a gradient reaches s beside the one through the norm.  kParams: dw and db are wanted.
template <int T, int V, bool kSum, bool kParams>
__global__ __launch_bounds__(cta_threads(T)) void norm_backward_kernel(
    const bf16* __restrict__ dy, const bf16* __restrict__ dsum, const bf16* __restrict__ s,
    const bf16* __restrict__ weight, const float* __restrict__ mean, const float* __restrict__ rstd,
    bf16* __restrict__ dx, bf16* __restrict__ dw, bf16* __restrict__ db, float* __restrict__ partials, long long rows,
    int channels, long long rows_per_cta) {
  chain_begin();
  constexpr int kAllWarps = cta_threads(T) / 32, kGroups = cta_threads(T) / T;
  constexpr bool kAhead = V <= 2;  // the next row's pieces fit the registers beside the column sums
  __shared__ float2 scratch[2 * kAllWarps];
  const int lane = threadIdx.x % T, group = threadIdx.x / T, pieces = channels >> 3;
  const long long begin = blockIdx.x * rows_per_cta;
  const long long end = begin + rows_per_cta < rows ? begin + rows_per_cta : rows;
  const float inv = 1.f / (float)channels;
  float aw[V][8], ab[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) aw[v][e] = ab[v][e] = 0.f;
  RowPieces<V> now;
  long long row = begin + group;
  if (row < end) load_row<T, V, kSum>(now, s, dy, dsum, mean, rstd, row, channels, lane);
  for (int turn = 0; row < end; turn ^= 1) {
    const long long next_row = row + kGroups;
    RowPieces<V> next = now;
    if (kAhead && next_row < end) load_row<T, V, kSum>(next, s, dy, dsum, mean, rstd, next_row, channels, lane);
    float2 part = make_float2(0.f, 0.f);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float h[8], w[8], c[8];
      unpack8(now.s[v], c);
      unpack8(now.dy[v], h);
      unpack8(lane + v * T < pieces ? load16(weight, lane + v * T) : make_uint4(0u, 0u, 0u, 0u), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float unit = (c[e] - now.mean) * now.rstd;
        if (kParams) {
          aw[v][e] = fmaf(h[e], unit, aw[v][e]);
          ab[v][e] += h[e];
        }
        const float hw = h[e] * w[e];
        part.x += hw;
        part.y = fmaf(hw, unit, part.y);
      }
    }
    const float2 total = group_sum<T>(part, scratch, turn);
    const float m1 = total.x * inv, m2 = total.y * inv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int p = lane + v * T;
      if (p < pieces) {
        float h[8], w[8], c[8], d[8];
        unpack8(now.s[v], c);
        unpack8(now.dy[v], h);
        unpack8(load16(weight, p), w);
        if (kSum) unpack8(now.ds[v], d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float unit = (c[e] - now.mean) * now.rstd;
          const float g = now.rstd * (h[e] * w[e] - m1 - unit * m2);
          c[e] = kSum ? g + d[e] : g;
        }
        reinterpret_cast<uint4*>(dx + row * channels)[p] = pack8(c);
      }
    }
    row = next_row;
    if (kAhead) {
      now = next;
    } else if (row < end) {
      load_row<T, V, kSum>(now, s, dy, dsum, mean, rstd, row, channels, lane);
    }
  }
  if (!kParams) return;
  // the CTA's groups are added in their order, then one partial per CTA leaves (or, of a single CTA, the result)
  if (kGroups > 1) {
    __shared__ float4 sums[kGroups > 1 ? (kGroups - 1) * T * 4 : 1];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      __syncthreads();
      if (group > 0) {
        float4* q = sums + (group - 1) * T * 4 + lane;
        q[0 * T] = make_float4(aw[v][0], aw[v][1], aw[v][2], aw[v][3]);
        q[1 * T] = make_float4(aw[v][4], aw[v][5], aw[v][6], aw[v][7]);
        q[2 * T] = make_float4(ab[v][0], ab[v][1], ab[v][2], ab[v][3]);
        q[3 * T] = make_float4(ab[v][4], ab[v][5], ab[v][6], ab[v][7]);
      }
      __syncthreads();
      if (group == 0) {
        for (int g = 0; g < kGroups - 1; ++g) {
          const float4* q = sums + g * T * 4 + lane;
          const float4 a = q[0 * T], b = q[1 * T], c = q[2 * T], d = q[3 * T];
          aw[v][0] += a.x; aw[v][1] += a.y; aw[v][2] += a.z; aw[v][3] += a.w;
          aw[v][4] += b.x; aw[v][5] += b.y; aw[v][6] += b.z; aw[v][7] += b.w;
          ab[v][0] += c.x; ab[v][1] += c.y; ab[v][2] += c.z; ab[v][3] += c.w;
          ab[v][4] += d.x; ab[v][5] += d.y; ab[v][6] += d.z; ab[v][7] += d.w;
        }
      }
    }
  }
  if (group > 0) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int p = lane + v * T;
    if (p >= pieces) continue;
    if (gridDim.x == 1) {
      reinterpret_cast<uint4*>(dw)[p] = pack8(aw[v]);
      reinterpret_cast<uint4*>(db)[p] = pack8(ab[v]);
    } else {
      float4* q = reinterpret_cast<float4*>(partials + (long long)blockIdx.x * 2 * channels) + 2 * p;
      q[0] = make_float4(aw[v][0], aw[v][1], aw[v][2], aw[v][3]);
      q[1] = make_float4(aw[v][4], aw[v][5], aw[v][6], aw[v][7]);
      q += channels / 4;
      q[0] = make_float4(ab[v][0], ab[v][1], ab[v][2], ab[v][3]);
      q[1] = make_float4(ab[v][4], ab[v][5], ab[v][6], ab[v][7]);
    }
  }
}

// dw[c], db[c] = sum over the slabs of partials[slab][2][C].  A CTA takes 32 of the 2C columns; each of its eight warps
// walks every eighth slab, and the warps' sums are added in their order.
__global__ __launch_bounds__(256) void sum_slabs_kernel(const float* __restrict__ partials, bf16* __restrict__ dw,
                                                        bf16* __restrict__ db, int slabs, int channels) {
  chain_begin();
  __shared__ float sums[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int column = blockIdx.x * 32 + lane, columns = 2 * channels;
  float a0 = 0.f, a1 = 0.f;
  if (column < columns) {
    int s = warp;
    for (; s + 8 < slabs; s += 16) {
      a0 += partials[(long long)s * columns + column];
      a1 += partials[(long long)(s + 8) * columns + column];
    }
    if (s < slabs) a0 += partials[(long long)s * columns + column];
  }
  sums[warp][lane] = a0 + a1;
  __syncthreads();
  if (warp != 0 || column >= columns) return;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) total += sums[w][lane];
  (column < channels ? dw[column] : db[column - channels]) = IO::store(total);
}

// ---- host side -----------------------------------------------------------------------------------------------------
constexpr int kMaxChannels = 512 * 4 * 8;
constexpr int kSlabsPerSm = 4;

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n > 0 ? n : 148;
}

struct NormPlan {
  int slabs;
  long long rows_per_cta;
};
// Slabs of at least four rows, and no more than `resident` CTAs per SM at once: fewer slabs mean fewer partials.
NormPlan plan_backward(long long rows, int resident) {
  const long long most = (long long)sm_count() * resident;
  long long slabs = (rows + 3) / 4;
  if (slabs > most) slabs = most;
  const long long per = (rows + slabs - 1) / slabs;
  return {(int)((rows + per - 1) / per), per};
}

// calls f with the group size and the pieces per thread that cover the channels
template <typename F>
int by_width(int channels, F&& f) {
  const int pieces = channels / 8;
  using std::integral_constant;
#define WIDTH(T, V) f(integral_constant<int, T>{}, integral_constant<int, V>{})
  if (pieces <= 32) return WIDTH(32, 1);
  if (pieces <= 64) return WIDTH(32, 2);
  if (pieces <= 128) return WIDTH(64, 2);
  if (pieces <= 256) return WIDTH(128, 2);
  if (pieces <= 512) return WIDTH(256, 2);
  if (pieces <= 1024) return WIDTH(512, 2);
  return WIDTH(512, 4);
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
  return by_width(channels, [&](auto t, auto v) {
    constexpr int T = decltype(t)::value, V = decltype(v)::value, kGroups = cta_threads(T) / T;
    const dim3 grid((unsigned)((rows + kGroups - 1) / kGroups)), block(cta_threads(T));
    const auto kernel = residual != nullptr ? norm_forward_kernel<T, V, true> : norm_forward_kernel<T, V, false>;
    launch_chained(kernel, grid, block, 0, s, static_cast<const bf16*>(x), static_cast<const bf16*>(residual),
                   static_cast<const bf16*>(weight), static_cast<const bf16*>(bias), static_cast<bf16*>(sum_out),
                   static_cast<bf16*>(out), mean, rstd, rows, channels, eps);
    return check_launch("norm_forward_kernel");
  });
}

extern "C" long long frwkv_pretrain_layer_norm_workspace_floats(long long rows, int channels) {
  if (rows <= 0 || channels <= 0) return 0;
  const long long slabs = frwkv::plan_backward(rows, frwkv::kSlabsPerSm).slabs;
  return slabs > 1 ? slabs * 2 * channels : 1;
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
  return by_width(channels, [&](auto t, auto v) {
    constexpr int T = decltype(t)::value, V = decltype(v)::value;
    const auto kernel = grad_weight != nullptr
                            ? (grad_sum != nullptr ? norm_backward_kernel<T, V, true, true> : norm_backward_kernel<T, V, false, true>)
                            : (grad_sum != nullptr ? norm_backward_kernel<T, V, true, false> : norm_backward_kernel<T, V, false, false>);
    int resident = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, cta_threads(T), 0) != cudaSuccess || resident < 1)
      return fail(FRWKV_ERR_CUDA, "pretrain_layer_norm_backward: %s", cudaGetErrorString(cudaGetLastError()));
    const NormPlan plan = plan_backward(rows, resident < kSlabsPerSm ? resident : kSlabsPerSm);
    launch_chained(kernel, dim3(plan.slabs), dim3(cta_threads(T)), 0, s, static_cast<const bf16*>(grad_out),
                   static_cast<const bf16*>(grad_sum), static_cast<const bf16*>(sum), static_cast<const bf16*>(weight), mean,
                   rstd, static_cast<bf16*>(grad_x), static_cast<bf16*>(grad_weight), static_cast<bf16*>(grad_bias),
                   workspace, rows, channels, plan.rows_per_cta);
    if (int rc = check_launch("norm_backward_kernel")) return rc;
    if (grad_weight == nullptr || plan.slabs == 1) return (int)FRWKV_OK;
    launch_chained(sum_slabs_kernel, dim3((2 * channels + 31) / 32), dim3(256), 0, s, static_cast<const float*>(workspace),
                   static_cast<bf16*>(grad_weight), static_cast<bf16*>(grad_bias), plan.slabs, channels);
    return check_launch("sum_slabs_kernel");
  });
}
