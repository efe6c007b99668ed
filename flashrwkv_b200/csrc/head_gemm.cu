// The three matrix products of the head's losses on the 5th-generation tensor cores:
//
//   statistics    z = x W^T                 per 128 columns: row maximum and sum of exponentials (and the exponentials)
//   dx = g W                                contraction over the vocabulary
//   dW = g^T x                              contraction over the rows
//
// The last two share a launch: the units of dW fill what the last units of dx leave of the device (a step of 4096 x 8192 x 512
// 134 us in two launches, 125 in one; 33 x 8191 x 512 44 and 39).
// One persistent kernel, specialised by warp and run by pairs of CTAs (tcgen05, cta_group::2): a pair owns a 256 x 256
// output tile, each CTA loads its 128 rows of A and its half of B, so that a byte of shared memory feeds twice the
// arithmetic of a single CTA's 128 x 256 tile, which is bound by the fill of its shared memory.
//   warp 0      producer: TMA tiles of 64 contraction values into a ring of five stages; both CTAs' bytes are counted on
//               the leader's barrier
//   warp 1      (leader) MMA issuer: four tcgen05.mma per stage into one of two accumulators in tensor memory; commits
//               release the stage, and hand over the accumulator, in both CTAs
//   warps 2..9  epilogue of the other accumulator meanwhile: a warp takes 32 rows and 128 columns (of the statistics it adds
//               a wide contraction's parts first, kPartChannels)
// All three operand layouts are read where they lie: x and W are K-major in z = x W^T; W in g W, and both g and x in g^T x,
// are MN-major (the contraction index numbers the rows of the matrix in memory).  The number of rows that take part is known
// on the device only (labels may be missing), so the kernels read it there.
// 4096 x 32768 x 2048 (0.55 TFLOP each): statistics 346 us, both gradients 734 (370 and 339 where dx or dW alone is wanted),
// tensor pipe 92 to 97 % active at the 1.45 to 1.55 GHz that the power cap leaves; the library's plain products of these
// shapes take 357, 355 and 346 us.  With few rows the loads of W bound it: 16 x 65536 x 1024 in 33 to 37 us for the
// statistics and 66 for both gradients (134 MB read, twice, and 134 written).
// Every wait is bounded; a role whose wait runs out sets the error flag and leaves, the others run into their own limits,
// outputs that could not be made are NaN.

#include <atomic>

#include "head_loss.cuh"
#include "umma_pair.cuh"

namespace frwkv {
namespace head {
namespace {

using bf16 = __nv_bfloat16;
using IO = Io16<bf16>;

constexpr int kHalf = kTile / 2, kBK = 64;
constexpr uint32_t kOperandBytes = kHalf * kBK * 2;  // 16 KB: 128 rows of an operand in a stage
constexpr int kEpilogueWarps = 8;  // two per quarter of the tensor-memory lanes, half of the columns each
constexpr uint32_t kBoxBytes = 32 * 64 * 2;  // what an epilogue warp hands to TMA: 32 rows of 64 16-bit values
constexpr int kThreads = 64 + 32 * kEpilogueWarps;

// A pair's CTA loads 128 rows of A and 128 of B per stage; a CTA alone 128 of A and all 256 of B.
template <int kCtas>
struct Ring {
  static constexpr uint32_t kBBytes = kOperandBytes * 2 / kCtas, kStageBytes = kOperandBytes + kBBytes;
  static constexpr int kStages = kCtas == 2 ? 5 : 4;
  static constexpr uint32_t kSmem = kStages * kStageBytes + kEpilogueWarps * kBoxBytes + 1024;  // + slack to align the tiles
};
constexpr uint32_t kTmemCols = 2 * kTile;
// the parts of a unit's contraction that take an accumulator each
template <bool kGrads>
__device__ __forceinline__ int parts_of(int blocks) {
  constexpr int kMost = (kGrads ? kGradPart : kPartChannels) / kBK;
  return (blocks + kMost - 1) / kMost;
}

// One launch makes the statistics; another both gradients, whose units follow one another (the long ones of dx first).
struct Params {
  CUtensorMap map_a, map_b;            // of x and W, or of g and W for dx
  CUtensorMap map_a_weight, map_b_weight;  // gradients: of g and x for dW
  CUtensorMap map_compact;             // of x, where some rows take no part or all are copied
  CUtensorMap map_out;                 // the exponentials, or the bf16 dW
  Rows rows;
  int channels, vocab;
  float log2_scale;        // statistics
  const int* main_column;
  float2* stats;
  int stats_tiles;
  bool power;              // the exponentials are wanted
  Splits splits_x, splits_w;  // gradients
  bf16* grad_x;            // null: not wanted
  bf16* grad_weight;
  float* partials_x;
  float* partials_w;
  GradFactor factor;
  bool add;                // to what partials_w holds
};

struct Unit {
  bool of_weight;  // gradients: dW, not dx
  int m0, n0, split, kb_begin, kb_end;
  int width;  // columns of the tile, a multiple of 32: the last tile of a row may need fewer than 256
};

// the units of one product, from the number of rows that take part
template <int kCtas>
struct Part {
  static constexpr int kRows = kHalf * kCtas;
  int tiles_m, tiles_n, units, kb_total, splits, columns;
  __device__ void set(bool wanted, int m, int n, int k, int parts) {
    columns = n;
    tiles_m = (m + kRows - 1) / kRows;
    tiles_n = (n + kTile - 1) / kTile;
    kb_total = (k + kBK - 1) / kBK;
    splits = parts;
    units = wanted ? tiles_m * tiles_n * splits : 0;
  }
  // Pairs that run at the same time work on neighbouring tiles of the same part of the contraction, so that they share
  // their operands in L2.  Statistics: rows vary fastest (the whole x against a few tiles of W); the gradients: columns.
  __device__ Unit at(int unit, bool rows_first) const {
    Unit u;
    const int tiles = tiles_m * tiles_n;
    u.split = unit / tiles;
    const int t = unit - u.split * tiles;
    u.m0 = (rows_first ? t % tiles_m : t / tiles_n) * kRows;
    u.n0 = (rows_first ? t / tiles_m : t % tiles_n) * kTile;
    const int right = columns - u.n0;
    u.width = right < kTile ? (right + 31) & ~31 : kTile;
    u.kb_begin = (int)((long long)kb_total * u.split / splits);
    u.kb_end = (int)((long long)kb_total * (u.split + 1) / splits);
    u.of_weight = false;
    return u;
  }
};
template <bool kGrads, int kCtas>
struct Work {
  Part<kCtas> first, second;  // the statistics, or dx and dW
  int units;
  __device__ Work(const Params& p, int rows_here) {
    if (kGrads) {
      first.set(p.grad_x != nullptr, rows_here, p.channels, p.vocab, p.partials_x != nullptr ? *p.splits_x.chosen : 1);
      second.set(p.grad_weight != nullptr, p.vocab, p.channels, rows_here, p.partials_w != nullptr ? *p.splits_w.chosen : 1);
    } else {
      first.set(true, rows_here, p.vocab, p.channels, 1);
      second.units = 0;
    }
    units = first.units + second.units;
  }
  __device__ Unit at(int unit) const {
    if (!kGrads || unit < first.units) return first.at(unit, !kGrads);
    Unit u = second.at(unit - first.units, false);
    u.of_weight = true;
    return u;
  }
};

__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8], bool wide) {
  if (wide) {
    stg256(p, make_uint4(v[0], v[1], v[2], v[3]), make_uint4(v[4], v[5], v[6], v[7]));
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// 64 columns of a warp's 32 rows, packed to 16 bits, to shared memory as TMA reads it and from there to global memory in
// whole lines; the warp's box is free again once the store before has read it.
template <typename T>
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, uint32_t box, const float* z, int lane) {
  if (lane == 0) umma2::bulk_wait_read();
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = Io16<T>::pack(z[8 * i + 2 * j], z[8 * i + 2 * j + 1]);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + lane * 128 + ((i ^ (lane & 7)) << 4)), "r"(o[0]),
                 "r"(o[1]), "r"(o[2]), "r"(o[3])
                 : "memory");
  }
  umma::fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    umma2::tma_store_2d(map, x, y, box);
    umma2::bulk_commit();
  }
}

template <bool kGrads, int kCtas>
__device__ __forceinline__ void head_gemm(const Params& prm, int* error_flag) {
  using R = Ring<kCtas>;
  constexpr bool kPair = kCtas == 2;
  constexpr int kStages = R::kStages;
  constexpr uint32_t kStageBytes = R::kStageBytes;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_holder;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = kPair ? umma2::cluster_rank() : 0u;
  const uint32_t tiles_base = (umma::smem_u32(smem_raw) + 1023u) & ~1023u;

  chain_release();
  if (tid == 32) {  // the maps are parameters of this launch: fetched while the kernel before still runs
    umma2::prefetch_map(&prm.map_a);
    umma2::prefetch_map(&prm.map_b);
    if (kGrads) {
      umma2::prefetch_map(&prm.map_a_weight);
      umma2::prefetch_map(&prm.map_b_weight);
    }
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      umma::mbar_init(&full_bar[i], 1);   // the leader's producer; the bytes of both CTAs
      umma::mbar_init(&empty_bar[i], 1);  // a commit
    }
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(&acc_full[i], 1);   // a commit
      umma::mbar_init(&acc_empty[i], kCtas * kEpilogueWarps);  // those of both CTAs
    }
    umma::mbar_fence_init();
  }
  if (warp == 1) {
    if (kPair)
      umma2::tmem_alloc(&tmem_holder, kTmemCols);
    else
      umma::tmem_alloc(&tmem_holder, kTmemCols);
  }
  umma::fence_before_sync();
  __syncthreads();
  if (kPair) umma2::cluster_sync();
  umma::fence_after_sync();
  const uint32_t tmem = tmem_holder;
  chain_wait();

  const int count = *prm.rows.count;
  const int left = count - prm.rows.piece_begin;
  const int rows_here = left < 0 ? 0 : (left < prm.rows.piece_rows ? left : prm.rows.piece_rows);
  const bool compact = prm.rows.copied || count != prm.rows.total;
  const Work<kGrads, kCtas> work(prm, rows_here);
  const int pair = blockIdx.x / kCtas, pairs = gridDim.x / kCtas;  // "pair" is the CTA where it works alone
  bool ok = true;

  const auto wait = [](uint64_t* bar, uint32_t parity) {  // by a whole warp, one outcome for all of it
    return __all_sync(0xffffffffu, umma::mbar_wait(bar, parity)) != 0;
  };
  if (warp == 0) {
    uint32_t it = 0;
    for (int unit = pair; unit < work.units && ok; unit += pairs) {
      const Unit u = work.at(unit);
      const bool a_mn = kGrads && u.of_weight;
      const CUtensorMap* map_a = a_mn ? &prm.map_a_weight : (!kGrads && compact ? &prm.map_compact : &prm.map_a);
      const CUtensorMap* map_b = !a_mn ? &prm.map_b : (compact ? &prm.map_compact : &prm.map_b_weight);
      const int a_row = kGrads ? 0 : prm.rows.piece_begin, b_row = a_mn ? prm.rows.piece_begin : 0;
      const int m = u.m0 + (int)rank * kHalf, n = u.n0 + (int)rank * (u.width / kCtas);
      for (int kb = u.kb_begin; kb < u.kb_end; ++kb, ++it) {
        const uint32_t s = it % kStages, ph = (it / kStages) & 1u;
        if (!wait(&empty_bar[s], ph ^ 1u)) { ok = false; break; }
        const uint32_t full = kPair ? umma2::in_leader(&full_bar[s]) : umma::smem_u32(&full_bar[s]);
        const uint32_t a_dst = tiles_base + s * kStageBytes, b_dst = a_dst + kOperandBytes;
        const int k = kb * kBK;
        const auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
          if (kPair)
            umma2::tma_load_2d(dst, map, x, y, full);
          else
            umma2::tma_load_2d_alone(dst, map, x, y, full);
        };
        if (umma2::elect_one()) {
          if (rank == 0) umma::mbar_expect_tx(&full_bar[s], kCtas * kStageBytes);
          if (a_mn) {
            load(a_dst, map_a, m, k);
            load(a_dst + 8192, map_a, m + 64, k);
          } else {
            load(a_dst, map_a, k, a_row + m);
          }
          if (kGrads) {
#pragma unroll
            for (int j = 0; j < 4 / kCtas; ++j) load(b_dst + j * 8192, map_b, n + 64 * j, b_row + k);
          } else {
            load(b_dst, map_b, k, n);
          }
        }
        __syncwarp();
      }
    }
    // the last commits must have arrived here before this CTA may leave
    for (uint32_t i = 0; i < (uint32_t)kStages && i < it && ok; ++i) {
      const uint32_t j = it - 1 - i;
      if (!wait(&empty_bar[j % kStages], (j / kStages) & 1u)) ok = false;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t b_desc = kGrads ? umma2::desc_mn_major(tiles_base + kOperandBytes) : umma2::desc_k_major(tiles_base + kOperandBytes);
      constexpr uint32_t kBStep = (kGrads ? 2048 : 32) >> 4;  // 16 contraction values
      const auto commit = [](uint64_t* bar) {
        if (kPair)
          umma2::commit_both(bar);
        else
          umma::mma_commit(bar);
      };
      uint32_t it = 0, t = 0;
      for (int unit = pair; unit < work.units && ok; unit += pairs) {
        const Unit u = work.at(unit);
        if (u.kb_begin == u.kb_end) continue;  // nothing to contract: the epilogue writes zeros
        const bool a_mn = kGrads && u.of_weight;
        const uint32_t idesc = umma2::idesc_bf16(kHalf * kCtas, u.width, a_mn, kGrads);
        const uint64_t a_desc = a_mn ? umma2::desc_mn_major(tiles_base) : umma2::desc_k_major(tiles_base);
        const uint32_t a_step = (a_mn ? 2048 : 32) >> 4;
        const int blocks = u.kb_end - u.kb_begin, parts = parts_of<kGrads>(blocks);
        for (int part = 0; part < parts && ok; ++part) {
          const int begin = u.kb_begin + blocks * part / parts;
          const int end = u.kb_begin + blocks * (part + 1) / parts;
          const uint32_t acc = t & 1u, aph = (t >> 1) & 1u;
          ++t;
          if (!wait(&acc_empty[acc], aph ^ 1u)) { ok = false; break; }
          umma::fence_after_sync();
          const uint32_t d_tmem = tmem + acc * kTile;
          for (int kb = begin; kb < end; ++kb, ++it) {
            const uint32_t s = it % kStages, ph = (it / kStages) & 1u;
            if (!wait(&full_bar[s], ph)) { ok = false; break; }
            umma::fence_after_sync();
            const uint64_t a = a_desc + s * (kStageBytes >> 4), b = b_desc + s * (kStageBytes >> 4);
            if (umma2::elect_one()) {
#pragma unroll
              for (int ks = 0; ks < kBK / 16; ++ks) {
                const uint32_t add = (kb > begin || ks > 0) ? 1u : 0u;
                if (kPair)
                  umma2::mma_bf16(d_tmem, a + ks * a_step, b + ks * kBStep, idesc, add);
                else
                  umma2::mma_bf16_alone(d_tmem, a + ks * a_step, b + ks * kBStep, idesc, add);
              }
              commit(&empty_bar[s]);
            }
            __syncwarp();
          }
          if (ok && umma2::elect_one()) commit(&acc_full[acc]);
          __syncwarp();
        }
      }
    }
  } else {
    const uint32_t quarter = warp & 3u;  // the tensor-memory lanes this warp may read: 32 * (warp % 4) ..
    const int column0 = (warp - 2) / 4 * kStatsTile;
    const uint32_t source0 = tmem + ((32u * quarter) << 16) + column0;
    const int row_in_tile = (int)rank * kHalf + 32 * (int)quarter + lane;
    const uint32_t box = tiles_base + kStages * kStageBytes + (warp - 2) * kBoxBytes;
    uint32_t t = 0;
    float factor = 1.f;
    if (kGrads) {
      factor = prm.factor.temperature;
      if (prm.factor.mean) factor /= (float)count;
      if (prm.factor.scale != nullptr) factor *= *prm.factor.scale;
      if (prm.factor.of_rows != nullptr) factor *= *prm.factor.of_rows;
    }
    for (int unit = pair; unit < work.units; unit += pairs) {
      const Unit u = work.at(unit);
      const bool empty = u.kb_begin == u.kb_end;
      uint32_t acc = 0;
      const int m = u.m0 + row_in_tile, n = u.n0 + column0;
      const int m_end = u.of_weight ? prm.vocab : rows_here;
      int main = -1;  // statistics: where the row's label lies in this warp's columns
      if (!kGrads && m < m_end) main = prm.main_column[prm.rows.piece_begin + m] - n;
      // The next accumulator.  Warp-uniform outcome: the tensor-memory loads below need the whole warp.  Once a wait has run
      // out, this unit and all later ones read as NaN.
      const auto take = [&] {
        acc = t & 1u;
        const uint32_t aph = (t >> 1) & 1u;
        ++t;
        if (ok && !wait(&acc_full[acc], aph)) ok = false;
        umma::fence_after_sync();
        return source0 + acc * kTile;
      };
      // it goes back to the issuer as soon as its last columns are in registers
      const auto release = [&] {
        if (ok) {
          umma::fence_before_sync();
          __syncwarp();
          if (lane == 0)
            umma2::arrive_cluster(kPair ? umma2::in_leader(&acc_empty[acc]) : umma::smem_u32(&acc_empty[acc]));
        }
      };
      float z[kStatsTile];
      for (int part = 0, parts = parts_of<kGrads>(u.kb_end - u.kb_begin); part < parts; ++part) {
        const uint32_t source = take();
        if (!ok) break;
        if (part == 0) {
          uint32_t(&v)[kStatsTile / 32][32] = reinterpret_cast<uint32_t(&)[kStatsTile / 32][32]>(z);
#pragma unroll
          for (int i = 0; i < kStatsTile / 32; ++i) umma::tmem_ld32(source + 32 * i, v[i]);
          umma::tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < kStatsTile / 16; ++i) {
            uint32_t v[16];
            umma::tmem_ld16(source + 16 * i, v);
            umma::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              asm volatile("" : "+r"(v[j]));  // there after the wait only
              z[16 * i + j] += __uint_as_float(v[j]);
            }
          }
        }
        release();
      }
      if (empty || !ok) {
#pragma unroll
        for (int j = 0; j < kStatsTile; ++j) z[j] = ok ? 0.f : quiet_nan();
      } else if (kGrads) {
#pragma unroll
        for (int j = 0; j < kStatsTile; ++j) z[j] *= factor;
      }
      if (!kGrads) {
        const int valid = prm.vocab - n;  // columns inside the vocabulary, possibly none or more than there are here
        if (valid > 0) {
          if (valid < kStatsTile) {
#pragma unroll
            for (int j = 0; j < kStatsTile; ++j) z[j] = j < valid ? z[j] : -INFINITY;
          }
          if (__any_sync(0xffffffffu, main >= 0 && main < kStatsTile)) {
#pragma unroll
            for (int j = 0; j < kStatsTile; ++j) z[j] = j == main ? -INFINITY : z[j];
          }
          // a NaN gets past the maximum, but not past the sum
          float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < kStatsTile; ++j) high[j & 3] = fmaxf(high[j & 3], z[j]);
          const float most = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
          const float reference = most == -INFINITY ? 0.f : most * prm.log2_scale;  // nothing here: zeros, not inf - inf
#pragma unroll
          for (int j = 0; j < kStatsTile; ++j) {
            z[j] = ex2_approx(fmaf(z[j], prm.log2_scale, -reference));
            sum[j & 3] += z[j];
          }
          if (m < m_end)
            prm.stats[(long long)m * prm.stats_tiles + n / kStatsTile] =
                make_float2(most == -INFINITY ? -INFINITY : reference, (sum[0] + sum[1]) + (sum[2] + sum[3]));
          // rows of a box that take no part get what is there: nothing reads it
          if (prm.power && m - lane < m_end) {
            store_box<__half>(&prm.map_out, n, m - lane, box, z, lane);
            if (valid > 64) store_box<__half>(&prm.map_out, n + 64, m - lane, box, z + 64, lane);
          }
        }
      } else {
        const long long slot = (long long)u.split * m_end;
        float* const partials = u.of_weight ? prm.partials_w : prm.partials_x;
        const bool inside = m < m_end;
        const int row = !u.of_weight && inside && partials == nullptr ? prm.rows.row_map[prm.rows.piece_begin + m] : m;
        const bool wide = (prm.channels & 15) == 0 && (reinterpret_cast<uintptr_t>(prm.grad_x) & 31u) == 0;
#pragma unroll
        for (int c0 = 0; c0 < kStatsTile; c0 += 64) {
          float* const y = z + c0;
          if (partials != nullptr) {
            if (!inside) continue;
            float* dst = partials + (slot + m) * prm.channels + n + c0;
#pragma unroll
            for (int h = 0; h < 64; h += 8) {
              if (n + c0 + h < prm.channels) {  // channels are a multiple of 8
                if (u.of_weight && prm.add) {
                  const float4 a = *reinterpret_cast<const float4*>(dst + h), b = *reinterpret_cast<const float4*>(dst + h + 4);
                  y[h] += a.x; y[h + 1] += a.y; y[h + 2] += a.z; y[h + 3] += a.w;
                  y[h + 4] += b.x; y[h + 5] += b.y; y[h + 6] += b.z; y[h + 7] += b.w;
                }
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(y[h + j]);
                store32(dst + h, o, true);
              }
            }
          } else if (u.of_weight) {
            if (n + c0 < prm.channels && m - lane < m_end) store_box<bf16>(&prm.map_out, n + c0, m - lane, box, y, lane);
          } else if (inside) {
            bf16* dst = prm.grad_x + (long long)row * prm.channels + n + c0;
#pragma unroll
            for (int h = 0; h < 64; h += 16) {
              uint32_t o[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = IO::pack(y[h + 2 * j], y[h + 2 * j + 1]);
              const int room = prm.channels - (n + c0 + h);
              if (room >= 16) {
                store32(dst + h, o, wide);
              } else if (room >= 8) {
                *reinterpret_cast<uint4*>(dst + h) = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          }
        }
      }
    }
  }
  if (warp >= 2 && lane == 0) umma2::bulk_wait();  // this warp's stores, before the kernel may end
  if (!ok) {
    if (error_flag != nullptr) atomicExch(error_flag, kGrads ? 2 : 1);
    // give copies and MMAs that may still be in flight time to finish before the shared and tensor memory go away
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  __syncwarp();
  umma::fence_before_sync();
  __syncthreads();
  if (kPair) umma2::cluster_sync();
  if (warp == 1) {
    if (kPair)
      umma2::tmem_dealloc(tmem, kTmemCols);
    else
      umma::tmem_dealloc(tmem, kTmemCols);
  }
}

template <bool kGrads>
__global__ __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) void head_gemm_kernel(const __grid_constant__ Params prm,
                                                                                          int* error_flag) {
  head_gemm<kGrads, 2>(prm, error_flag);
}
template <bool kGrads>
__global__ __launch_bounds__(kThreads, 1) void head_gemm_alone_kernel(const __grid_constant__ Params prm, int* error_flag) {
  head_gemm<kGrads, 1>(prm, error_flag);
}

// ---- host side -----------------------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// [rows][columns] 16-bit values (copied as they are) with rows `stride` values apart, boxes of 64 columns x box_rows,
// 128-byte swizzle, zeros outside
bool make_map(CUtensorMap* map, const void* base, long long rows, long long columns, long long stride, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {64u, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  return encode_tiled() != nullptr &&
         encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long long tiles_of(long long n) { return (n + kTile - 1) / kTile; }

// `units`: at most so many
template <bool kGrads, int kCtas>
int launch(const Params& prm, long long units, int* error_flag, cudaStream_t stream) {
  constexpr auto kernel = kCtas == 2 ? head_gemm_kernel<kGrads> : head_gemm_alone_kernel<kGrads>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 64;
  if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Ring<kCtas>::kSmem);
    if (e != cudaSuccess) return fail(FRWKV_ERR_CUDA, "pretrain_head_loss: %s", cudaGetErrorString(e));
    if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  const int most = pair_count() * 2 / kCtas;
  const int grid = kCtas * (int)(units < most ? units : most);
  launch_chained(kernel, dim3(grid), dim3(kThreads), Ring<kCtas>::kSmem, stream, prm, error_flag);
  return check_launch("head_gemm_kernel");
}

int map_failure() { return fail(FRWKV_ERR_CUDA, "pretrain_head_loss: cuTensorMapEncodeTiled failed"); }

}  // namespace

int pair_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 74;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2) return 74;
  if (dev < 64) known[dev].store(n / 2, std::memory_order_relaxed);
  return n / 2;
}

int launch_logit_stats(const void* x, const void* x_compact, const void* weight, const Rows& rows, int channels, int vocab,
                       float log2_scale, const int* main_column, float2* stats, void* power, long long ldp,
                       int* error_flag,
                       cudaStream_t stream) {
  const bool few = one_cta(rows.piece_rows);
  Params prm{};
  prm.rows = rows;
  prm.channels = channels;
  prm.vocab = vocab;
  prm.log2_scale = log2_scale;
  prm.main_column = main_column;
  prm.stats = stats;
  prm.stats_tiles = (vocab + kStatsTile - 1) / kStatsTile;
  prm.power = power != nullptr;
  if (!make_map(&prm.map_a, x, rows.total, channels, channels, kHalf) ||
      !make_map(&prm.map_compact, x_compact, rows.total, channels, rows.ldx, kHalf) ||
      !make_map(&prm.map_b, weight, vocab, channels, channels, few ? kTile : kHalf) ||
      (power != nullptr && !make_map(&prm.map_out, power, rows.piece_rows, ldp, ldp, 32)))
    return map_failure();
  if (few) return launch<false, 1>(prm, tiles_of(vocab), error_flag, stream);
  return launch<false, 2>(prm, tiles_of(rows.piece_rows) * tiles_of(vocab), error_flag, stream);
}

int launch_gradients(const void* g, long long ldg, const void* x, const void* x_compact, const void* weight, const Rows& rows,
                     int channels, int vocab, const GradTarget& to_x, const GradTarget& to_weight, const GradFactor& factor,
                     bool add, int* error_flag, cudaStream_t stream) {
  Params prm{};
  prm.rows = rows;
  prm.channels = channels;
  prm.vocab = vocab;
  prm.splits_x = to_x.splits;
  prm.splits_w = to_weight.splits;
  prm.grad_x = static_cast<bf16*>(to_x.grad);
  prm.grad_weight = static_cast<bf16*>(to_weight.grad);
  prm.partials_x = to_x.partials;
  prm.partials_w = to_weight.partials;
  prm.factor = factor;
  prm.add = add;
  if (!make_map(&prm.map_a, g, rows.piece_rows, vocab, ldg, kHalf) ||
      !make_map(&prm.map_b, weight, vocab, channels, channels, kBK) ||
      !make_map(&prm.map_a_weight, g, rows.piece_rows, vocab, ldg, kBK) ||
      !make_map(&prm.map_b_weight, x, rows.total, channels, channels, kBK) ||
      !make_map(&prm.map_compact, x_compact, rows.total, channels, rows.ldx, kBK) ||
      (to_weight.grad != nullptr && to_weight.partials == nullptr &&
       !make_map(&prm.map_out, to_weight.grad, vocab, channels, channels, 32)))
    return map_failure();
  // at most so many units; a product with parts may be cut finer than the host knows and takes every pair
  const bool alone = one_cta(rows.piece_rows);
  const auto units = [&](const GradTarget& t, long long m) {
    const long long tiles = (alone ? (m + kHalf - 1) / kHalf : tiles_of(m)) * tiles_of(channels);
    return t.grad == nullptr ? 0 : (t.partials != nullptr ? tiles << 10 : tiles);
  };
  const long long most = units(to_x, rows.piece_rows) + units(to_weight, vocab);
  return alone ? launch<true, 1>(prm, most, error_flag, stream) : launch<true, 2>(prm, most, error_flag, stream);
}

}  // namespace head
}  // namespace frwkv
