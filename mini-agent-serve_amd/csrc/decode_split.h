// decode_split.h - what the split-KV decode attentions share: the arguments, the choice of the splits on
// the host and of each row's on the device, the output's store, and the kernel that merges a row's splits.
#pragma once

#include <algorithm>

#include "device.h"

namespace mas {
namespace {

constexpr int kChunk = 256;          // positions per chunk
constexpr float kNegInf = -__builtin_huge_valf();

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_stride, q_head_stride;
  const uint16_t* k_cache;
  const uint16_t* v_cache;
  int64_t page_stride, entry_stride, head_stride, num_pages;
  const int32_t* block_tables;
  int64_t bt_stride, max_blocks;
  const int32_t* seq_lens;
  int hq, hk, group, log2_page, max_splits;
  int split_len;     // longest split: 64, 128, or a multiple of the 256-position chunk
  int row_target;    // small grids: splits wanted per row (the GPU's SIMDs over rows x kv heads)
  float scale_log2;  // bmm1_scale * log2(e)
  float out_scale;   // bmm2_scale
  float* part_o;     // [batch][hq][max_splits][D]
  float* part_ml;    // [batch][hq][max_splits][2]: running max (log2 domain), sum
  void* out;                // bf16, or fp8 e4m3fn codes when out_fp8
  int64_t out_stride, out_head_stride;
  int out_fp8;              // out = e4m3fn(clamp(bf16(O) / quant scale, +-448)): the o_proj input quantize
  const float* quant_scale_dev;
  float quant_scale_host;
  uint32_t* err;
};


// seq_lens[b] clamped to [0, max_blocks * page_size].
__device__ __forceinline__ int kv_len(const DecodeArgs& a, int b) {
  const int64_t L = a.seq_lens[b];
  const int64_t cap = a.max_blocks << a.log2_page;
  return static_cast<int>(L < 0 ? 0 : (L > cap ? cap : L));
}

// The split length of a row of L positions, chosen from the row's own length: 256 positions, or,
// in small grids (4+ splits wanted per row), 128 or 64 when the row's share L / row_target is that
// short; at most split_len, and at least the fewest 64-position units that keep the row within the
// grid's max_splits. The grid is sized from the block table's reach, which can far exceed the rows
// (a graph captured for the longest context): a row then still gets splits as short as its own
// length calls for.
__device__ __forceinline__ int row_split_len(const DecodeArgs& a, int L) {
  // large grids: the host's split for rows of 4+ such splits, 256 positions for shorter rows
  int len = L >= 4 * a.split_len ? a.split_len : 256;
  if (a.row_target >= 4) len = L <= 64 * a.row_target ? 64 : (L <= 128 * a.row_target ? 128 : 256);
  len = min(len, a.split_len);
  if (L > len * a.max_splits) len = 64 * (((L + 63) / 64 + a.max_splits - 1) / a.max_splits);  // within the grid
  return len;
}

// The output element(s) of row b, query head h, starting at head-dim column `col`: bf16 y, or its
// fp8 quantize (the o_proj input quantize of devstral2.py:93-95,110-111) with out_fp8.
template <int N>
__device__ __forceinline__ void store_output(const DecodeArgs& a, int b, int h, int col, const float (&y)[N]) {
  const int64_t at = b * a.out_stride + h * a.out_head_stride + col;
  uint32_t w[(N + 1) / 2];  // bf16 pairs
  if constexpr (N == 1) {
    w[0] = pack_bf16x2(y[0], 0.f);
  } else {
#pragma unroll
    for (int e = 0; e < N / 2; ++e) w[e] = pack_bf16x2(y[2 * e], y[2 * e + 1]);
  }
  if (a.out_fp8) {
    const float qs = a.quant_scale_dev != nullptr ? *a.quant_scale_dev : a.quant_scale_host;
    const float rcp = 1.0f / qs;
    float qv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int ee = e < N ? e : 0;
      const float v = (ee & 1) ? bf16_hi(w[ee / 2]) : bf16_lo(w[ee / 2]);
      qv[e] = div_by_scale(v, qs, rcp);
    }
    const uint32_t codes = fp8x4_saturate_encode(qv[0], qv[1], qv[2], qv[3]);
    uint8_t* dst = static_cast<uint8_t*>(a.out) + at;
    if constexpr (N == 1) {
      dst[0] = static_cast<uint8_t>(codes);
    } else if constexpr (N == 2) {
      *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(codes);
    } else {
      *reinterpret_cast<uint32_t*>(dst) = codes;
    }
  } else {
    uint16_t* dst = static_cast<uint16_t*>(a.out) + at;
    if constexpr (N == 1) {
      dst[0] = static_cast<uint16_t>(w[0]);
    } else if constexpr (N == 2) {
      *reinterpret_cast<uint32_t*>(dst) = w[0];
    } else {
      *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
    }
  }
}

// Max over the 64 lanes of a wavefront.
__device__ __forceinline__ float wave_max(float v) {
  v = row_max16(v);
  const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 0));
  const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16));
  const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 32));
  const float r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 48));
  return fmaxf(fmaxf(r0, r1), fmaxf(r2, r3));
}

// One wavefront per (query head, row): lane s reads split s's (max, sum) (64 splits per pass), the
// weights are broadcast with readlane, and each lane accumulates D / 64 head-dim elements.
// kSplitLen: the split length of a row, as the split kernel takes it.
template <int D, int (*kSplitLen)(const DecodeArgs&, int) = row_split_len>
__global__ __launch_bounds__(64) void decode_attn_combine(DecodeArgs a) {
  constexpr int DPL = D / 64;  // head-dim elements per lane
  const int lane = threadIdx.x;
  const int h = blockIdx.x, b = blockIdx.y;
  const int64_t raw = a.seq_lens[b];
  const int64_t cap = a.max_blocks << a.log2_page;
  // reported at the end: a global atomic here would turn the loads below into waits on every load
  const bool len_bad = raw < 0 || raw > cap;
  const int L = static_cast<int>(raw < 0 ? 0 : (raw > cap ? cap : raw));
  const int split_len = kSplitLen(a, L);
  const int nsplit = (L + split_len - 1) / split_len;
  if (nsplit == 1) {  // the split kernel wrote this row's output
    if (len_bad && h == 0 && lane == 0) report(a.err, MAS_ERRBIT_POSITION);
    return;
  }
  const int64_t base = (static_cast<int64_t>(b) * a.hq + h) * a.max_splits;
  float acc[DPL];
#pragma unroll
  for (int e = 0; e < DPL; ++e) acc[e] = 0.f;
  float lsum = 0.f;
  constexpr int kOneRound = 32, kGroup = 8;
  if (nsplit <= kOneRound) {
    // Every load in one round trip: lane s reads split s's (max, sum), and all splits' partial O
    // rows are loaded, in groups of 8 as far as the row's splits go (indices past the last split
    // clamped to it, weighted 0), before the max is known. Same weights and summation order as the general path below.
    const int last = nsplit > 0 ? nsplit - 1 : 0;
    const int sl = lane < nsplit ? lane : last;
    const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + (base + sl) * 2);
    const float* po = a.part_o + base * D + DPL * lane;
    float v[kOneRound][DPL];
    auto load_group = [&](int u0) {
#pragma unroll
      for (int u = u0; u < u0 + kGroup; ++u) {
        const int su = u < nsplit ? u : last;
#pragma unroll
        for (int e = 0; e < DPL; ++e) v[u][e] = po[su * D + e];
      }
    };
    load_group(0);
#pragma unroll
    for (int u0 = kGroup; u0 < kOneRound; u0 += kGroup)
      if (nsplit > u0) load_group(u0);  // uniform
    const float m_lane = lane < nsplit ? ml[0] : kNegInf;
    const float mx = wave_max(m_lane);
    if (mx != kNegInf) {
      const float wgt = lane < nsplit ? __builtin_amdgcn_exp2f(m_lane - mx) : 0.f;
      lsum = wgt * ml[1];
#pragma unroll
      for (int u = 0; u < kOneRound; ++u) {
        if (u < nsplit) {
          const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wgt), u));
#pragma unroll
          for (int e = 0; e < DPL; ++e) acc[e] = __builtin_fmaf(wj, v[u][e], acc[e]);
        }
      }
    }
  } else {
    float mx = kNegInf;
    for (int s = lane; s < nsplit; s += 64) mx = fmaxf(mx, a.part_ml[(base + s) * 2]);
    mx = wave_max(mx);
    if (mx != kNegInf) {
      for (int s0 = 0; s0 < nsplit; s0 += 64) {
        float wgt = 0.f;
        if (s0 + lane < nsplit) {
          const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + (base + s0 + lane) * 2);
          wgt = __builtin_amdgcn_exp2f(ml[0] - mx);
          lsum = __builtin_fmaf(wgt, ml[1], lsum);
        }
        const int cnt = min(64, nsplit - s0);
        const float* po = a.part_o + (base + s0) * D + DPL * lane;
        // eight splits' partials loaded before any is used, so their loads are in flight together
        constexpr int kU = 8;
        int j = 0;
        for (; j + kU <= cnt; j += kU) {
          float v[kU][DPL];
#pragma unroll
          for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int e = 0; e < DPL; ++e) v[u][e] = po[(j + u) * D + e];
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wgt), j + u));
#pragma unroll
            for (int e = 0; e < DPL; ++e) acc[e] = __builtin_fmaf(wj, v[u][e], acc[e]);
          }
        }
        for (; j < cnt; ++j) {
          const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wgt), j));
#pragma unroll
          for (int e = 0; e < DPL; ++e) acc[e] = __builtin_fmaf(wj, po[j * D + e], acc[e]);
        }
      }
    }
  }
  if (len_bad && h == 0 && lane == 0) report(a.err, MAS_ERRBIT_POSITION);
  const float denom = wave_sum(lsum);
  const float scale = denom > 0.f ? a.out_scale / denom : 0.f;
  float y[DPL];
#pragma unroll
  for (int e = 0; e < DPL; ++e) y[e] = acc[e] * scale;
  store_output<DPL>(a, b, h, DPL * lane, y);
}

// Workspace bytes of the partials: (max, sum) and an unnormalised O row per (row, query head, split).
int64_t decode_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t head_dim, int64_t splits) {
  return batch * num_q_heads * (splits > 0 ? splits : 1) * (head_dim + 2) * 4;
}

}  // namespace
}  // namespace mas
