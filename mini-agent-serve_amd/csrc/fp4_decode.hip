// fp4_decode.hip - paged decode attention over the 4-bit KV cache that fp4_cache.hip writes.
//
// For decode row b and query head h (kv head h / G, G = Hq / Hk), over the positions p < seq_lens[b], whose
// codes and powers (fp4.h) sit at page = block_tables[b, p / page_size], entry = p % page_size:
//   s_p = bmm1_scale * (q[b, h] . k_p),   out[b, h] = bmm2_scale * sum_p softmax(s)_p * v_p,
// k_p and v_p the values the codes stand for; fp32 sums, rounded once to bf16 (decode attention over the
// bf16 cache, devstral2.py:184-196, on another cache format).
//
// Split-KV as there (decode_split.h): a workgroup of four wavefronts per (kv head, split, row), then the merge of
// the splits. The wavefronts take the split's steps of 32 positions (two 16-position tiles) in turn, each entirely
// in registers, and add up through LDS at the end:
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16: lane (n, r) loads quarter r of key row n (32 codes of head_dim 128, one
//     block) and decodes it (v_cvt_scalef32_pk_bf16_fp4, exact); the columns of B are the kv head's query heads, with
//     the head dim numbered as the lanes hold it. (The scaled MFMAs take e2m1 operands as they lie in memory, but
//     sum groups of 8 products in a window of 14 bits below the largest - checked on MI355X - where the bf16 ones keep
//     24: with queries as two e4m3 terms, scores of large terms were off by up to 2^-10 of them.)
//   P^T = softmax weights in the result's layout: lane (n, r) holds head n at positions 4 r + j of both
//     tiles, which is the layout of the B operand of the next product when its 32 positions are numbered that way.
//   O^T += V^T P^T on v_mfma_f32_16x16x32_bf16: lane (n, r) reads, for its 8 positions, the D / 16 codes of
//     head-dim elements D / 16 * n .. and decodes them; a byte permute per word pairs positions instead of elements.
//     P enters as two bf16 terms, so it keeps 16 significant bits.
// The softmax's reference m is lazy: a step's weights are taken against the m the row has, and only where a
// lane's sum over the step passes 2^8 (or is NaN or infinite: the first step's m is -inf) does m move to the maximum.
// What bounds it: HBM for long rows (68 bytes per head and position at head_dim 128, each of keys and values: 64 rows of
// up to 8192, 295 MB, 59 us back to back, 67 us from cold caches), launch and memory latency for few (one row of 4096: 5.0 us
// and 3.9 for the merge).
#include "decode_split.h"
#include "fp4.h"

namespace mas {
namespace {

constexpr float kSumMost = 256.f;

// `bytes` of memory at a wavefront-uniform address as a raw buffer resource (dword 3 = the 32-bit data format that
// untyped buffer loads take on gfx9): loads take a scalar base, a 32-bit lane offset and a scalar one, with no vector
// arithmetic, and give zeros past the end.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
}

// Two wavefronts share less of a workgroup's start and merge (200 rows of up to 1000 at head_dim 64 12.3 -> 16.2 us, 24 rows
// of up to 3000 20.6 -> 21.2); with eight of this size a CU holds one workgroup (14.4, 28.6; 64 rows of up to 8192
// 60 -> 82 us).
constexpr int kWaves = 4;
constexpr int kStep = 32;                    // positions a wavefront takes at a time
constexpr int kRound = kWaves * kStep;       // and a workgroup
constexpr int kMaxSplitLen = 1024;           // positions per split, at most, while max_splits reach
constexpr int kMaxSplits = 128;
// Workgroups of a launch: the splits of a table far wider than its rows are mostly empty, and each costs 1.3 ns. 64 rows of
// 300 positions under a table of 131072 took 79 us with all 128 splits and 21 with these 8192 workgroups (16384: 29; 4096:
// 17), rows of 2000 to 4300 99 and 47 (54; 45), one row as long as the table among them 106 and 77 (58; 121).
constexpr int64_t kMostItems = 8192;
constexpr int kLongestSplit = 16384;             // positions; as many more workgroups as that takes
constexpr int64_t kMaxItems = int64_t{1} << 23;  // but no more than this (a grid is below 2^32 threads)

// A row's split length: its share of row_target splits, in whole rounds, at most kMaxSplitLen; and such that its splits
// fit the grid and the workspace.
__device__ __forceinline__ int fp4_split_len(const DecodeArgs& a, int L) {
  const int rounds = (L + kRound - 1) / kRound;
  const int share = (rounds + a.row_target - 1) / a.row_target;
  const int least = (rounds + a.max_splits - 1) / a.max_splits;
  return kRound * max(max(min(share, kMaxSplitLen / kRound), least), 1);
}

struct Fp4DecodeArgs : DecodeArgs {
  int batch;
  uint32_t splits_inverse;  // 2^32 / max_splits, rounded up: exact quotients of what is below 2^25 (0: of 1)
  int heads_share;  // kv heads' codes share 128-byte lines
  int code_bytes, power_bytes;  // from a head's first code (power) to the end of its last page's, in a cache below 2 GiB
  Fp4Cache c;
};

// One step's keys and values as they lie in the cache.
template <int D>
struct Fp4Loads {
  static constexpr int KW = D / 32;                       // words of a lane's quarter of a key row
  static constexpr int KP = D == 256 ? 2 : 1;             // powers of it
  static constexpr int VW = D / 128 > 0 ? D / 128 : 1;    // words of value codes per position (64: half a word)
  uint32_t k[2][KW];
  uint32_t ks[2][KP];
  uint32_t v[2][4][VW];
  uint32_t vs[2];
  int count[2];  // valid positions of each tile (wavefront-uniform)
};

// kWide: a cache tensor of 2 GiB or more, whose tiles each get buffer resources of their own; else one resource per tensor
// serves every tile at a 32-bit scalar offset, which leaves the scalar unit a third of the work (it serves all of a CU's
// wavefronts).
template <int D, bool kWide>
__global__ __launch_bounds__(64 * kWaves, D <= 128 ? 3 : 2) void fp4_decode_split(Fp4DecodeArgs a) {
  using Loads = Fp4Loads<D>;
  constexpr int EL = D / 16;     // head-dim elements per lane of the value operand: EL n ..
  constexpr int NB = EL / 2;     // their code bytes per position
  const int lane = threadIdx.x & 63;
  const int wave = wave_id_uniform();
  // Workgroups go to the XCDs round-robin by id. Where heads share 128-byte lines (the NHD layout up to head_dim 128),
  // all kv heads of a (split, row) item run on one XCD, so that a line comes from memory once: 64 rows of up to 8192
  // positions 102 -> 67 us. Elsewhere the heads are dealt out, which balances the XCDs better (HND 62 -> 60 us). A row
  // shorter than the table has only its first splits to do: those of row b are rotated by b + b / 4 over the items.
  // (No branch before the row's length is there, so the arguments load at once, and the length right after them; and no
  // divisions but one: 24 rows of up to 3000 20.5 -> 20.0 us, 62 of up to 600 17.9 -> 17.5, one of 4096 7.65 -> 7.58.)
  const unsigned id = blockIdx.x, hk = a.hk, queue = a.heads_share ? id / kXcds : id;
  const unsigned dealt = queue / hk, item = a.heads_share ? dealt * kXcds + id % kXcds : dealt;
  const int kvh = static_cast<int>(queue - dealt * hk);
  const auto by_splits = [&](unsigned x) { return a.splits_inverse != 0 ? __umulhi(x, a.splits_inverse) : x; };
  const unsigned b_of = by_splits(item), y = item - b_of * a.max_splits;
  const bool no_row = b_of >= static_cast<unsigned>(a.batch);  // the grid is rounded up
  const int b = no_row ? a.batch - 1 : static_cast<int>(b_of);
  const unsigned turned = y + (a.max_splits & 1 ? 0u : b_of + (b_of >> 2));
  const int split = static_cast<int>(turned - by_splits(turned) * a.max_splits);
  const int L = kv_len(a, b);
  const int split_len = fp4_split_len(a, L);
  const int start = split * split_len;
  if (no_row) return;
  if (split == 0 && kvh == 0 && threadIdx.x == 0) {
    const int64_t raw = a.seq_lens[b];
    if (raw < 0 || raw > a.max_blocks << a.log2_page) report(a.err, MAS_ERRBIT_POSITION);
  }
  if (start >= L) {
    if (split == 0) {  // a row with no position
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = threadIdx.x; i < a.group * (D / 4); i += 64 * kWaves)
        store_output<4>(a, b, kvh * a.group + i / (D / 4), 4 * (i % (D / 4)), zero);
    }
    return;
  }
  const int end = min(start + split_len, L);
  const int G = a.group;
  const int n = lane & 15, r = lane >> 4;

  // A tile's page id is a scalar load, a step ahead of the tile's own loads (constant address space, so that it
  // counts on another counter than those: a vector load here would wait for all of them).
  const auto bt = (const __attribute__((address_space(4))) int32_t*)(a.block_tables + b * a.bt_stride);
  const int last_entry = (end - 1) >> a.log2_page;
  struct Ids {
    int32_t page[2];
  };
  auto fetch = [&](int pos) {
    return Ids{{bt[min(pos >> a.log2_page, last_entry)], bt[min((pos + 16) >> a.log2_page, last_entry)]}};
  };
  const int begin = start + wave * kStep;  // this wavefront's first step
  Ids ids = fetch(begin);
  // B operands of S^T = K Q^T: head n, head-dim elements D / 4 r + 8 j + 0..7 (zeros past the group)
  constexpr int KJ = D / 32;
  bf16x8 q[KJ];
  {
    const uint16_t* row = a.q + b * a.q_stride + static_cast<int64_t>(kvh * G + (n < G ? n : 0)) * a.q_head_stride;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      u32x4 v = load_cached(row + D / 4 * r + 8 * j);
      if (n >= G) v = u32x4{0u, 0u, 0u, 0u};
      q[j] = __builtin_bit_cast(bf16x8, v);
    }
  }

  const uint32_t es = static_cast<uint32_t>(a.c.entry_stride), ps = static_cast<uint32_t>(a.c.page_size);
  // this lane's byte offsets in a tile: its quarter of its key row, its value rows' codes, and their powers
  const uint32_t k_off = n * es + D / 8 * r;
  const uint32_t ks_off = (D / 4 * r / kFp4Block) * ps + n;
  const uint32_t v_off = 4 * r * es + n * NB;
  const uint32_t vs_off = (n * EL / kFp4Block) * ps + 4 * r;
  const int mask = static_cast<int>(a.c.page_size) - 1;
  const uint8_t* const k_head = a.c.k + kvh * a.c.head_stride;
  const uint8_t* const v_head = a.c.v + kvh * a.c.head_stride;
  const uint8_t* const ks_head = a.c.k_scale + kvh * a.c.scale_head_stride;
  const uint8_t* const vs_head = a.c.v_scale + kvh * a.c.scale_head_stride;

  const uint32_t pages_u32 = static_cast<uint32_t>(min(a.c.num_pages, static_cast<int64_t>(INT32_MAX)));
  bool bad = false;
  // Issues the loads of the step at `pos`, whose pages are in `ids`, and fetches the next step's. Rows past the row's
  // end, and all of a tile on a page id outside the cache (page 0 is read), are loaded and do not count.
  const __amdgpu_buffer_rsrc_t k_all = buffer_of(k_head, a.code_bytes), v_all = buffer_of(v_head, a.code_bytes);
  const __amdgpu_buffer_rsrc_t ks_all = buffer_of(ks_head, a.power_bytes), vs_all = buffer_of(vs_head, a.power_bytes);
  auto issue = [&](Loads& st, int pos) {
    __amdgpu_buffer_rsrc_t k_at[2] = {k_all, k_all}, v_at[2] = {v_all, v_all};
    __amdgpu_buffer_rsrc_t ks_at[2] = {ks_all, ks_all}, vs_at[2] = {vs_all, vs_all};
    uint32_t at[2], sat[2];  // the tiles' first rows and powers, from the resources' bases
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int p = pos + 16 * t;
      const uint32_t page_id = static_cast<uint32_t>(ids.page[t]);
      const bool ok = page_id < pages_u32;
      const uint32_t page = ok ? page_id : 0u, slot = static_cast<uint32_t>(p & mask);
      int count = min(end - p, 16);
      asm("" : "+s"(count));  // (a clamp would become a vector median)
      st.count[t] = ok ? max(count, 0) : 0;
      bad |= !ok;
      if constexpr (kWide) {
        const int64_t code = static_cast<int64_t>(page) * a.c.page_stride + slot * es;
        const int64_t power = static_cast<int64_t>(page) * a.c.scale_page_stride + slot;
        const int bytes = 15 * static_cast<int>(es) + D / 2, sbytes = static_cast<int>(D / kFp4Block * ps - slot);
        k_at[t] = buffer_of(k_head + code, bytes);
        v_at[t] = buffer_of(v_head + code, bytes);
        ks_at[t] = buffer_of(ks_head + power, sbytes);
        vs_at[t] = buffer_of(vs_head + power, sbytes);
        at[t] = sat[t] = 0;
      } else {
        at[t] = page * static_cast<uint32_t>(a.c.page_stride) + slot * es;
        sat[t] = page * static_cast<uint32_t>(a.c.scale_page_stride) + slot;
      }
    }
    ids = fetch(pos + kRound);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (D == 64) {
        const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(k_at[t], k_off, at[t], 0);
        st.k[t][0] = x[0];
        st.k[t][1] = x[1];
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(k_at[t], k_off + 16 * h, at[t], 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) st.k[t][4 * h + i] = x[i];
        }
      }
#pragma unroll
      for (int h = 0; h < Loads::KP; ++h) st.ks[t][h] = __builtin_amdgcn_raw_buffer_load_b8(ks_at[t], ks_off, sat[t] + h * ps, 0);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (D == 64) {
          st.v[t][i][0] = __builtin_amdgcn_raw_buffer_load_b16(v_at[t], v_off, at[t] + i * es, 0);
        } else if constexpr (D == 128) {
          st.v[t][i][0] = __builtin_amdgcn_raw_buffer_load_b32(v_at[t], v_off, at[t] + i * es, 0);
        } else {
          const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(v_at[t], v_off, at[t] + i * es, 0);
          st.v[t][i][0] = x[0];
          st.v[t][i][1] = x[1];
        }
      }
      st.vs[t] = __builtin_amdgcn_raw_buffer_load_b32(vs_at[t], vs_off, sat[t], 0);
    }
  };

  float m_run = kNegInf, l_run = 0.f;  // head n's reference (in all four lanes), this lane's share of its sum
  f32x4 acc[EL];  // O^T: element j of acc[e] holds O[head n][EL (4 r + j) + e]
#pragma unroll
  for (int e = 0; e < EL; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](Loads& st) {
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const float f = __uint_as_float(st.ks[t][j * Loads::KP / KJ] << 23);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fp4x8_decode(st.k[t][j], f)), q[j],
                                                       s[t], 0, 0, 0);
      }
      s[t] *= a.scale_log2;
      if (st.count[t] < 16) {  // uniform: the row's end, or a page outside the cache
        const int left = st.count[t] - 4 * r;  // valid positions of this lane's four
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j >= left) {
            s[t][j] = kNegInf;
#pragma unroll
            for (int x = 0; x < Loads::VW; ++x) st.v[t][j][x] = 0u;
          }
        // (a power of 255 would make even zeros NaN)
        st.vs[t] = left >= 4 ? st.vs[t] : left <= 0 ? 0u : st.vs[t] & ((1u << (8 * left)) - 1u);
      }
    }
    float p[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] - m_run);
      sum += p[e];
    }
    const uint64_t over = __builtin_amdgcn_ballot_w64(!(sum <= kSumMost));
    if (over != 0) {  // some head's reference moves
      const uint32_t heads = static_cast<uint32_t>(over | over >> 16 | over >> 32 | over >> 48) & 0xffffu;
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const bool moves = (heads >> n) & 1u;
      const float m_new = moves ? fmaxf(m_run, mx) : m_run;
      const float alpha = moves && m_run != kNegInf ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int e = 0; e < EL; ++e) acc[e] *= alpha;
      const float m_use = m_run == kNegInf ? 0.f : m_run;
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] - m_use);
        sum += p[e];
      }
    }
    l_run += sum;
    u32x4 ph, pl;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ph[e] = pack_bf16x2(p[2 * e], p[2 * e + 1]);
      pl[e] = pack_bf16x2(p[2 * e] - bf16_lo(ph[e]), p[2 * e + 1] - bf16_hi(ph[e]));
    }
    const bf16x8 p_hi = __builtin_bit_cast(bf16x8, ph), p_lo = __builtin_bit_cast(bf16x8, pl);
    float f[2][4];  // the positions' powers, as the decode's scales
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f[t][0] = __uint_as_float(st.vs[t] << 23);
      f[t][1] = __uint_as_float(st.vs[t] << 15);
      f[t][2] = __uint_as_float(st.vs[t] << 7);
      f[t][3] = __uint_as_float(st.vs[t] >> 1);
    }
    auto weigh = [&](auto byte) {
      constexpr int c = decltype(byte)::value;
      u32x4 even, odd;  // elements 2 c and 2 c + 1 of this lane at its 8 positions
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = fp4x2_decode<c & 3>(st.v[t][2 * i][c >> 2], f[t][2 * i]);
          const uint32_t y = fp4x2_decode<c & 3>(st.v[t][2 * i + 1][c >> 2], f[t][2 * i + 1]);
          even[2 * t + i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
          odd[2 * t + i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
      const bf16x8 ve = __builtin_bit_cast(bf16x8, even), vo = __builtin_bit_cast(bf16x8, odd);
      acc[2 * c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, p_lo, acc[2 * c], 0, 0, 0);
      acc[2 * c + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, p_lo, acc[2 * c + 1], 0, 0, 0);
      acc[2 * c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, p_hi, acc[2 * c], 0, 0, 0);
      acc[2 * c + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, p_hi, acc[2 * c + 1], 0, 0, 0);
    };
    weigh(std::integral_constant<int, 0>{});
    weigh(std::integral_constant<int, 1>{});
    if constexpr (NB > 2) {
      weigh(std::integral_constant<int, 2>{});
      weigh(std::integral_constant<int, 3>{});
    }
    if constexpr (NB > 4) {
      weigh(std::integral_constant<int, 4>{});
      weigh(std::integral_constant<int, 5>{});
      weigh(std::integral_constant<int, 6>{});
      weigh(std::integral_constant<int, 7>{});
    }
  };

  // Two load buffers used in turn: a step is computed while the next one's loads are in flight.
  const int nsteps = begin < end ? (end - begin + kRound - 1) / kRound : 0;
  if (nsteps > 0) {
    Loads ld0, ld1;
    issue(ld0, begin);
    int i = 0;
    for (; i + 2 < nsteps; i += 2) {
      issue(ld1, begin + (i + 1) * kRound);
      compute(ld0);
      issue(ld0, begin + (i + 2) * kRound);
      compute(ld1);
    }
    if (i + 1 < nsteps) {
      issue(ld1, begin + (i + 1) * kRound);
      compute(ld0);
      compute(ld1);
    } else {
      compute(ld0);
    }
  }
  if (__builtin_amdgcn_ballot_w64(bad) != 0 && lane == 0) report(a.err, MAS_ERRBIT_PAGE);

  // ---- the wavefronts' sums: each brings its own to the workgroup's reference and puts them into LDS
  constexpr int OROW = D + 4;  // floats per LDS row: the 16 heads' rows start 4 banks apart
  __shared__ __align__(16) float o_lds[kWaves][16 * OROW];
  __shared__ float m_lds[kWaves][16], l_lds[kWaves][16], m_all_lds[16];
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (r == 0) m_lds[wave][n] = m_run;
  __syncthreads();
  const float m_all = fmaxf(fmaxf(m_lds[0][n], m_lds[1][n]), fmaxf(m_lds[2][n], m_lds[3][n]));
  // (a wavefront without a finite score has sums of zero, or NaN ones where its scores are)
  const float factor = m_run == kNegInf ? (l_run != l_run ? l_run : 0.f) : __builtin_amdgcn_exp2f(m_run - m_all);
  if (n < G) {
    if (r == 0) l_lds[wave][n] = l_run * factor;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < EL; e += 4)
        *reinterpret_cast<f32x4*>(&o_lds[wave][n * OROW + EL * (4 * r + j) + e]) =
            f32x4{acc[e][j] * factor, acc[e + 1][j] * factor, acc[e + 2][j] * factor, acc[e + 3][j] * factor};
  }
  if (wave == 0 && r == 0) m_all_lds[n] = m_all;
  __syncthreads();
  constexpr int kVecs = D / 4;  // 16-byte pieces per head row
  for (int i = threadIdx.x; i < G * kVecs; i += 64 * kWaves) {
    const int g = i / kVecs, c = i % kVecs;
    f32x4 o = *reinterpret_cast<const f32x4*>(&o_lds[0][g * OROW + 4 * c]);
    float l = l_lds[0][g];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      o += *reinterpret_cast<const f32x4*>(&o_lds[w][g * OROW + 4 * c]);
      l += l_lds[w][g];
    }
    const int h = kvh * G + g;
    if (L <= split_len) {  // the row's only split: its output
      const float sc = l > 0.f ? a.out_scale / l : 0.f;
      const float y[4] = {o[0] * sc, o[1] * sc, o[2] * sc, o[3] * sc};
      store_output<4>(a, b, h, 4 * c, y);
    } else {
      const int64_t at = (static_cast<int64_t>(b) * a.hq + h) * a.max_splits + split;
      __builtin_nontemporal_store(o, reinterpret_cast<f32x4*>(a.part_o + at * D + 4 * c));
      // (scores that are all NaN leave no maximum: any one makes the merge take the split's NaN in)
      if (c == 0) *reinterpret_cast<f32x2*>(a.part_ml + at * 2) = f32x2{l != l && m_all_lds[g] == kNegInf ? 0.f : m_all_lds[g], l};
    }
  }
}

template <int D>
int launch_fp4_decode(const Fp4DecodeArgs& a, int64_t batch, bool wide, hipStream_t s) {
  const int64_t items = cdiv(batch * a.max_splits, kXcds) * kXcds;  // (row, split), with the XCDs' remainder
  const dim3 grid(static_cast<uint32_t>(items * a.hk));
  if (wide) hipLaunchKernelGGL((fp4_decode_split<D, true>), grid, dim3(64 * kWaves), 0, s, a);
  else hipLaunchKernelGGL((fp4_decode_split<D, false>), grid, dim3(64 * kWaves), 0, s, a);
  if (const int st = launch_status(); st != MAS_OK || a.max_splits == 1) return st;  // (no row of several splits)
  hipLaunchKernelGGL((decode_attn_combine<D, fp4_split_len>), dim3(static_cast<uint32_t>(a.hq), static_cast<uint32_t>(batch)),
                     dim3(64), 0, s, a);
  return launch_status();
}

}  // namespace
}  // namespace mas

extern "C" int mas_paged_decode_attention_fp4(void* out, int64_t out_stride, int64_t out_head_stride, const void* q,
                                              int64_t q_stride, int64_t q_head_stride, const void* k_cache,
                                              const void* v_cache, int64_t page_stride, int64_t entry_stride,
                                              int64_t head_stride, const void* k_scale, const void* v_scale,
                                              int64_t scale_page_stride, int64_t scale_head_stride, int64_t num_pages,
                                              int64_t page_size, const int32_t* block_tables,
                                              int64_t block_table_stride, int64_t max_blocks, const int32_t* seq_lens,
                                              int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                              int64_t head_dim, float bmm1_scale, float bmm2_scale, int out_fp8,
                                              const float* out_scale_dev, float out_scale_host, void* workspace,
                                              int64_t workspace_bytes, uint32_t* err, hipStream_t stream) {
  using namespace mas;
  if (batch < 0 || num_q_heads < 0 || num_kv_heads < 0 || max_blocks < 0 || workspace_bytes < 0)
    return MAS_ERR_INVALID_VALUE;
  Fp4DecodeArgs a{};
  a.c.k = static_cast<uint8_t*>(const_cast<void*>(k_cache));
  a.c.v = static_cast<uint8_t*>(const_cast<void*>(v_cache));
  a.c.page_stride = page_stride;
  a.c.entry_stride = entry_stride;
  a.c.head_stride = head_stride;
  a.c.k_scale = static_cast<uint8_t*>(const_cast<void*>(k_scale));
  a.c.v_scale = static_cast<uint8_t*>(const_cast<void*>(v_scale));
  a.c.scale_page_stride = scale_page_stride;
  a.c.scale_head_stride = scale_head_stride;
  a.c.num_pages = num_pages;
  a.c.page_size = page_size;
  if (const int st = check_fp4_cache(a.c); st != MAS_OK) return st;
  if (batch == 0 || num_q_heads == 0) return MAS_OK;
  if (num_kv_heads == 0 || num_q_heads % num_kv_heads != 0) return MAS_ERR_INVALID_VALUE;
  const int64_t group = num_q_heads / num_kv_heads;
  if (group > 16 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return MAS_ERR_UNSUPPORTED;
  const int64_t cap = max_blocks * page_size;
  // (a page's rows are addressed with 32-bit byte offsets)
  if (cap > (int64_t{1} << 30) || batch > 65535 || num_kv_heads > 65535 || num_q_heads > 65535 ||
      batch * num_kv_heads > kMaxItems || entry_stride < 0 || page_size * entry_stride > INT32_MAX)
    return MAS_ERR_UNSUPPORTED;
  if (out == nullptr || q == nullptr || seq_lens == nullptr ||
      (cap > 0 && (block_tables == nullptr || num_pages == 0)))
    return MAS_ERR_INVALID_VALUE;
  if (out_fp8 && out_scale_dev == nullptr && !(out_scale_host > 0.f)) return MAS_ERR_INVALID_VALUE;
  if (!aligned16(q) || !aligned16(out) || q_stride % 8 != 0 || q_head_stride % 8 != 0 || out_stride % 8 != 0 ||
      out_head_stride % 8 != 0 || !aligned16(workspace))
    return MAS_ERR_MISALIGNED;
  // Splits wanted per row: four workgroups per CU over the (row, kv head) pairs. The longest row a table can hold
  // then has the more of those and of kMaxSplitLen-position splits; fewer where the launch or the workspace would not
  // hold them.
  int cus = 0;
  if (workspace == nullptr) return MAS_ERR_INVALID_VALUE;
  if (const int st = device_cu_count(&cus); st != MAS_OK) return st;
  const int64_t target = std::max<int64_t>(1, 4 * static_cast<int64_t>(cus) / (batch * num_kv_heads));
  const int64_t held = workspace_bytes / decode_workspace_bytes(batch, num_q_heads, head_dim, 1);
  if (held < 1) return MAS_ERR_INVALID_VALUE;
  const int64_t pairs = batch * num_kv_heads;
  const int64_t wanted = std::max(std::min(target, cdiv(cap, kRound)), cdiv(cap, kMaxSplitLen));
  const int64_t launched = std::min(std::max(kMostItems / pairs, cdiv(cap, kLongestSplit)), kMaxItems / pairs);
  const int64_t splits = std::max<int64_t>(1, std::min({wanted, launched, int64_t{kMaxSplits}, held}));
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride;
  a.q_head_stride = q_head_stride;
  a.num_pages = num_pages;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.hq = static_cast<int>(num_q_heads);
  a.hk = static_cast<int>(num_kv_heads);
  a.group = static_cast<int>(group);
  while ((int64_t{1} << a.log2_page) < page_size) ++a.log2_page;
  a.batch = static_cast<int>(batch);
  a.heads_share = num_kv_heads > 1 && head_stride > -128 && head_stride < 128;
  a.splits_inverse = splits > 1 ? static_cast<uint32_t>(((uint64_t{1} << 32) + splits - 1) / splits) : 0;
  a.row_target = static_cast<int>(target);
  a.max_splits = static_cast<int>(splits);
  a.scale_log2 = bmm1_scale * 1.4426950408889634f;
  a.out_scale = bmm2_scale;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + batch * num_q_heads * splits * head_dim;
  a.out = out;
  a.out_stride = out_stride;
  a.out_head_stride = out_head_stride;
  a.out_fp8 = out_fp8 != 0;
  a.quant_scale_dev = out_scale_dev;
  a.quant_scale_host = out_scale_host;
  a.err = err;
  // A head's codes reach over the pages before the last one, that page's rows and one row; its powers likewise.
  const int64_t code_bytes = (num_pages - 1) * page_stride + (page_size - 1) * entry_stride + head_dim / 2;
  const int64_t power_bytes = (num_pages - 1) * scale_page_stride + head_dim / kFp4Block * page_size;
  const bool wide = page_stride < 0 || scale_page_stride < 0 || code_bytes > INT32_MAX || power_bytes > INT32_MAX;
  a.code_bytes = wide ? 0 : static_cast<int>(code_bytes);
  a.power_bytes = wide ? 0 : static_cast<int>(power_bytes);
  switch (head_dim) {
    case 64: return launch_fp4_decode<64>(a, batch, wide, stream);
    case 128: return launch_fp4_decode<128>(a, batch, wide, stream);
    default: return launch_fp4_decode<256>(a, batch, wide, stream);
  }
}
