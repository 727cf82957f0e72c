// fp4_cache.hip - a step's key / value rows into the 4-bit KV cache, and rows of it back.
//
// The paged append of kv_store.hip (the same two forms of destination, devstral2.py:170-173,289) with the
// rows quantized on the way (fp4.h): for each block of 32 elements of a head,
//   s = the power byte of max |x|,   code_i = e2m1(x_i / 2^(s - 127)),
// and the reverse, y_i = e2m1(code_i) 2^(s - 127) as bf16, exact, for rows named by their slots.
//
// A lane holds 8 elements (one 16-byte load), four lanes a block: its maximum is a packed 16-bit maximum over
// the magnitudes' bits and two quad permutes. One wavefront per (one or four tokens, keys or values, 512 elements), all
// its tokens' loads issued before their destinations are resolved. Four tokens that follow each other in a page, from an
// entry that is a multiple of four (a prompt's), store their powers as one word per block; others a byte each.
// What bounds it: memory at prompts (8192 tokens of 8 heads of 128, 42.5 MB each: store 11.0 us, load 7.5 us; a large
// copy reaches 4.8 TB/s here), the launch and the destinations' chain of loads at a decode batch (3.1 and 2.6 us).
#include "fp4.h"

namespace mas {
namespace {

struct Fp4Args : Fp4Cache {
  // the tokens' rows: sources of the store, destinations of the load
  uint16_t* key;
  int64_t key_stride, key_head_stride;
  uint16_t* value;
  int64_t value_stride, value_head_stride;
  // block-table form
  const int32_t* batch_indices;
  const int32_t* positions;
  const int32_t* kv_indices;
  int64_t num_indices;
  const int32_t* kv_indptr;
  int64_t batch;
  // slot form
  const int64_t* slots;
  int64_t rows;
  int vec_per_head, vec_per_row;  // of 8 elements
  int parts;                      // wavefronts per (its tokens, tensor)
  int log2_page;
  uint32_t* err;
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, false));
}

// Where token t's row lies: byte offsets of its codes and powers, less the head's and the block's. Each lane resolves
// one token (lane % kTokens), so a wavefront's four take one chain of dependent loads (resolved in turn, with scalar loads,
// the store of 64 tokens took 5.4 us for 3.2).
struct Dest {
  int64_t code, power;
  int page, entry;
  bool ok;
};
template <bool kSlotForm, int kTokens>
__device__ __forceinline__ Dest dest_of(const Fp4Args& a, int64_t t) {
  Dest d{0, 0, 0, 0, false};
  if (t >= a.rows) return d;
  int64_t page = -1, entry = 0;
  uint32_t bad = 0;
  if constexpr (kSlotForm) {
    const int64_t slot = a.slots[t];
    if (slot < 0) return d;
    page = slot >> a.log2_page;
    entry = slot & (a.page_size - 1);
    if (page >= a.num_pages) bad = MAS_ERRBIT_SLOT;
  } else {
    const int64_t b = a.batch_indices[t], p = a.positions[t];
    if (b < 0 || b >= a.batch) {
      bad = MAS_ERRBIT_BATCH;
    } else if (p < 0) {
      bad = MAS_ERRBIT_POSITION;
    } else {
      const int64_t idx = a.kv_indptr[b] + (p >> a.log2_page);
      if (idx < 0 || idx >= a.num_indices || idx >= a.kv_indptr[b + 1]) {
        bad = MAS_ERRBIT_PAGE;
      } else {
        page = a.kv_indices[idx];
        entry = p & (a.page_size - 1);
        if (page < 0 || page >= a.num_pages) bad = MAS_ERRBIT_PAGE;
      }
    }
  }
  if (bad != 0) {
    if ((threadIdx.x & (kWave - 1)) < kTokens) report(a.err, bad);
    return d;
  }
  d.code = page * a.page_stride + entry * a.entry_stride;
  d.power = page * a.scale_page_stride + entry;
  d.page = static_cast<int>(page);
  d.entry = static_cast<int>(entry);
  d.ok = true;
  return d;
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
  const auto lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
  const auto hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// What a wavefront works on, and its lane's place in the rows.
struct Place {
  int64_t t0;
  int count;   // tokens
  bool is_v, live;
  int h, col;  // head, 8-element vector in it
};
template <int kTokens>
__device__ __forceinline__ Place place_of(const Fp4Args& a) {
  const int lane = threadIdx.x & (kWave - 1);
  const unsigned per_group = 2u * static_cast<unsigned>(a.parts);
  const unsigned group = blockIdx.x / per_group, rem = blockIdx.x - group * per_group;
  const unsigned part = rem >> 1;
  const int v = static_cast<int>(part) * kWave + lane;
  const int h = v / a.vec_per_head;
  const int64_t t0 = static_cast<int64_t>(group) * kTokens;
  const int64_t left = a.rows - t0;
  return {t0, left < kTokens ? static_cast<int>(left) : kTokens, (rem & 1u) != 0, v < a.vec_per_row, h,
          v - h * a.vec_per_head};
}

template <bool kSlotForm, int kTokens>
__global__ __launch_bounds__(kWave) void fp4_store(Fp4Args a) {
  const Place p = place_of<kTokens>(a);
  const uint16_t* src = p.is_v ? a.value + p.t0 * a.value_stride + p.h * a.value_head_stride
                               : a.key + p.t0 * a.key_stride + p.h * a.key_head_stride;
  const int64_t row = p.is_v ? a.value_stride : a.key_stride;
  u32x4 w[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    w[i] = u32x4{0u, 0u, 0u, 0u};
    if (p.live && i < p.count) w[i] = load_stream(src + i * row + 8 * p.col);
  }
  load_fence();
  const Dest d = dest_of<kSlotForm, kTokens>(a, p.t0 + (threadIdx.x & (kTokens - 1)));
  const uint64_t ok = __builtin_amdgcn_ballot_w64(d.ok);
  const int page0 = __builtin_amdgcn_readlane(d.page, 0), entry0 = __builtin_amdgcn_readlane(d.entry, 0);
  const bool follows = d.ok && d.page == page0 && d.entry == entry0 + static_cast<int>(threadIdx.x & (kTokens - 1));
  const bool run = kTokens == 4 && (entry0 & 3) == 0 && (__builtin_amdgcn_ballot_w64(follows) & 15u) == 15u;  // uniform
  uint32_t power[kTokens], codes[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max_u16x2(m, w[i][j] & 0x7fff7fffu);
    m = max_u16x2(m, dpp_u32<0xb1>(m));  // quad_perm [1,0,3,2]
    m = max_u16x2(m, dpp_u32<0x4e>(m));  // quad_perm [2,3,0,1]
    power[i] = fp4_power(max(m & 0xffffu, m >> 16));
    codes[i] = power[i] == 255u ? 0u : fp4x8_encode(w[i], power[i]);
  }
  if (!p.live) return;
  uint8_t* const dst = (p.is_v ? a.v : a.k) + p.h * a.head_stride + 4 * p.col;
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (ok >> i & 1u) *reinterpret_cast<uint32_t*>(dst + lane_of(d.code, i)) = codes[i];
  if ((p.col & 3) != 0) return;
  uint8_t* const sdst = (p.is_v ? a.v_scale : a.k_scale) + p.h * a.scale_head_stride + (p.col >> 2) * a.page_size;
  if (run) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < kTokens; ++i) word |= power[i] << (8 * i & 31);
    *reinterpret_cast<uint32_t*>(sdst + lane_of(d.power, 0)) = word;
  } else {
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
      if (ok >> i & 1u) sdst[lane_of(d.power, i)] = static_cast<uint8_t>(power[i]);
  }
}

// Rows of the cache as bf16; a slot that is negative or past the cache gives zeros.
template <int kTokens>
__global__ __launch_bounds__(kWave) void fp4_load(Fp4Args a) {
  const Place p = place_of<kTokens>(a);
  const Dest d = dest_of<true, kTokens>(a, p.t0 + (threadIdx.x & (kTokens - 1)));
  const uint64_t ok = __builtin_amdgcn_ballot_w64(d.ok);
  if (!p.live) return;
  const uint8_t* const src = (p.is_v ? a.v : a.k) + p.h * a.head_stride + 4 * p.col;
  const uint8_t* const ssrc = (p.is_v ? a.v_scale : a.k_scale) + p.h * a.scale_head_stride + (p.col >> 2) * a.page_size;
  uint32_t codes[kTokens], power[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    codes[i] = power[i] = 0u;
    if (ok >> i & 1u) {
      codes[i] = *reinterpret_cast<const uint32_t*>(src + lane_of(d.code, i));
      power[i] = ssrc[lane_of(d.power, i)];
    }
  }
  uint16_t* const dst = p.is_v ? a.value + p.t0 * a.value_stride + p.h * a.value_head_stride
                               : a.key + p.t0 * a.key_stride + p.h * a.key_head_stride;
  const int64_t row = p.is_v ? a.value_stride : a.key_stride;
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (i < p.count) store_stream(dst + i * row + 8 * p.col, fp4x8_decode(codes[i], __uint_as_float(power[i] << 23)));
}

// Tokens per wavefront: four where that leaves enough wavefronts. A wavefront of four waits longer for their destinations
// (MI355X, 8 heads of 128, store and load: 64 tokens 3.1 and 2.5 us with one, 3.8 and 3.1 with four; 1024 tokens 4.3
// and 3.6, 4.2 and 3.3; 4096 tokens 9.6 and 6.4, 7.1 and 4.9).
int64_t tokens_per_wave(int64_t rows, int64_t parts) { return rows * parts < 2048 ? 1 : 4; }

// Fills the row geometry and checks it; MAS_OK with *empty set when there is nothing to do.
int check_rows(Fp4Args& a, int64_t num_heads, int64_t head_dim, bool* empty) {
  if (a.rows < 0 || num_heads < 0 || head_dim < 0) return MAS_ERR_INVALID_VALUE;
  if (const int st = check_fp4_cache(a); st != MAS_OK) return st;
  if (head_dim % kFp4Block != 0 || num_heads * head_dim / 8 > INT32_MAX) return MAS_ERR_UNSUPPORTED;
  *empty = a.rows == 0 || num_heads == 0 || head_dim == 0;
  if (*empty) return MAS_OK;
  if (a.key == nullptr || a.value == nullptr) return MAS_ERR_INVALID_VALUE;
  if (!aligned16(a.key) || !aligned16(a.value) || a.key_stride % 8 != 0 || a.key_head_stride % 8 != 0 ||
      a.value_stride % 8 != 0 || a.value_head_stride % 8 != 0)
    return MAS_ERR_MISALIGNED;
  while ((int64_t{1} << a.log2_page) < a.page_size) ++a.log2_page;
  a.vec_per_head = static_cast<int>(head_dim / 8);
  a.vec_per_row = static_cast<int>(num_heads * head_dim / 8);
  a.parts = static_cast<int>(cdiv(a.vec_per_row, kWave));
  // (a grid is below 2^32 threads)
  return cdiv(a.rows, tokens_per_wave(a.rows, a.parts)) * 2 * a.parts * kWave > UINT32_MAX ? MAS_ERR_UNSUPPORTED : MAS_OK;
}

enum class Move { kAppend, kStore, kLoad };
int launch_rows(Move move, const Fp4Args& a, hipStream_t stream) {
  const int64_t tokens = tokens_per_wave(a.rows, a.parts);
  const dim3 grid(static_cast<uint32_t>(cdiv(a.rows, tokens) * 2 * a.parts)), block(kWave);
  if (tokens == 1) {
    if (move == Move::kAppend) hipLaunchKernelGGL((fp4_store<false, 1>), grid, block, 0, stream, a);
    else if (move == Move::kStore) hipLaunchKernelGGL((fp4_store<true, 1>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL(fp4_load<1>, grid, block, 0, stream, a);
  } else {
    if (move == Move::kAppend) hipLaunchKernelGGL((fp4_store<false, 4>), grid, block, 0, stream, a);
    else if (move == Move::kStore) hipLaunchKernelGGL((fp4_store<true, 4>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL(fp4_load<4>, grid, block, 0, stream, a);
  }
  return launch_status();
}

Fp4Args cache_args(void* k_cache, void* v_cache, int64_t page_stride, int64_t entry_stride, int64_t head_stride,
                   void* k_scale, void* v_scale, int64_t scale_page_stride, int64_t scale_head_stride,
                   int64_t num_pages, int64_t page_size) {
  Fp4Args a{};
  a.k = static_cast<uint8_t*>(k_cache);
  a.v = static_cast<uint8_t*>(v_cache);
  a.page_stride = page_stride;
  a.entry_stride = entry_stride;
  a.head_stride = head_stride;
  a.k_scale = static_cast<uint8_t*>(k_scale);
  a.v_scale = static_cast<uint8_t*>(v_scale);
  a.scale_page_stride = scale_page_stride;
  a.scale_head_stride = scale_head_stride;
  a.num_pages = num_pages;
  a.page_size = page_size;
  return a;
}

}  // namespace
}  // namespace mas

extern "C" int mas_append_paged_kv_cache_fp4(void* k_cache, void* v_cache, int64_t page_stride, int64_t entry_stride,
                                             int64_t head_stride, void* k_scale, void* v_scale,
                                             int64_t scale_page_stride, int64_t scale_head_stride, int64_t num_pages,
                                             int64_t page_size, const void* key, int64_t key_stride,
                                             int64_t key_head_stride, const void* value, int64_t value_stride,
                                             int64_t value_head_stride, const int32_t* batch_indices,
                                             const int32_t* positions, const int32_t* kv_indices, int64_t num_indices,
                                             const int32_t* kv_indptr, int64_t batch, int64_t rows, int64_t num_heads,
                                             int64_t head_dim, uint32_t* err, hipStream_t stream) {
  using namespace mas;
  Fp4Args a = cache_args(k_cache, v_cache, page_stride, entry_stride, head_stride, k_scale, v_scale,
                         scale_page_stride, scale_head_stride, num_pages, page_size);
  a.key = static_cast<uint16_t*>(const_cast<void*>(key));
  a.key_stride = key_stride;
  a.key_head_stride = key_head_stride;
  a.value = static_cast<uint16_t*>(const_cast<void*>(value));
  a.value_stride = value_stride;
  a.value_head_stride = value_head_stride;
  a.batch_indices = batch_indices;
  a.positions = positions;
  a.kv_indices = kv_indices;
  a.num_indices = num_indices;
  a.kv_indptr = kv_indptr;
  a.batch = batch;
  a.rows = rows;
  a.err = err;
  bool empty = false;
  if (const int st = check_rows(a, num_heads, head_dim, &empty); st != MAS_OK || empty) return st;
  if (batch_indices == nullptr || positions == nullptr || kv_indptr == nullptr || batch < 0 || num_indices < 0 ||
      (num_indices > 0 && kv_indices == nullptr))
    return MAS_ERR_INVALID_VALUE;
  return launch_rows(Move::kAppend, a, stream);
}

namespace mas {
namespace {
// The slot forms: rows into the cache, or out of it.
int by_slots(bool store, Fp4Args a, void* key, int64_t key_stride, int64_t key_head_stride, void* value,
             int64_t value_stride, int64_t value_head_stride, const int64_t* slot_mapping, int64_t rows,
             int64_t num_heads, int64_t head_dim, uint32_t* err, hipStream_t stream) {
  a.key = static_cast<uint16_t*>(key);
  a.key_stride = key_stride;
  a.key_head_stride = key_head_stride;
  a.value = static_cast<uint16_t*>(value);
  a.value_stride = value_stride;
  a.value_head_stride = value_head_stride;
  a.slots = slot_mapping;
  a.rows = rows;
  a.err = err;
  bool empty = false;
  if (const int st = check_rows(a, num_heads, head_dim, &empty); st != MAS_OK || empty) return st;
  if (slot_mapping == nullptr) return MAS_ERR_INVALID_VALUE;
  return launch_rows(store ? Move::kStore : Move::kLoad, a, stream);
}
}  // namespace
}  // namespace mas

extern "C" int mas_store_kv_slots_fp4(void* k_cache, void* v_cache, int64_t page_stride, int64_t entry_stride,
                                      int64_t head_stride, void* k_scale, void* v_scale, int64_t scale_page_stride,
                                      int64_t scale_head_stride, int64_t num_pages, int64_t page_size, const void* key,
                                      int64_t key_stride, int64_t key_head_stride, const void* value,
                                      int64_t value_stride, int64_t value_head_stride, const int64_t* slot_mapping,
                                      int64_t rows, int64_t num_heads, int64_t head_dim, uint32_t* err,
                                      hipStream_t stream) {
  using namespace mas;
  return by_slots(true,
                  cache_args(k_cache, v_cache, page_stride, entry_stride, head_stride, k_scale, v_scale,
                             scale_page_stride, scale_head_stride, num_pages, page_size),
                  const_cast<void*>(key), key_stride, key_head_stride, const_cast<void*>(value), value_stride,
                  value_head_stride, slot_mapping, rows, num_heads, head_dim, err, stream);
}

extern "C" int mas_load_kv_slots_fp4(void* key, int64_t key_stride, int64_t key_head_stride, void* value,
                                     int64_t value_stride, int64_t value_head_stride, const void* k_cache,
                                     const void* v_cache, int64_t page_stride, int64_t entry_stride,
                                     int64_t head_stride, const void* k_scale, const void* v_scale,
                                     int64_t scale_page_stride, int64_t scale_head_stride, int64_t num_pages,
                                     int64_t page_size, const int64_t* slot_mapping, int64_t rows, int64_t num_heads,
                                     int64_t head_dim, uint32_t* err, hipStream_t stream) {
  using namespace mas;
  return by_slots(false,
                  cache_args(const_cast<void*>(k_cache), const_cast<void*>(v_cache), page_stride, entry_stride,
                             head_stride, const_cast<void*>(k_scale), const_cast<void*>(v_scale), scale_page_stride,
                             scale_head_stride, num_pages, page_size),
                  key, key_stride, key_head_stride, value, value_stride, value_head_stride, slot_mapping, rows,
                  num_heads, head_dim, err, stream);
}
