// fp4_cache.hip - a step's key / value rows into the 4-bit KV cache, and rows of it back.
//
// The paged append of kv_store.hip (the same two forms of destination, devstral2.py:170-173,289) with the
// rows quantized on the way (fp4.h): for each block of 32 elements of a head,
//   s = the power byte of max |x|,   code_i = e2m1(x_i / 2^(s - 127)),
// and the reverse, y_i = e2m1(code_i) 2^(s - 127) as bf16, exact, for rows named by their slots.
//
// A lane holds 8 elements (one 16-byte load), four lanes a block: its maximum is a packed 16-bit maximum over
// the magnitudes' bits and two quad permutes. One wavefront per (token, keys or values, 512 elements); like
// the bf16 store, the row's loads are issued before the destination is resolved.
#include "fp4.h"
#include "kv_dest.h"

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
  int parts;                      // wavefronts per (token, tensor)
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

// What a wavefront works on, and its lane's place in the row.
struct Place {
  int64_t t;
  bool is_v, live;
  int h, col;  // head, 8-element vector in it
};
__device__ __forceinline__ Place place_of(const Fp4Args& a) {
  const int lane = threadIdx.x & (kWave - 1);
  const unsigned per_token = 2u * static_cast<unsigned>(a.parts);
  const unsigned t = blockIdx.x / per_token, rem = blockIdx.x - t * per_token;
  const unsigned part = rem >> 1;
  const int v = static_cast<int>(part) * kWave + lane;
  const int h = v / a.vec_per_head;
  return {static_cast<int64_t>(t), (rem & 1u) != 0, v < a.vec_per_row, h, v - h * a.vec_per_head};
}

template <bool kSlotForm>
__global__ __launch_bounds__(kWave) void fp4_store(Fp4Args a) {
  const Place p = place_of(a);
  u32x4 w{};
  if (p.live) {
    const uint16_t* src = p.is_v ? a.value + p.t * a.value_stride + p.h * a.value_head_stride
                                 : a.key + p.t * a.key_stride + p.h * a.key_head_stride;
    w = load_stream(src + 8 * p.col);
  }
  load_fence();
  int64_t page = 0, entry = 0;
  if (!resolve<kSlotForm>(a, p.t, &page, &entry)) return;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max_u16x2(m, w[i] & 0x7fff7fffu);
  m = max_u16x2(m, dpp_u32<0xb1>(m));  // quad_perm [1,0,3,2]
  m = max_u16x2(m, dpp_u32<0x4e>(m));  // quad_perm [2,3,0,1]
  const uint32_t power = fp4_power(max(m & 0xffffu, m >> 16));
  const uint32_t codes = power == 255u ? 0u : fp4x8_encode(w, power);
  if (!p.live) return;
  uint8_t* dst = (p.is_v ? a.v : a.k) + page * a.page_stride + entry * a.entry_stride + p.h * a.head_stride;
  *reinterpret_cast<uint32_t*>(dst + 4 * p.col) = codes;
  if ((p.col & 3) == 0)
    (p.is_v ? a.v_scale : a.k_scale)[page * a.scale_page_stride + p.h * a.scale_head_stride +
                                     (p.col >> 2) * a.page_size + entry] = static_cast<uint8_t>(power);
}

// Rows of the cache as bf16; a slot that is negative or past the cache gives zeros.
__global__ __launch_bounds__(kWave) void fp4_load(Fp4Args a) {
  const Place p = place_of(a);
  int64_t page = 0, entry = 0;
  const bool ok = resolve<true>(a, p.t, &page, &entry);
  if (!p.live) return;
  u32x4 y{};
  if (ok) {
    const uint8_t* src = (p.is_v ? a.v : a.k) + page * a.page_stride + entry * a.entry_stride + p.h * a.head_stride;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + 4 * p.col);
    const uint32_t power = (p.is_v ? a.v_scale : a.k_scale)[page * a.scale_page_stride + p.h * a.scale_head_stride +
                                                            (p.col >> 2) * a.page_size + entry];
    y = fp4x8_decode(codes, __uint_as_float(power << 23));
  }
  uint16_t* dst = p.is_v ? a.value + p.t * a.value_stride + p.h * a.value_head_stride
                         : a.key + p.t * a.key_stride + p.h * a.key_head_stride;
  store_stream(dst + 8 * p.col, y);
}

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
  a.vec_per_head = static_cast<int>(head_dim / 8);
  a.vec_per_row = static_cast<int>(num_heads * head_dim / 8);
  a.parts = static_cast<int>(cdiv(a.vec_per_row, kWave));
  return a.rows * 2 * a.parts > INT32_MAX ? MAS_ERR_UNSUPPORTED : MAS_OK;
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
  hipLaunchKernelGGL(fp4_store<false>, dim3(static_cast<uint32_t>(rows * 2 * a.parts)), dim3(kWave), 0, stream, a);
  return launch_status();
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
  const dim3 grid(static_cast<uint32_t>(rows * 2 * a.parts));
  if (store) hipLaunchKernelGGL(fp4_store<true>, grid, dim3(kWave), 0, stream, a);
  else hipLaunchKernelGGL(fp4_load, grid, dim3(kWave), 0, stream, a);
  return launch_status();
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
