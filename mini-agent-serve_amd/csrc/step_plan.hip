// step_plan.hip - a step's index tensors from its rows' lengths, on the device.
//
// What the reference's runner fills on the host for every step (ModelRunner.prepare,
// miniagentserve/engine/model_runner.py:176-225) and its block manager hands it pages for
// (miniagentserve/engine/block_manager.py:43-73). Row r holds c_r positions and gets n_r new tokens, rows in order:
//   cu_seqlens_q[r + 1] = sum of n_0 .. n_r,  seq_lens[r] = c_r + n_r;
//   token t of row r (cu[r] <= t < cu[r + 1]): position p = c_r + t - cu[r], batch index r,
//     slot = page * page_size + p % page_size with page = block_tables[r, p / page_size];
//   the pages of blocks ceil(c_r / page_size) .. ceil((c_r + n_r) / page_size) - 1 are taken from the free ring
//     in row order and written to the row's block table.
// Rows are served as long as the free pages and the token count reach: from the first row that does not fit
// on, rows get no token (MAS_ERRBIT_POOL). A row with a negative length or one past its table is passed over
// (MAS_ERRBIT_POSITION).
//
// One thread per token, and every workgroup sums the rows' tokens and pages itself, 256 rows at a time (a row
// per thread, both sums in one pass of wavefront scans), until its own tokens are covered: no workgroup
// waits for another, and one launch does it. What bounds it: the latencies of the lengths, the page and the stores.
// 256 decode rows 3.2 us, 64 decode rows and 8 prompts (8384 tokens) 4.1 us; with 64-bit shuffled scans, four barriers and
// a search for every token 4.4 and 5.1 us.
#include <type_traits>

#include "device.h"

namespace mas {
namespace {

constexpr int kPlanBlock = 256;
constexpr int kPlanWaves = kPlanBlock / kWave;

struct StepArgs {
  int32_t* positions;
  int32_t* batch_indices;
  int64_t* slots;
  int32_t* cu;
  int32_t* seq_lens;
  int64_t* range_out;
  int32_t* tables;
  int64_t bt_stride, max_blocks;
  const int32_t* new_lens;
  const int32_t* cached_lens;
  int64_t rows;
  const int32_t* free_pages;
  int64_t ring;
  const int64_t* range;
  int64_t page_size, num_tokens;
  int log2_page;  // -1: page_size is no power of two
  uint32_t* err;
};

// Sums stop at 2^32 - 1, which is more than any count of tokens or pages that is served.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
// Inclusive scan over the wavefront: by DPP within rows of 16 lanes, then the rows' totals.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {
  const auto from = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = add_sat(v, from(v, std::integral_constant<int, 0x111>{}));  // row_shr 1, 2, 4, 8
  v = add_sat(v, from(v, std::integral_constant<int, 0x112>{}));
  v = add_sat(v, from(v, std::integral_constant<int, 0x114>{}));
  v = add_sat(v, from(v, std::integral_constant<int, 0x118>{}));
  const auto total = [&](int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l)); };
  const uint32_t r0 = total(15), r1 = add_sat(r0, total(31)), r2 = add_sat(r1, total(47));
  return add_sat(v, lane < 16 ? 0u : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}

__global__ __launch_bounds__(kPlanBlock) void plan_step(StepArgs a) {
  __shared__ uint32_t sums[2][2][kPlanWaves];            // (256 rows' parity) the wavefronts' tokens and pages
  __shared__ uint32_t tops[2][kPlanWaves];               // what they serve of them
  __shared__ int all[kPlanWaves];                        // whether that is all
  __shared__ int ends[kPlanBlock];                       // token past the row's last one
  __shared__ int row_new[kPlanBlock], row_cached[kPlanBlock], row_page[kPlanBlock];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kPlanBlock + tid;
  const int64_t last_t = min(static_cast<int64_t>(blockIdx.x + 1) * kPlanBlock, a.num_tokens);
  const bool writer = blockIdx.x == 0;  // of the rows' outputs
  const int64_t head = a.range[0], tail = a.range[1];
  const uint32_t avail = static_cast<uint32_t>(head < 0 || tail < head ? 0 : min(tail - head, a.ring));
  const uint32_t most = static_cast<uint32_t>(a.num_tokens);
  // (a 64-bit remainder takes a few hundred cycles)
  const int64_t head_at = a.ring <= 0 || head < 0 ? 0
                          : head <= UINT32_MAX    ? static_cast<uint32_t>(head) % static_cast<uint32_t>(a.ring)
                                                  : head % a.ring;
  const int64_t reach = a.max_blocks * a.page_size;
  const uint32_t ps = static_cast<uint32_t>(a.page_size);
  const auto pages_of = [&](uint32_t x) { return a.log2_page >= 0 ? x >> a.log2_page : x / ps; };

  uint32_t tokens = 0, pages = 0;  // of the rows served so far
  bool open = true, found = false;
  uint32_t bits = 0;
  int parity = 0;
  for (int64_t base = 0; base < a.rows; base += kPlanBlock, parity ^= 1) {
    const int64_t row = base + tid;
    const bool in = row < a.rows;
    const int64_t n_raw = in ? a.new_lens[row] : 0, c = in ? a.cached_lens[row] : 0;
    const bool valid = n_raw >= 0 && c >= 0 && c + n_raw <= reach;
    const uint32_t n = valid ? static_cast<uint32_t>(n_raw) : 0u;
    // (a valid row's lengths are at most 2^30)
    const uint32_t have = valid ? pages_of(static_cast<uint32_t>(c) + ps - 1) : 0u;
    const uint32_t need = valid ? pages_of(static_cast<uint32_t>(c) + n + ps - 1) - have : 0u;
    uint32_t tok = wave_scan(n, lane), pag = wave_scan(need, lane);
    if (lane == kWave - 1) {
      sums[parity][0][wave] = tok;
      sums[parity][1][wave] = pag;
    }
    __syncthreads();  // (and the previous 256 rows' shared values are read)
    uint32_t tok0 = tokens, pag0 = pages;
#pragma unroll
    for (int w = 0; w < kPlanWaves - 1; ++w)
      if (w < wave) {
        tok0 = add_sat(tok0, sums[parity][0][w]);
        pag0 = add_sat(pag0, sums[parity][1][w]);
      }
    tok = add_sat(tok, tok0);
    pag = add_sat(pag, pag0);
    // (the sums grow with the row, so the rows served are the first ones)
    const bool served = open && tok <= most && pag <= avail;
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(served);
    const int last = 63 - __builtin_clzll(lanes | 1);
    const int top_tok = __builtin_amdgcn_readlane(static_cast<int>(tok), last);
    const int top_pag = __builtin_amdgcn_readlane(static_cast<int>(pag), last);
    if (lane == 0) {
      tops[0][wave] = lanes != 0 ? top_tok : 0;
      tops[1][wave] = lanes != 0 ? top_pag : 0;
      all[wave] = lanes == ~uint64_t{0};
    }
    row_new[tid] = served ? static_cast<int>(n) : 0;
    row_cached[tid] = static_cast<int>(c);
    row_page[tid] = static_cast<int>(served ? pag - need : 0);
    ends[tid] = served ? static_cast<int>(tok) : INT32_MAX;  // (no token of these rows comes so far)
    __syncthreads();
    const uint32_t before = tokens;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      tokens = max(tokens, tops[0][w]);
      pages = max(pages, tops[1][w]);
      open = open && all[w] != 0;
    }
    if (writer && in) {
      a.cu[row + 1] = static_cast<int32_t>(served ? tok : tokens);
      a.seq_lens[row] = static_cast<int32_t>(c + (served ? n : 0));
      if (!valid) bits |= MAS_ERRBIT_POSITION;
      else if (!served && n > 0) bits |= MAS_ERRBIT_POOL;
    }
    if (t >= before && t < tokens) {  // this thread's token lies in these rows
      found = true;
      // the first row whose end is past t: among decode rows, a token each, row t - before; else by halving
      int lo = static_cast<int>(min(t - before, static_cast<int64_t>(kPlanBlock - 1))), hi = lo;
      if (ends[lo] <= t || (lo > 0 && ends[lo - 1] > t)) {
        lo = 0;
        hi = kPlanBlock - 1;
      }
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int64_t r = base + lo;
      const uint32_t cached = static_cast<uint32_t>(row_cached[lo]);
      const uint32_t pos = cached + static_cast<uint32_t>(static_cast<int>(t) - (ends[lo] - row_new[lo]));
      const uint32_t first = pages_of(cached + ps - 1), block = pages_of(pos), entry = pos - block * ps;
      int32_t* const table = a.tables + r * a.bt_stride;
      int32_t page;
      if (block < first) {
        page = table[block];
      } else {
        int64_t at = head_at + row_page[lo] + (block - first);
        if (at >= a.ring) at -= a.ring;
        page = a.free_pages[at];
        if (entry == 0) table[block] = page;
      }
      a.positions[t] = static_cast<int32_t>(pos);
      a.batch_indices[t] = static_cast<int32_t>(r);
      a.slots[t] = page < 0 ? -1 : static_cast<int64_t>(page) * a.page_size + entry;
      if (page < 0) report(a.err, MAS_ERRBIT_PAGE);
    }
    if (!writer && (tokens >= last_t || !open)) break;  // uniform: this workgroup's tokens are written
  }
  if (!found && t < a.num_tokens) {  // a padding token
    a.positions[t] = 0;
    a.batch_indices[t] = -1;
    a.slots[t] = -1;
  }
  if (writer) {
    if (bits != 0) report(a.err, bits);
    if (tid == 0) {
      a.cu[0] = 0;
      a.range_out[0] = head + pages;
      a.range_out[1] = tail;
    }
  }
}

}  // namespace
}  // namespace mas

extern "C" int mas_plan_step(int32_t* positions, int32_t* batch_indices, int64_t* slot_mapping, int32_t* cu_seqlens_q,
                             int32_t* seq_lens, int64_t* free_range_out, int32_t* block_tables,
                             int64_t block_table_stride, int64_t max_blocks, const int32_t* new_lens,
                             const int32_t* cached_lens, int64_t rows, const int32_t* free_pages,
                             int64_t num_free_pages, const int64_t* free_range, int64_t page_size, int64_t num_tokens,
                             uint32_t* err, hipStream_t stream) {
  using namespace mas;
  if (rows < 0 || num_tokens < 0 || page_size <= 0 || max_blocks < 0 || num_free_pages < 0)
    return MAS_ERR_INVALID_VALUE;
  if (cu_seqlens_q == nullptr || free_range == nullptr || free_range_out == nullptr || free_range == free_range_out)
    return MAS_ERR_INVALID_VALUE;
  if (rows > 0 && (new_lens == nullptr || cached_lens == nullptr || seq_lens == nullptr || seq_lens == new_lens ||
                   seq_lens == cached_lens || (max_blocks > 0 && block_tables == nullptr)))
    return MAS_ERR_INVALID_VALUE;
  if (num_tokens > 0 && (positions == nullptr || batch_indices == nullptr || slot_mapping == nullptr))
    return MAS_ERR_INVALID_VALUE;
  if (num_free_pages > 0 && free_pages == nullptr) return MAS_ERR_INVALID_VALUE;
  // positions, token counts and pages are 32-bit numbers
  if (page_size > (1 << 30) || max_blocks * page_size > (int64_t{1} << 30) || num_tokens > INT32_MAX - 1 ||
      rows > INT32_MAX - 1 || num_free_pages > INT32_MAX)
    return MAS_ERR_UNSUPPORTED;
  const StepArgs a{positions, batch_indices, slot_mapping, cu_seqlens_q, seq_lens, free_range_out, block_tables,
                   block_table_stride, max_blocks, new_lens, cached_lens, rows, free_pages, num_free_pages, free_range,
                   page_size, num_tokens, (page_size & (page_size - 1)) == 0 ? __builtin_ctzll(page_size) : -1, err};
  const int64_t blocks = num_tokens > 0 ? cdiv(num_tokens, kPlanBlock) : 1;
  hipLaunchKernelGGL(plan_step, dim3(static_cast<uint32_t>(blocks)), dim3(kPlanBlock), 0, stream, a);
  return launch_status();
}
