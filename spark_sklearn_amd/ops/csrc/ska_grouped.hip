// Grouped-row operators -- MI355X (gfx950, CDNA4) only.
//
// Rows that belong to groups (the keys of a keyed model, the experts of a
// routed layer): a stable sort of the rows' group ids, the rows' way into
// group order and back, and the product of each group's run of rows with
// that group's own weights.  M = T*k entries (row t has k ids); `slots` is a
// permutation of the entries, the ones without a group last, so that an
// entry is kept exactly when its slot is below offsets[G].
//
// No kernel trusts the values of offsets and slots for its addresses: an
// offset is clamped to the rows there are, a slot outside them is skipped.

#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <ATen/EmptyTensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <tuple>
#include <type_traits>

#include "ska_rows.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

hipStream_t stream_now() {
  return at::cuda::getCurrentCUDAStream().stream();
}

void check_launch() {
  hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "HIP launch failed: ", hipGetErrorString(e));
}

// Refusals, with the types and words of the reference's (grouped_rows.py).
constexpr int64_t kMaxGroups = (1 << 24) - 1;
constexpr int64_t kMaxWidth = (1 << 21) - 1;
constexpr int64_t kMaxRows = (1ll << 31) - (1 << 16) - 1;

// Whether the kernels can read a tensor: subclasses that wrap others, fake
// tensors and zeros that are only noted as such have no memory behind them,
// and what lies behind a functional tensor may be out of date.  The storage is
// looked at, since a view's pointer is not null where its storage's is, and a
// storage may have been made smaller than its tensor (freed parameters).
bool has_memory(const at::Tensor& t) {
  if (t.numel() == 0) return true;
  if (t.layout() != at::kStrided || !t.has_storage() ||
      t.key_set().has(c10::DispatchKey::Functionalize))
    return false;
  const c10::Storage& storage = t.storage();
  return storage.data() != nullptr &&
         at::detail::computeStorageNbytes(t.sizes(), t.strides(),
                                          t.itemsize(), t.storage_offset()) <=
             storage.nbytes();
}

// No address goes to a kernel but through here.  Inputs are checked on entry;
// what torch makes of them, and outputs, may still be fakes (under a mode).
template <typename T>
T* ptr(const at::Tensor& t) {
  TORCH_CHECK_TYPE(has_memory(t), "grouped-row operators take no tensors "
                   "without memory (wrappers, fake tensors)");
  return reinterpret_cast<T*>(t.data_ptr());
}

// A tensor's values as they lie in memory: a lazy negation (the imaginary part
// of a conjugate has one) is carried out.
at::Tensor as_stored(const at::Tensor& t) {
  return t.is_neg() ? t.resolve_neg() : t;
}

at::Tensor whole(const at::Tensor& t) { return as_stored(t).contiguous(); }

// The kernels have no forward-mode derivatives, and a tensor that came back
// without its tangent would pass for a constant.  (A meta tensor is on another
// device, which the checks of devices say.)
void check_plain(const char* name, const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.is_meta() || has_memory(t), name,
                   " must be a tensor with memory of its own (no wrapper or "
                   "fake tensor, dense)");
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), name,
                              " has a tangent: grouped-row operators have no "
                              "forward-mode derivatives");
}

// A trace would record the allocations of the outputs and not the kernels.
void check_not_traced() {
  TORCH_CHECK(!torch::jit::tracer::isTracing(),
              "grouped-row operators cannot be traced on a GPU");
}

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  return (float)v;
}

__device__ __forceinline__ int clampi(int v, int lo, int hi) {
  return v < lo ? lo : (v > hi ? hi : v);
}

// ---------------------------------------------------------------------------
// group_rows: a stable counting sort by id.  An id outside [0, G) is the key
// G, so that such entries come last, in their own order.
// ---------------------------------------------------------------------------
template <typename I>
__device__ __forceinline__ int key_of(I id, int G) {
  return (id < 0 || id >= (I)G) ? G : (int)id;
}

constexpr int kSmallEntries = 2048;
constexpr int kSmallGroups = 65536;

// LDS accesses before and after it keep their order within the wave.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Few entries: one block sorts key * 2048 + entry, which makes the order
// stable, in LDS: compare and exchange at distances of halves.  Distances
// up to 64 stay within a wave, where no barrier is needed.  (Comparing each of
// 2012 entries with every other took 158 us.)
template <typename I>
__global__ __launch_bounds__(1024) void sort_small_kernel(
    const I* __restrict__ ids, int M, int G, int size,
    int* __restrict__ offsets, int* __restrict__ slots,
    int* __restrict__ order) {
  static_assert((kSmallGroups + 1l) * kSmallEntries < (1l << 32));
  __shared__ unsigned item[kSmallEntries];
  const int tid = threadIdx.x, threads = blockDim.x;
  for (int i = tid; i < size; i += threads)
    item[i] = i < M ? (unsigned)key_of<I>(ids[i], G) * kSmallEntries + i
                    : 0xffffffffu;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int d = run / 2; d > 0; d /= 2) {
      for (int t = tid; t < size / 2; t += threads) {
        // the pair of elements d apart that thread t owns
        const int a = (t & -d) * 2 + (t & (d - 1)), b = a + d;
        const unsigned x = item[a], y = item[b];
        const bool up = (a & run) == 0;
        if ((x > y) == up) {
          item[a] = y;
          item[b] = x;
        }
      }
      // a wave's 64 threads own 128 neighbouring elements while d <= 64
      if (d > 64 || (d == 1 && run >= 64))
        __syncthreads();
      else
        wave_fence();
    }
  __syncthreads();
  for (int i = tid; i < M; i += threads) {
    const int entry = item[i] & (kSmallEntries - 1);
    order[i] = entry;
    slots[entry] = i;
  }
  for (int g = tid; g <= G; g += threads)
    offsets[g] = ska::lower_bound(item, M, (unsigned)g * kSmallEntries);
}

// Many entries: passes over a digit of the key, low digit first.  One pass
// sorts up to kBins keys; more groups take two.  A pass counts each block's
// digits, sums the counts over the blocks before it, and places the entries.
// No atomic decides an order, so that the sort is stable.  10^6 entries take
// 32 us for 64 groups and 50 for 4096 (10 and 23 us of it counting and
// placing); what bounds it is the chain of LDS accesses of 64 entries after
// the other, and 4-byte stores to places apart.
constexpr int kBins = 8192;
constexpr int kSortWaves = 4;

template <typename I, bool FIRST>
__device__ __forceinline__ int sort_key(const I* ids, const int* keys, int G,
                                        int i) {
  return FIRST ? key_of<I>(ids[i], G) : keys[i];
}

// Keys first .. last - 1, STEP lanes side by side and four reads under way.
template <typename I, bool FIRST, int STEP, typename Do>
__device__ __forceinline__ void sort_walk(const I* ids, const int* keys, int G,
                                          long first, long last, int lane,
                                          Do work) {
  for (long i0 = first; i0 < last; i0 += 4 * STEP) {
    int key[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long i = i0 + u * STEP + lane;
      key[u] = i < last ? sort_key<I, FIRST>(ids, keys, G, (int)i) : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long i = i0 + u * STEP + lane;
      work(i, key[u], i < last);
    }
  }
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(
    const I* __restrict__ ids, const int* __restrict__ keys, int M, int G,
    int shift, int mask, int bins, int tile, int blocks,
    int* __restrict__ table) {
  extern __shared__ int count[];
  for (int b = threadIdx.x; b < bins; b += 256) count[b] = 0;
  __syncthreads();
  const long first = (long)blockIdx.x * tile;
  const int last = (int)min(first + tile, (long)M);
  sort_walk<I, FIRST, 256>(ids, keys, G, first, last, threadIdx.x,
                           [&](long, int key, bool in) {
                             const int digit = (key >> shift) & mask;
                             if (in) atomicAdd(&count[digit], 1);
                           });
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 256)
    table[(long)blockIdx.x * bins + b] = count[b];
}

__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// A bin's counts in the blocks first .. last - 1 become their running sums from
// `at` on, 16 of them under way at a time (one by one, a read behind each
// write, 48 blocks took 7 us, so 4).
__device__ __forceinline__ int scan_column(int* column, long bins, int first,
                                           int last, int at) {
  for (int b0 = first; b0 < last; b0 += 16) {
    int n[16];
#pragma unroll
    for (int u = 0; u < 16; ++u)
      n[u] = b0 + u < last ? column[(b0 + u) * bins] : 0;
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      if (b0 + u < last) column[(b0 + u) * bins] = at;
      at += n[u];
    }
  }
  return at;
}

// A bin's counts become the numbers of such entries in the blocks before, and
// total[bin] their sum.  64 bins a block, whose 16 waves share the blocks (10^6
// entries, 4096 groups: 11 us with 4 waves, 7 with 16).
__global__ __launch_bounds__(1024) void sort_scan_kernel(
    int bins, int blocks, int* __restrict__ table, int* __restrict__ total) {
  __shared__ int sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bin = blockIdx.x * 64 + lane;
  const int part = (blocks + 15) / 16;
  const int first = wave * part, last = min(blocks, first + part);
  int sum = 0;
  if (bin < bins) {
#pragma unroll 16
    for (int b = first; b < last; ++b) sum += table[(long)b * bins + bin];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < wave; ++w) at += sums[w][lane];
  if (bin >= bins) return;
  if (wave == 15) total[bin] = at + sum;
  scan_column(table + bin, bins, first, last, at);
}

// The bins' first positions; where one pass sorts, these are the offsets.  A
// thread has up to 8 neighbouring bins.
__global__ __launch_bounds__(1024) void sort_base_kernel(
    int bins, const int* __restrict__ total, int* __restrict__ base) {
  constexpr int kOwn = kBins / 1024;
  __shared__ int wave_sum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int own[kOwn], sum = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int b = tid * kOwn + i;
    own[i] = b < bins ? total[b] : 0;
    sum += own[i];
  }
  const int s = wave_scan(sum, lane);
  if (lane == 63) wave_sum[wave] = s;
  __syncthreads();
  int at = s - sum;
  for (int w = 0; w < wave; ++w) at += wave_sum[w];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int b = tid * kOwn + i;
    if (b < bins) base[b] = at;
    at += own[i];
  }
}

// Both of these at once, for up to 1024 bins and few blocks.
constexpr int kFewBlocks = 64;
__global__ __launch_bounds__(1024) void sort_scan_few_kernel(
    int bins, int blocks, int* __restrict__ table, int* __restrict__ base) {
  __shared__ int wave_sum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int sum = 0;
  if (tid < bins) sum = scan_column(table + tid, bins, 0, blocks, 0);
  const int s = wave_scan(sum, lane);
  if (lane == 63) wave_sum[wave] = s;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += wave_sum[w];
  if (tid < bins) base[tid] = before + s - sum;
}

// Places a block's entries: each wave owns a contiguous part of the block's
// tile and a row of counters.  Among 64 entries a lane's place is the number
// of lower lanes with its digit.
template <typename I, bool FIRST, bool LAST>
__global__ __launch_bounds__(256) void sort_place_kernel(
    const I* __restrict__ ids, const int* __restrict__ keys,
    const int* __restrict__ entries, int M, int G, int shift, int mask,
    int bits, int bins, int tile, int blocks, const int* __restrict__ table,
    const int* __restrict__ base, int* __restrict__ keys_out,
    int* __restrict__ order, int* __restrict__ slots) {
  extern __shared__ int place[];  // [kSortWaves][bins]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = threadIdx.x; b < bins * kSortWaves; b += 256) place[b] = 0;
  __syncthreads();
  const int part = tile / kSortWaves;
  const long first = (long)blockIdx.x * tile + (long)wave * part;
  const long last = min(first + part, (long)M);
  int* mine = place + wave * bins;
  sort_walk<I, FIRST, 64>(ids, keys, G, first, last, lane,
                          [&](long, int key, bool in) {
                            const int digit = (key >> shift) & mask;
                            if (in) atomicAdd(&mine[digit], 1);
                          });
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 256) {
    int at = base[b] + table[(long)blockIdx.x * bins + b];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      int n = place[w * bins + b];
      place[w * bins + b] = at;
      at += n;
    }
  }
  __syncthreads();
  volatile int* at = mine;
  sort_walk<I, FIRST, 64>(
      ids, keys, G, first, last, lane, [&](long i, int key, bool in) {
        const int digit = (key >> shift) & mask;
        unsigned long long same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
          const bool one = (digit >> b) & 1;
          const unsigned long long set = __ballot(one);
          same &= one ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int start = in ? at[digit] : 0;
        wave_fence();
        if (in && rank == 0) at[digit] = start + __popcll(same);
        wave_fence();
        if (in) {
          const int pos = start + rank;
          const int entry = FIRST ? (int)i : entries[i];
          order[pos] = entry;
          if (!LAST || !FIRST) keys_out[pos] = key;
          if (LAST) slots[entry] = pos;
        }
      });
}

__global__ void sort_offsets_kernel(const int* __restrict__ keys, int M,
                                    int G, int* __restrict__ offsets) {
  for (long g = (long)blockIdx.x * blockDim.x + threadIdx.x; g <= G;
       g += (long)gridDim.x * blockDim.x)
    offsets[g] = ska::lower_bound(keys, M, (int)g);
}

template <typename I>
void sort_launch(const I* ids, int M, int G, int* offsets, int* slots,
                 int* order, at::TensorOptions opt) {
  hipStream_t s = stream_now();
  // us for 100 / 1000 / 2048 entries in one block, and in the passes below:
  // 64 groups 7 / 14 / 20, and 13; 4096 groups 9 / 16 / 23, and 21
  if (M <= (G < 2048 ? kSmallEntries / 2 : kSmallEntries) &&
      G <= kSmallGroups) {
    int size = 2;
    while (size < M) size *= 2;
    // size / 2 threads sort, G + 1 look up offsets
    const int threads = std::max(size / 2, std::min(1024, G + 1));
    sort_small_kernel<I><<<1, (threads + 63) / 64 * 64, 0, s>>>(
        ids, M, G, size, offsets, slots, order);
    check_launch();
    return;
  }
  int bits = 1;
  while ((G >> bits) != 0) ++bits;  // keys are 0 .. G
  // One pass has as many counters a block as groups.  us for one / two:
  // 4096 groups, 25000 entries 30 / 27, 100000 31 / 38; 6000 groups, 100000
  // 44 / 39, 300000 48 / 50; 8000 groups, 3000 entries 46 / 22
  const bool one = G + 1 <= kBins && M >= 40l * (G - 2750);
  const int digit = one ? bits : (bits + 1) / 2;
  const int mask = (1 << digit) - 1;
  const int bins = one ? G + 1 : 1 << digit;
  // 512 entries a block at least, and not fewer than half its counters; about
  // 256 blocks while these are short, and as many at most as the scan of their
  // counts is worth
  const long most = bins <= 1024 ? 4096 : 1024;
  int tile = 512;
  while (tile < bins / 2 || (tile * 256l < M && tile < 8192) ||
         tile * most < M)
    tile *= 2;
  const int blocks = (int)(((long)M + tile - 1) / tile);
  at::Tensor table = at::empty({(int64_t)bins * blocks + 2 * bins}, opt);
  int* tab = ptr<int>(table);
  int* total = tab + (long)bins * blocks;
  int* base = one ? offsets : total + bins;
  at::Tensor pairs;
  int *k0 = nullptr, *e0 = nullptr, *k1 = nullptr;
  if (!one) {
    pairs = at::empty({3 * (int64_t)M}, opt);
    k0 = ptr<int>(pairs);
    e0 = k0 + M;
    k1 = e0 + M;
  }
  const size_t lds = (size_t)bins * 4;
  auto step = [&](auto first, auto last, int shift) {
    constexpr bool F = decltype(first)::value, L = decltype(last)::value;
    sort_count_kernel<I, F><<<blocks, 256, lds, s>>>(
        ids, k0, M, G, shift, mask, bins, tile, blocks, tab);
    if (bins <= 1024 && blocks <= kFewBlocks) {
      sort_scan_few_kernel<<<1, (bins + 63) / 64 * 64, 0, s>>>(bins, blocks,
                                                               tab, base);
    } else {
      sort_scan_kernel<<<(bins + 63) / 64, 1024, 0, s>>>(bins, blocks, tab,
                                                        total);
      sort_base_kernel<<<1, 1024, 0, s>>>(bins, total, base);
    }
    sort_place_kernel<I, F, L><<<blocks, 256, lds * kSortWaves, s>>>(
        ids, k0, e0, M, G, shift, mask, digit, bins, tile, blocks, tab, base,
        L ? k1 : k0, L ? order : e0, slots);
    check_launch();
  };
  auto set_lds = [&](auto kern) {
    hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void*>(kern),
        hipFuncAttributeMaxDynamicSharedMemorySize, kBins * 4 * kSortWaves);
    TORCH_CHECK(e == hipSuccess, "HIP error: ", hipGetErrorString(e));
  };
  if (one) {
    set_lds(sort_place_kernel<I, true, true>);
    step(std::true_type{}, std::true_type{}, 0);
  } else {
    set_lds(sort_place_kernel<I, true, false>);
    set_lds(sort_place_kernel<I, false, true>);
    step(std::true_type{}, std::false_type{}, 0);
    step(std::false_type{}, std::true_type{}, digit);
    sort_offsets_kernel<<<std::min(1024, (G + 256) / 256), 256, 0, s>>>(
        k1, M, G, offsets);
    check_launch();
  }
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> group_rows(
    const at::Tensor& ids_in, int64_t n_groups) {
  check_not_traced();
  TORCH_CHECK_VALUE(ids_in.is_cuda(), "ids must be on a GPU, got ",
                    ids_in.device());
  TORCH_CHECK_TYPE(ids_in.dtype() == at::kInt || ids_in.dtype() == at::kLong,
                   "ids must be int32 or int64, got ", ids_in.dtype());
  TORCH_CHECK_VALUE(ids_in.dim() == 1 || ids_in.dim() == 2,
                    "ids must have one or two dimensions");
  TORCH_CHECK_VALUE(n_groups >= 1 && n_groups <= kMaxGroups,
                    "n_groups must be in [1, ", kMaxGroups, "], got ",
                    n_groups);
  TORCH_CHECK_VALUE(ids_in.numel() <= kMaxRows, "too many entries");
  check_plain("ids", ids_in);
  c10::cuda::CUDAGuard guard(ids_in.device());
  at::Tensor ids = whole(ids_in);
  auto opt = ids.options().dtype(at::kInt);
  const int M = (int)ids.numel(), G = (int)n_groups;
  at::Tensor slots = at::empty(ids.sizes(), opt);
  at::Tensor order = at::empty({M}, opt);
  if (M == 0) return {at::zeros({G + 1}, opt), slots, order};
  at::Tensor offsets = at::empty({G + 1}, opt);
  if (ids.dtype() == at::kInt)
    sort_launch<int>(ptr<int>(ids), M, G, ptr<int>(offsets),
                     ptr<int>(slots), ptr<int>(order), opt);
  else
    sort_launch<int64_t>(ptr<int64_t>(ids), M, G,
                         ptr<int>(offsets), ptr<int>(slots),
                         ptr<int>(order), opt);
  return {offsets, slots, order};
}

// ---------------------------------------------------------------------------
// Rows into group order and back.  `lanes` lanes (a power of two up to 64)
// share a row and walk it in vectors of 16 bytes.  Rows of an odd width
// start at odd addresses, which the loads and stores here may have; the
// elements behind the last whole vector go one by one.
// ---------------------------------------------------------------------------
// 16 bytes that may begin at any value: one load or store instruction.
typedef unsigned Bytes16 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef T Values __attribute__((ext_vector_type(16 / sizeof(T))));
  Values v;
};

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p, int n) {
  Vec<T> r;
  if (n >= Vec<T>::N) {
    r.v = __builtin_bit_cast(decltype(r.v),
                             *reinterpret_cast<const Bytes16*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& r, int n) {
  if (n >= Vec<T>::N) {
    *reinterpret_cast<Bytes16*>(p) = __builtin_bit_cast(Bytes16, r.v);
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

template <int N>
using Count = std::integral_constant<int, N>;

// A lane's share of a row of F values: `some(at, Count<U>)` for U vectors at
// `at`, `at` + step, ..., as many in flight; then `one(at)` for the values
// behind the last whole vector, a lane each.
template <int V, int U, typename Some, typename One>
__device__ __forceinline__ void walk_row(int F, int lane, int lanes,
                                         Some some, One one) {
  const int whole = F / V * V, step = lanes * V;
  int at = lane * V;
  for (; at + (U - 1) * step < whole; at += U * step) some(at, Count<U>{});
  for (; at < whole; at += step) some(at, Count<1>{});
  for (int e = whole + lane; e < F; e += lanes) one(e);
}

template <typename T>
__device__ __forceinline__ Vec<T> get(const T* p) {
  Vec<T> r;
  r.v = __builtin_bit_cast(decltype(r.v),
                           *reinterpret_cast<const Bytes16*>(p));
  return r;
}

template <typename T>
__device__ __forceinline__ void put(T* p, const Vec<T>& r) {
  *reinterpret_cast<Bytes16*>(p) = __builtin_bit_cast(Bytes16, r.v);
}

// In row order, so that a row is read once for its k places.  Bound by memory:
// 10^6 rows of 256 float32 move in 365 us (5.6 TB/s, where a copy of that size
// has 5.4).  Loads that the compiler took apart into pieces of 2 bytes, because
// the values' type was an array, had 3.1.
template <typename T, int U>
__global__ __launch_bounds__(256) void gather_kernel(
    const T* __restrict__ x, long x_pitch, const int* __restrict__ slots,
    const int* __restrict__ kept_end, int T_rows, int k, int F, int lanes,
    T* __restrict__ out) {
  constexpr int V = Vec<T>::N;
  const int per = 256 / lanes;
  const int M = T_rows * k;
  const int S = clampi(*kept_end, 0, M);
  const int step = lanes * V;
  for (long t = (long)blockIdx.x * per + threadIdx.x / lanes; t < T_rows;
       t += (long)gridDim.x * per) {
    const T* src = x + t * x_pitch;
    walk_row<V, U>(
        F, threadIdx.x % lanes, lanes,
        [&](int at, auto n) {
          constexpr int N = decltype(n)::value;
          Vec<T> v[N];
#pragma unroll
          for (int u = 0; u < N; ++u) v[u] = get(src + at + u * step);
          for (int j = 0; j < k; ++j) {
            const int s = slots[t * k + j];
            if ((unsigned)s >= (unsigned)M) continue;
            T* to = out + (long)s * F + at;
#pragma unroll
            for (int u = 0; u < N; ++u) {
              Vec<T> w = v[u];
              if (s >= S) w.v = (T)0.f;
              put(to + u * step, w);
            }
          }
        },
        [&](int at) {
          const T v = src[at];
          for (int j = 0; j < k; ++j) {
            const int s = slots[t * k + j];
            if ((unsigned)s < (unsigned)M)
              out[(long)s * F + at] = s < S ? v : (T)0.f;
          }
        });
  }
}

// y[t] = sum over the kept entries of w[t, j] * rows[slots[t, j]], in the
// order of j and in 32 bits, rounded once; J rows are read at a time.
template <typename T, typename W, int J, int U>
__global__ __launch_bounds__(256) void combine_kernel(
    const T* __restrict__ rows, long pitch, const int* __restrict__ slots,
    const int* __restrict__ kept_end, const W* __restrict__ weights,
    int T_rows, int k, int F, int lanes, T* __restrict__ y) {
  constexpr int V = Vec<T>::N;
  const int per = 256 / lanes;
  const int S = clampi(*kept_end, 0, T_rows * k);
  const int step = lanes * V;
  for (long t = (long)blockIdx.x * per + threadIdx.x / lanes; t < T_rows;
       t += (long)gridDim.x * per) {
    walk_row<V, U>(
        F, threadIdx.x % lanes, lanes,
        [&](int at, auto n) {
          constexpr int N = decltype(n)::value;
          float acc[N][V] = {};
          for (int j0 = 0; j0 < k; j0 += J) {
            bool kept[J];
            float w[J];
            Vec<T> v[J][N];
#pragma unroll
            for (int j = 0; j < J; ++j) {
              const long e = t * k + j0 + j;
              const int s = j0 + j < k ? slots[e] : -1;
              kept[j] = (unsigned)s < (unsigned)S;
              w[j] = kept[j] && weights ? (float)weights[e] : 1.f;
              // an entry that is left out reads the first row, for nothing
              const T* src = rows + (kept[j] ? (long)s * pitch : 0) + at;
#pragma unroll
              for (int u = 0; u < N; ++u) v[j][u] = get(src + u * step);
            }
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
              for (int u = 0; u < N; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                  const float next = acc[u][i] + w[j] * to_f(v[j][u].v[i]);
                  acc[u][i] = kept[j] ? next : acc[u][i];
                }
          }
#pragma unroll
          for (int u = 0; u < N; ++u) {
            Vec<T> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = (T)acc[u][i];
            put(y + t * F + at + u * step, o);
          }
        },
        [&](int at) {
          float acc = 0.f;
          for (int j = 0; j < k; ++j) {
            const int s = slots[t * k + j];
            if ((unsigned)s >= (unsigned)S) continue;
            const float w = weights ? (float)weights[t * k + j] : 1.f;
            acc += w * to_f(rows[(long)s * pitch + at]);
          }
          y[t * F + at] = (T)acc;
        });
  }
}

// Backward of combine, in row order: dy[t] is read once for J rows, each row
// once; drows (where asked for) and the dot products leave with them.  Bound by
// memory: 8191 x 2 rows of 1001 float16 take 20 us (4.1 TB/s).  The products
// w * dy are rounded to the rows' type, the type that a gradient of rows has.
template <typename T, typename W, int J, int U>
__global__ __launch_bounds__(256) void combine_back_kernel(
    const T* __restrict__ dy, long dy_pitch, const T* __restrict__ rows,
    long pitch, const int* __restrict__ slots,
    const int* __restrict__ kept_end, const W* __restrict__ weights,
    int T_rows, int k, int F, int lanes, T* __restrict__ drows,
    W* __restrict__ dw) {
  constexpr int V = Vec<T>::N;
  const int per = 256 / lanes;
  const int M = T_rows * k;
  const int S = clampi(*kept_end, 0, M);
  const int lane = threadIdx.x % lanes;
  const int step = lanes * V;
  for (long t0 = (long)blockIdx.x * per; t0 < T_rows;
       t0 += (long)gridDim.x * per) {
    const long t = t0 + threadIdx.x / lanes;
    const bool in = t < T_rows;
    for (int j0 = 0; j0 < k; j0 += J) {
      int s[J];
      float w[J], dot[J] = {};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        s[j] = in && j0 + j < k ? slots[t * k + j0 + j] : -1;
        w[j] = 1.f;
        if (weights && (unsigned)s[j] < (unsigned)S)
          w[j] = (float)weights[t * k + j0 + j];
      }
      if (in)
        walk_row<V, U>(
            F, lane, lanes,
            [&](int at, auto n) {
              constexpr int N = decltype(n)::value;
              Vec<T> d[N], r[J][N];
#pragma unroll
              for (int u = 0; u < N; ++u)
                d[u] = get(dy + t * dy_pitch + at + u * step);
              if (dw) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                  const bool kept = (unsigned)s[j] < (unsigned)S;
                  const T* src = rows + (kept ? (long)s[j] * pitch : 0) + at;
#pragma unroll
                  for (int u = 0; u < N; ++u) r[j][u] = get(src + u * step);
                }
              }
#pragma unroll
              for (int j = 0; j < J; ++j) {
                if ((unsigned)s[j] >= (unsigned)M) continue;
                const bool kept = s[j] < S;
#pragma unroll
                for (int u = 0; u < N; ++u) {
                  if (dw && kept) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                      dot[j] += to_f(d[u].v[i]) * to_f(r[j][u].v[i]);
                  }
                  if (drows) {
                    Vec<T> o;
#pragma unroll
                    for (int i = 0; i < V; ++i)
                      o.v[i] = kept ? (T)(w[j] * to_f(d[u].v[i])) : (T)0.f;
                    put(drows + (long)s[j] * F + at + u * step, o);
                  }
                }
              }
            },
            [&](int at) {
              const float d = to_f(dy[t * dy_pitch + at]);
#pragma unroll
              for (int j = 0; j < J; ++j) {
                if ((unsigned)s[j] >= (unsigned)M) continue;
                const bool kept = s[j] < S;
                if (dw && kept)
                  dot[j] += d * to_f(rows[(long)s[j] * pitch + at]);
                if (drows)
                  drows[(long)s[j] * F + at] = kept ? (T)(w[j] * d) : (T)0.f;
              }
            });
      if (dw) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          for (int d = lanes >> 1; d > 0; d >>= 1)
            dot[j] += __shfl_xor(dot[j], d);
          if (in && lane == 0 && j0 + j < k) dw[t * k + j0 + j] = (W)dot[j];
        }
      }
    }
  }
}

int lanes_for(int F, int vec) {
  int lanes = 1;
  while (lanes < 64 && lanes * vec < F) lanes *= 2;
  return lanes;
}

#define SKA_TYPES(dtype, ...)                                             \
  [&] {                                                                   \
    if ((dtype) == at::kFloat) {                                          \
      using T = float;                                                    \
      return __VA_ARGS__();                                               \
    }                                                                     \
    if ((dtype) == at::kBFloat16) {                                       \
      using T = __bf16;                                                   \
      return __VA_ARGS__();                                               \
    }                                                                     \
    if ((dtype) == at::kHalf) {                                           \
      using T = _Float16;                                                 \
      return __VA_ARGS__();                                               \
    }                                                                     \
    TORCH_CHECK(false, "rows must be float32, bfloat16 or float16");      \
  }()

unsigned row_blocks(long rows, int per) {
  return (unsigned)std::min<long>((rows + per - 1) / per, 1 << 22);
}

// A matrix whose rows may lie apart but are contiguous in themselves.
at::Tensor packed_rows(const at::Tensor& t_in) {
  const at::Tensor t = as_stored(t_in);
  if (t.size(0) == 0 || t.size(1) == 0) return t;
  // the product kernels' offsets in a tile of 256 rows pass no 31 bits
  const bool fits =
      (t.size(1) == 1 || t.stride(1) == 1) &&
      (t.size(0) == 1 ||
       (t.stride(0) >= t.size(1) && t.stride(0) < (1 << 22)));
  return fits ? t : t.contiguous();
}

void check_rows(const char* name, const at::Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be on a GPU, got ", t.device());
  check_plain(name, t);
  TORCH_CHECK_TYPE(t.dtype() == at::kFloat || t.dtype() == at::kBFloat16 ||
                       t.dtype() == at::kHalf,
                   name, " must be float32, bfloat16 or float16, got ",
                   t.dtype());
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must be a matrix, got shape ",
                    t.sizes());
  TORCH_CHECK_VALUE(t.size(1) <= kMaxWidth, name, " must have at most ",
                    kMaxWidth, " columns");
  TORCH_CHECK_VALUE(t.size(0) <= kMaxRows, name, " has too many rows");
}

void check_ints(const char* name, const at::Tensor& t,
                const at::Tensor& rows) {
  check_plain(name, t);
  TORCH_CHECK_TYPE(t.dtype() == at::kInt, name, " must be int32, got ",
                   t.dtype());
  TORCH_CHECK_VALUE(t.device() == rows.device(), name, " is on ", t.device(),
                    ", the rows are on ", rows.device());
}

void check_same(const char* name, const at::Tensor& t,
                const at::Tensor& rows) {
  check_plain(name, t);
  TORCH_CHECK_TYPE(t.dtype() == rows.dtype(), name, " must be ", rows.dtype(),
                   " like the rows, got ", t.dtype());
  TORCH_CHECK_VALUE(t.device() == rows.device(), name, " is on ", t.device(),
                    ", the rows on ", rows.device());
}

struct Plan {
  at::Tensor offsets, slots;  // [G + 1], [T, k]
};

Plan check_plan(const at::Tensor& rows, const at::Tensor& offsets,
                const at::Tensor& slots) {
  check_ints("plan.offsets", offsets, rows);
  check_ints("plan.slots", slots, rows);
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 2,
                    "plan.offsets must have n_groups + 1 values");
  TORCH_CHECK_VALUE(slots.dim() == 1 || slots.dim() == 2,
                    "plan.slots must have one or two dimensions");
  TORCH_CHECK_VALUE(slots.numel() <= kMaxRows, "too many entries");
  return {whole(offsets),
          whole(slots.dim() == 1 ? slots.unsqueeze(1) : slots)};
}

at::Tensor gather_rows(const at::Tensor& x_in, const at::Tensor& offsets,
                       const at::Tensor& slots) {
  c10::cuda::CUDAGuard guard(x_in.device());
  at::Tensor x = packed_rows(x_in);
  const int T_rows = (int)x.size(0), F = (int)x.size(1);
  const int k = (int)slots.size(1);
  at::Tensor out = at::empty({(int64_t)T_rows * k, F}, x.options());
  if (out.numel() == 0) return out;
  SKA_TYPES(x.scalar_type(), [&] {
    const int lanes = lanes_for(F, Vec<T>::N), per = 256 / lanes;
    gather_kernel<T, 4><<<row_blocks(T_rows, per), 256, 0, stream_now()>>>(
        ptr<T>(x), x.stride(0), ptr<int>(slots),
        ptr<int>(offsets) + offsets.numel() - 1, T_rows, k, F, lanes,
        ptr<T>(out));
    check_launch();
  });
  return out;
}

at::Tensor combine_rows(const at::Tensor& rows_in, const at::Tensor& offsets,
                        const at::Tensor& slots,
                        const c10::optional<at::Tensor>& weights) {
  c10::cuda::CUDAGuard guard(rows_in.device());
  at::Tensor rows = packed_rows(rows_in);
  const int T_rows = (int)slots.size(0), k = (int)slots.size(1);
  const int F = (int)rows.size(1);
  at::Tensor y = at::empty({T_rows, F}, rows.options());
  if (y.numel() == 0) return y;
  if (k == 0) return y.zero_();
  SKA_TYPES(rows.scalar_type(), [&] {
    const int lanes = lanes_for(F, Vec<T>::N), per = 256 / lanes;
    const int* end = ptr<int>(offsets) + offsets.numel() - 1;
    auto go = [&](auto kern, auto* w) {
      kern<<<row_blocks(T_rows, per), 256, 0, stream_now()>>>(
          ptr<T>(rows), rows.stride(0), ptr<int>(slots), end, w, T_rows,
          k, F, lanes, ptr<T>(y));
      check_launch();
    };
    auto pick = [&](auto* w) {
      using W = std::decay_t<decltype(*w)>;
      // two rows at a time, and four vectors of each where a lane has so
      // many: 16384 x 4 rows of 2048 bfloat16 take 68 us so (4.9 TB/s; 83
      // with two vectors), 32768 x 2 rows of 1024 take 35 (52 with four)
      const bool wide = F / Vec<T>::N >= 4 * lanes;
      if (k == 1)
        wide ? go(combine_kernel<T, W, 1, 4>, w)
             : go(combine_kernel<T, W, 1, 2>, w);
      else
        wide ? go(combine_kernel<T, W, 2, 4>, w)
             : go(combine_kernel<T, W, 2, 2>, w);
    };
    if (!weights || weights->dtype() == at::kFloat)
      pick(weights ? ptr<float>(*weights) : (float*)nullptr);
    else
      pick(ptr<T>(*weights));
  });
  return y;
}

// (drows, dw); one that is not asked for comes back undefined.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>>
combine_rows_backward(const at::Tensor& dy_in, const at::Tensor& rows_in,
                      const at::Tensor& offsets, const at::Tensor& slots,
                      const c10::optional<at::Tensor>& weights,
                      bool need_rows, bool need_weights) {
  c10::cuda::CUDAGuard guard(dy_in.device());
  at::Tensor dy = packed_rows(dy_in);
  at::Tensor rows = need_weights ? packed_rows(rows_in) : dy;
  const int T_rows = (int)slots.size(0), k = (int)slots.size(1);
  const int F = (int)dy.size(1);
  c10::optional<at::Tensor> drows, dw;
  if (need_rows)
    drows = at::empty({(int64_t)T_rows * k, F}, dy.options());
  if (need_weights) dw = at::empty(slots.sizes(), weights->options());
  if (slots.numel() == 0 || (!need_rows && !need_weights)) return {drows, dw};
  if (F == 0) {
    if (dw) dw->zero_();
    return {drows, dw};
  }
  SKA_TYPES(dy.scalar_type(), [&] {
    const int lanes = lanes_for(F, Vec<T>::N), per = 256 / lanes;
    const int* end = ptr<int>(offsets) + offsets.numel() - 1;
    auto go = [&](auto kern, auto* w) {
      kern<<<row_blocks(T_rows, per), 256, 0, stream_now()>>>(
          ptr<T>(dy), dy.stride(0), ptr<T>(rows), rows.stride(0),
          ptr<int>(slots), end, w, T_rows, k, F, lanes,
          drows ? ptr<T>(*drows) : nullptr,
          dw ? ptr<std::decay_t<decltype(*w)>>(*dw) : nullptr);
      check_launch();
    };
    auto pick = [&](auto* w) {
      using W = std::decay_t<decltype(*w)>;
      const bool wide = F / Vec<T>::N >= 4 * lanes;
      if (k == 1)
        wide ? go(combine_back_kernel<T, W, 1, 4>, w)
             : go(combine_back_kernel<T, W, 1, 2>, w);
      else
        wide ? go(combine_back_kernel<T, W, 2, 4>, w)
             : go(combine_back_kernel<T, W, 2, 2>, w);
    };
    if (!weights || weights->dtype() == at::kFloat)
      pick(weights ? ptr<float>(*weights) : (float*)nullptr);
    else
      pick(ptr<T>(*weights));
  });
  return {drows, dw};
}

// ---------------------------------------------------------------------------
// Grouped products.  Row tiles (2^shift rows) are cut inside each group.  Tile
// i is found from the offsets alone: group g's first tile has the index
// floor(offsets[g] / 2^shift) + g, which leaves every group room for its tiles
// (ceil(n / R) <= floor((a + n) / R) - floor(a / R) + 1), so the grid needs
// no count from the device.  The rows behind the last group are a group of
// their own, whose outputs are zero.
// ---------------------------------------------------------------------------
struct Segment {
  int group, start, first, end;  // the tile's rows; first >= end: none
};

__device__ __forceinline__ int edge(const int* offsets, int g, int G, int M) {
  return g <= 0 ? 0 : (g > G ? M : clampi(offsets[g], 0, M));
}

// The last group g with floor(offsets[g] >> shift) + g * each <= at, and its
// rows.  Each round, the lanes look at evenly spaced groups; the last round
// has the group's own edges at hand, so that 62 groups take one read and 3906
// take two.
struct Group {
  int g, start, end;
};

__device__ __forceinline__ Group find_group(const int* offsets, int G, int M,
                                            int at, int shift, int each) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = G + 1;  // the groups lo .. lo + n - 1 are left
  while (true) {
    const int step = (n + 62) / 63;
    const int g = lo + lane * step;
    const int e = edge(offsets, min(g, G + 1), G, M);
    const bool in = lane * step < n && (e >> shift) + g * each <= at;
    // offsets do not decrease, so these are the lanes up to some lane; lane 0
    // counts in any case
    const unsigned long long set = __ballot(in) | 1ull;
    const int last = 63 - __builtin_clzll(set);
    if (step == 1)
      return {__builtin_amdgcn_readfirstlane(lo + last),
              __builtin_amdgcn_readlane(e, last),
              __builtin_amdgcn_readlane(e, last + 1)};
    lo += last * step;
    n = min(step, n - last * step);
  }
}

__device__ __forceinline__ Segment find_segment(const int* offsets, int G,
                                                int M, int tile, int shift) {
  const Group of = find_group(offsets, G, M, tile, shift, 1);
  const long first =
      of.start + ((long)(tile - ((of.start >> shift) + of.g)) << shift);
  return {of.g, of.start, (int)min(first, (long)of.end), of.end};
}

// Where a part of a group's rows leaves its sums.  A group of n > R = 2^shift
// rows has ceil(n / R) <= 2 floor(n / R) parts, so that the places of two such
// groups do not meet and 2 (rows / R + 1) of them are enough.
__device__ __forceinline__ long part_place(int start, int shift) {
  return 2l * (start >> shift);
}

// Where there are more groups than rows: one block a row, which has the tile
// that begins at its row, if one does.
__device__ __forceinline__ Segment find_segment_at(const int* offsets, int G,
                                                   int M, int row,
                                                   int shift) {
  const Group of = find_group(offsets, G, M, row, 0, 0);
  const bool head = ((row - of.start) & ((1 << shift) - 1)) == 0;
  return {of.g, of.start, head ? row : of.end, of.end};
}

__host__ __device__ constexpr int log2_of(int v) {
  return v <= 1 ? 0 : 1 + log2_of(v >> 1);
}

// ---------------------------------------------------------------------------
// Products on v_mfma_f32_16x16x32 (16-bit types) and v_mfma_f32_16x16x4
// (float32).  All three are
//
//     out[m, n] = sum_c A[m, c] * B[n, c]
//
//   forward   A = rows (m = s, c = f)    B = weight[g] (n, c = f)
//   drows     A = dy   (m = s, c = n')   B = weight[g] (n = f, c = n')
//   dweight   A = dy   (m = n', c = s)   B = rows      (n = f, c = s)
//
// An operand lies in memory along c ("along") or across it ("across": m or n
// is the contiguous index).  Tiles of 128 bytes of c (KS steps) go to LDS in
// granules of 16 bytes (V values), by buffer loads that write LDS themselves; a
// lane out of range writes zeros.  An along tile is [m][KS]: granule j of row m
// lies at j ^ swap(m), and a fragment is one 16-byte read.  An across tile is
// [KS][m]: its fragments are two transposing reads of 4 values of c each (16
// lanes read 4 rows of 32 bytes), or 4 single reads of float32; granules are
// moved by bits of c so that these rows lie in different banks.
//
// A lane of either operand holds the V steps from (lane >> 4) * V of a half
// tile.  That both agree is all that the sum needs: for float32, four
// instructions take one of the four steps each.
//
// The matrix instruction gets B first: a lane then holds 4 neighbouring n of
// one m, and stores them together.
//
// Sums leave in their operands' type, rounded once: 32-bit outputs of 16-bit
// operands would double the bytes that the next call reads, which bound most
// calls, for what a caller with 16-bit tensors rounds away anyhow.  A gradient
// through three calls carries three such roundings.
// ---------------------------------------------------------------------------
enum Mode { kForward, kDRows, kDWeight };

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef __bf16 Frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 go(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> {
  typedef _Float16 Frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 go(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Mma<float> {
  typedef f32x4 Frag;
  static __device__ __forceinline__ f32x4 go(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
#define SKA_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

// One operand's tile of EXT rows (m or n) by KS steps of c.  With FRAGS > 1
// the rows of FRAGS neighbouring fragments are dealt out 4 at a time: row r of
// fragment j is (r / 4) * 4 * FRAGS + j * 4 + r % 4 of their 16 * FRAGS.  A
// lane of the product then holds 4 * FRAGS neighbouring n.
template <typename T, int EXT, bool ACROSS, int THREADS, int FRAGS>
struct Tile {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int KS = 8 * V;
  static constexpr int kGranules = EXT * KS / V;
  static constexpr int kPer = kGranules / THREADS;
  static constexpr int kAcross = EXT / V;  // granules of one step of c
  static constexpr int kBytes = kGranules * 16;

  // how the granules of an along row, or of an across step, are moved, so
  // that the 8 rows of 8 lanes (the 4 steps of 16) lie in different banks
  static __device__ __forceinline__ int swap(int row) {
    const int high = FRAGS == 1 ? row >> 2 : FRAGS == 2 ? row >> 3 : row >> 4;
    return (row & 3) | (high & 1) << 2;
  }
  static __device__ __forceinline__ int move(int c) {
    if (V == 4) {
      const int q = (c >> 2) & 3;
      return (FRAGS == 1   ? q << 2
              : FRAGS == 2 ? (q & 1) | (q & 2) << 2
                           : q) &
             (kAcross - 1);
    }
    if (FRAGS == 1)
      return (((c & 3) << 1) | (((c >> 3) & 1) << 3)) & (kAcross - 1);
    if (FRAGS == 2)
      return ((c & 1) | ((c & 2) << 1) | (c & 8)) & (kAcross - 1);
    return ((c & 1) | ((c & 2) << 2)) & (kAcross - 1);
  }
  // the first row and step of the granule at LDS place g
  static __device__ __forceinline__ void place(int g, int& row, int& c) {
    if (ACROSS) {
      c = g / kAcross;
      row = ((g % kAcross) ^ move(c)) * V;
    } else {
      row = g >> 3;
      c = ((g & 7) ^ swap(row)) * V;
    }
  }
  static __device__ __forceinline__ long at(int row, int c, long pitch) {
    return ACROSS ? c * pitch + row : row * pitch + c;
  }
  // Granules are read whole below these bounds.  An across granule at the
  // edge may run into the next row, whose values meet outputs that are not
  // stored, unless it would leave the matrix: `room` is the number of values
  // from `src` to the matrix's end.
  struct Bounds {
    int rows, steps;
    bool ragged;  // some granules are left to fill()
  };
  static __device__ __forceinline__ Bounds bounds(long pitch, int rows,
                                                  int steps, long room) {
    if (ACROSS) {
      const bool cut = rows % V && (min(steps, KS) - 1) * pitch +
                                           ((rows + V - 1) & -V) >
                                       room;
      return {cut ? rows & -V : rows, steps, cut};
    }
    return {rows, steps & -V, steps < KS && steps % V};
  }
  // One of a wave's kPer loads.  Written in assembly, because the compiler
  // would wait for all loads under way before it reads LDS; whoever reads the
  // tile waits for them itself.
  static __device__ __forceinline__ void load_async(const T* src, long pitch,
                                                    Bounds b, char* lds,
                                                    int i) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned long base = reinterpret_cast<unsigned long>(src);
    // base, no stride, 2^31 - 1 bytes, raw
    const i32x4 rsrc = {(int)base, (int)(base >> 32) & 0xffff, 0x7fffffff,
                        0x00020000};
    const unsigned to = __builtin_amdgcn_readfirstlane(
        (unsigned)(uintptr_t)SKA_LDS(void, lds) + wave * 1024);
    int row, c;
    place(i * THREADS + wave * 64 + lane, row, c);
    const bool in = row < b.rows && c < b.steps;
    const unsigned off = in ? (unsigned)at(row, c, pitch) * (unsigned)sizeof(T)
                            : 0x80000000u;
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to + i * THREADS * 16),
        "v"(off), "s"(rsrc)
        : "memory", "m0");
  }
  // The granules that load_async leaves out, after its loads have ended.
  static __device__ __forceinline__ void fill(const T* src, long pitch,
                                              int rows, int steps, Bounds b,
                                              char* lds) {
#pragma unroll 1
    for (int i = 0; i < kPer; ++i) {
      const int g = i * THREADS + threadIdx.x;
      int row, c;
      place(g, row, c);
      const int n = ACROSS ? (row >= b.rows && c < steps ? rows - row : 0)
                           : (c >= b.steps && row < rows ? steps - c : 0);
      T* to = reinterpret_cast<T*>(lds + g * 16);
      const T* from = src + at(row, c, pitch);
      for (int e = 0; e < min(n, V); ++e) to[e] = from[e];
    }
  }
  // rows that begin at odd addresses: through registers
  static __device__ __forceinline__ void load_regs(const T* src, long pitch,
                                                   int rows, int steps,
                                                   Bounds b,
                                                   Vec<T> (&v)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int row, c;
      place(i * THREADS + threadIdx.x, row, c);
      int n = row < b.rows && c < b.steps ? V : 0;
      if (b.ragged && n == 0 && row < rows && c < steps)
        n = ACROSS ? rows - row : steps - c;
      v[i] = load_vec(src + (n > 0 ? at(row, c, pitch) : 0), n);
    }
  }
  static __device__ __forceinline__ void store_regs(const Vec<T> (&v)[kPer],
                                                    char* lds) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      *reinterpret_cast<Vec<T>*>(lds + (i * THREADS + threadIdx.x) * 16) =
          v[i];
  }
  // fragment j of the rows from row0, in a half of the tile's steps
  static __device__ __forceinline__ typename Mma<T>::Frag frag(
      const char* lds, int row0, int j, int half) {
    const int lane = threadIdx.x & 63;
    const int r = lane & 15, q = lane >> 4;
    const int c0 = half * (KS / 2) + q * V;
    if constexpr (ACROSS && V == 8) {
      // lane (4 * step + s) of 16 reads rows 4 * s .. 4 * s + 3 of the fragment
      const int row = row0 + (FRAGS == 1 ? j * 16 + (r & 3) * 4
                                         : (r & 3) * 4 * FRAGS + j * 4);
      s16x4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + h * 4 + (r >> 2);
        const int g = (row >> 3) ^ move(c);
        v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            SKA_LDS(s16x4, lds + (c * kAcross + g) * 16 + (row & 4) * 2));
      }
      const s16x8 w = {v[0][0], v[0][1], v[0][2], v[0][3],
                       v[1][0], v[1][1], v[1][2], v[1][3]};
      return __builtin_bit_cast(typename Mma<T>::Frag, w);
    }
    const int row = row0 + (FRAGS == 1 ? j * 16 + r
                                       : (r >> 2) * 4 * FRAGS + j * 4 +
                                             (r & 3));
    if constexpr (ACROSS) {
      typename Mma<T>::Frag v;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int g = (row / V) ^ move(c0 + i);
        v[i] = *reinterpret_cast<const T*>(
            lds + ((c0 + i) * kAcross + g) * 16 + row % V * sizeof(T));
      }
      return v;
    }
    return *reinterpret_cast<const typename Mma<T>::Frag*>(
        lds + (row * 8 + ((c0 / V) ^ swap(row))) * 16);
  }
};

// Waits for a wave's own loads.
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), nothing else
}

// A barrier for what the block wrote to LDS itself; loads under way go on.
__device__ __forceinline__ void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct Product {
  const void* a;
  const void* b;
  const void* bias;  // forward: [G, N]
  void* out;   // dweight: null for the sums alone, in the same order
  void* sums;  // dweight: null, or the sum of A over c, [G, M]
  const int* offsets;
  long a_pitch, b_pitch;
  int G, M, N, C;  // dweight: M rows of out a group, C rows in all
  // dweight over parts of a group's rows: 2^shift rows each (0: whole
  // groups), whose sums go to part [.][M][N] and part_sums [.][M] unless the
  // group has but one
  int shift;
  float* part;
  float* part_sums;
  int tiles;  // output tiles of the launch
  int run;    // of neighbouring tiles that go to one XCD
};

// One tile of the output: its operands and where it goes.
template <typename T>
struct Job {
  const T *a, *b;
  long a_room, b_room, out_row;
  int group, rows, cols, n0;
  int steps;  // of c; 0: an output of zeros
  bool parted;
};

// Tile number `tile` of the launch, if there is such a one.
template <typename T, int BM, int BN, int MODE>
__device__ __forceinline__ bool find_job(const Product& p, int tile,
                                         Job<T>& job) {
  const int nt = p.out ? (p.N + BN - 1) / BN : 1;
  const int mt = p.tiles / nt;
  const T* A = reinterpret_cast<const T*>(p.a);
  const T* B = reinterpret_cast<const T*>(p.b);
  if (MODE == kDWeight) {
    job.n0 = (tile % nt) * BN;
    tile /= nt;
    const int each = (p.M + BM - 1) / BM;
    const int unit = tile / each;
    const int m0 = (tile % each) * BM;
    int first, start = 0;
    job.parted = false;
    if (p.shift) {
      const Segment seg = find_segment(p.offsets, p.G, p.C, unit, p.shift);
      if (seg.first >= seg.end || seg.group >= p.G) return false;
      job.group = seg.group;
      first = seg.first;
      start = seg.start;
      job.steps = ska::part_end(first, seg.end, p.shift) - first;
      job.parted = seg.end - seg.start > (1 << p.shift);
    } else {
      job.group = unit;
      first = __builtin_amdgcn_readfirstlane(edge(p.offsets, unit, p.G, p.C));
      job.steps = __builtin_amdgcn_readfirstlane(
                      edge(p.offsets, unit + 1, p.G, p.C)) -
                  first;
    }
    job.rows = min(BM, p.M - m0);
    job.out_row = (job.parted ? part_place(start, p.shift) +
                                    ((first - start) >> p.shift)
                              : (long)job.group) *
                      p.M +
                  m0;
    job.a = A + first * p.a_pitch + m0;
    job.b = B + first * p.b_pitch + job.n0;
    job.a_room = (long)(p.C - first - 1) * p.a_pitch + p.M - m0;
    job.b_room = (long)(p.C - first - 1) * p.b_pitch + p.N - job.n0;
  } else {
    // The row tiles are gone through in bands of 1024 columns: the blocks
    // that an XCD runs at a time then share rows and weights alike.
    constexpr int kBand = 1024 / BN;
    const int band = tile / (mt * kBand);
    const int wide = min(kBand, nt - band * kBand);
    tile -= band * mt * kBand;
    job.n0 = (band * kBand + tile % wide) * BN;
    tile /= wide;
    const Segment seg = find_segment(p.offsets, p.G, p.M, tile, log2_of(BM));
    if (seg.first >= seg.end) return false;
    job.parted = false;
    job.group = seg.group;
    job.rows = min(BM, seg.end - seg.first);
    job.steps = seg.group < p.G ? p.C : 0;
    job.out_row = seg.first;
    job.a = A + seg.first * p.a_pitch;
    job.a_room = 0;
    const long weights = (long)p.N * p.C;
    job.b = B + min(seg.group, p.G - 1) * weights +
            (MODE == kForward ? job.n0 * (long)p.C : job.n0);
    job.b_room = (long)(p.C - 1) * p.N + p.N - job.n0;
    if (seg.group < p.G - 1) job.b_room += weights;
  }
  job.cols = min(BN, p.N - job.n0);
  return true;
}

// 8192^3 bfloat16 in one group: 858 us, 1281 TFLOP/s (1308 for a library's
// product); 65536 x 2048 x 1024 in 64 groups: 310 us, 886, since the groups'
// last tiles are half empty and 1160 tiles take five rounds of 256 CUs, not
// 4.5. What it took from there on: loads spread among the matrix instructions
// (1166 -> 1067 us at 8192^3; all at once they hold up the waves) and the
// bands of find_job (-> 895; at 65536 x 2048 x 1024 65% of the L2's reads now
// hit).  What did not help: four waves with fragments of two half steps (797
// TFLOP/s), waves that take turns at LDS and the matrix unit (708), three tiles
// in LDS, one block a CU that goes through many tiles.
//
// Tiles of c in LDS, filled by loads that write it (ASYNC) or through
// registers: two, or one (not AHEAD) for short contractions, whose blocks hide
// each other's loads and of which more then fit a CU.
template <typename T, int BM, int BN, int WM, int WN, int MODE, bool ASYNC,
          bool AHEAD = true>
__global__ __launch_bounds__(WM* WN * 64, 2) void product_kernel(Product p) {
  constexpr int kThreads = WM * WN * 64;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Tile<T, BM, MODE == kDWeight, kThreads, 1> TA;
  typedef Tile<T, BN, MODE != kForward, kThreads, FN> TB;
  constexpr int KS = TA::KS;
  static_assert(ASYNC || AHEAD);
  __shared__ __align__(16) char lds[AHEAD ? 2 : 1][TA::kBytes + TB::kBytes];

  // Blocks go round the 8 XCDs: each XCD gets runs of neighbouring tiles, whose
  // operands its L2 then holds.
  const int at = blockIdx.x >> 3;
  const int tile =
      (at / p.run * 8 + (blockIdx.x & 7)) * p.run + at % p.run;
  Job<T> job;
  if (tile >= p.tiles || !find_job<T, BM, BN, MODE>(p, tile, job)) return;

  const long a_step = MODE == kDWeight ? KS * p.a_pitch : KS;
  const long b_step = MODE == kForward ? KS : KS * p.b_pitch;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

  // A tile's operands at step c, and which of their granules are whole.
  struct Source {
    const T *a, *b;
    typename TA::Bounds ba;
    typename TB::Bounds bb;
    int steps;
  };
  auto source = [&](int c) {
    const long at = c / KS;
    return Source{
        job.a + at * a_step, job.b + at * b_step,
        TA::bounds(p.a_pitch, job.rows, job.steps - c,
                   job.a_room - at * a_step),
        TB::bounds(p.b_pitch, job.cols, job.steps - c,
                   job.b_room - at * b_step),
        job.steps - c};
  };
  constexpr int kLoads = TA::kPer + TB::kPer;
  Vec<T> ra[ASYNC ? 1 : TA::kPer], rb[ASYNC ? 1 : TB::kPer];
  auto load = [&](const Source& s, int buf, int i) {
    if (i < TA::kPer)
      TA::load_async(s.a, p.a_pitch, s.ba, lds[buf], i);
    else
      TB::load_async(s.b, p.b_pitch, s.bb, lds[buf] + TA::kBytes,
                     i - TA::kPer);
  };
  auto load_regs = [&](const auto& s) {
    TA::load_regs(s.a, p.a_pitch, job.rows, s.steps, s.ba, ra);
    TB::load_regs(s.b, p.b_pitch, job.cols, s.steps, s.bb, rb);
  };
  f32x4 acc[FM][FN] = {};
  // The sums of the weights' gradients go over a group's rows, as many as
  // these may be.  In float32 they are taken in parts of 512 rows, since an
  // addition's rounding grows with the sum so far: over 32768 rows they are
  // 4e-7 off (in the 2-norm), a library's single sum 3e-6.  16-bit results
  // round far more.
  constexpr bool PARTS = sizeof(T) == 4 && MODE == kDWeight;
  constexpr int kPart = 512 / KS;
  f32x4 total[PARTS ? FM : 1][PARTS ? FN : 1] = {};
  // The sums over c of A: a product with ones, of which each of the WN waves
  // that hold the same rows takes FS fragments.
  constexpr int FS = FM / WN > 0 ? FM / WN : 1;
  f32x4 sum[FS] = {}, total_sum[FS] = {};
  const bool sums = MODE == kDWeight && p.sums && job.n0 == 0;
  const int mine = wave % WN;
  typename Mma<T>::Frag ones;
#pragma unroll
  for (int i = 0; i < TA::V; ++i) ones[i] = (T)1.f;

  if (job.steps > 0) {
    if constexpr (ASYNC) {
      const Source from = source(0);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load(from, 0, i);
    } else {
      load_regs(source(0));
    }
  }
  int buf = 0;
#pragma unroll 1
  for (int c = 0; c < job.steps; c += KS) {
    // Tile c lands.  At the barrier all waves have also read the tile
    // before, whose place the loads of the next then take.
    if constexpr (ASYNC) {
      wait_loads();
      const Source s = source(c);
      if (s.ba.ragged)
        TA::fill(s.a, p.a_pitch, job.rows, s.steps, s.ba, lds[buf]);
      if (s.bb.ragged)
        TB::fill(s.b, p.b_pitch, job.cols, s.steps, s.bb,
                 lds[buf] + TA::kBytes);
    } else {
      TA::store_regs(ra, lds[buf]);
      TB::store_regs(rb, lds[buf] + TA::kBytes);
    }
    block_barrier();
    // Behind the last tile these loads write zeros, for nobody.
    const Source next = source(c + KS);
    if constexpr (!ASYNC)
      if (next.steps > 0) load_regs(next);
    const char* la = lds[buf];
    const char* lb = lds[buf] + TA::kBytes;
    // 2 FM groups of FN matrix instructions.  Each group reads the fragments
    // of the next and, in the first half, issues its share of the loads: all
    // at once they would hold up the waves, since the vector memory takes
    // them no faster than 64 bytes a clock.
    typename Mma<T>::Frag fa[2], fb[2][FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[0][j] = TB::frag(lb, wn, j, 0);
    fa[0] = TA::frag(la, wm, 0, 0);
#pragma unroll
    for (int g = 0; g < 2 * FM; ++g) {
      const int h = g / FM, i = g % FM;
      if (g + 1 < 2 * FM)
        fa[(g + 1) & 1] = TA::frag(la, wm, (g + 1) % FM, (g + 1) / FM);
      if (h == 0) {
#pragma unroll
        for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j)
          fb[1][j] = TB::frag(lb, wn, j, 1);
        if constexpr (ASYNC && AHEAD) {
#pragma unroll
          for (int l = i * kLoads / FM; l < (i + 1) * kLoads / FM; ++l)
            load(next, buf ^ 1, l);
        }
      }
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = Mma<T>::go(fb[h][j], fa[g & 1], acc[i][j]);
      if (MODE == kDWeight && sums && i / FS == mine)
        sum[i % FS] = Mma<T>::go(ones, fa[g & 1], sum[i % FS]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (PARTS) {
      if (c / KS % kPart == kPart - 1 || next.steps <= 0) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            total[i][j] += acc[i][j];
            acc[i][j] = next.steps > 0 ? f32x4{} : total[i][j];
          }
#pragma unroll
        for (int i = 0; i < FS; ++i) {
          total_sum[i] += sum[i];
          sum[i] = next.steps > 0 ? f32x4{} : total_sum[i];
        }
      }
    }
    if constexpr (AHEAD) {
      buf ^= 1;
    } else if (next.steps > 0) {
      block_barrier();
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load(next, 0, i);
    }
  }

  // LDS is not given back with loads under way.
  if constexpr (ASYNC) wait_loads();

  // lane: row m = lane & 15 of each fragment, 4 * FN neighbouring columns
  T* out = reinterpret_cast<T*>(p.out);
  const T* bias = reinterpret_cast<const T*>(p.bias);
  const int n = wn + (lane >> 4) * 4 * FN;
  const int left = job.cols - n;
  if (left > 0 && (MODE != kDWeight || out)) {
    constexpr int V = TA::V, kStores = 4 * FN / V;
    Vec<T> extra[kStores] = {};
    const bool biased = MODE == kForward && bias && job.group < p.G;
    if (biased) {
#pragma unroll
      for (int j = 0; j < kStores; ++j)
        extra[j] = load_vec(bias + (long)job.group * p.N + job.n0 + n + j * V,
                            left - j * V);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = wm + i * 16 + (lane & 15);
      if (m >= job.rows) continue;
      const long at = (job.out_row + m) * p.N + job.n0 + n;
      if (MODE == kDWeight && job.parted) {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          if (left >= j * 4 + 4) {
            *reinterpret_cast<Bytes16*>(p.part + at + j * 4) =
                __builtin_bit_cast(Bytes16, acc[i][j]);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (j * 4 + r < left) p.part[at + j * 4 + r] = acc[i][j][r];
          }
        }
        continue;
      }
#pragma unroll
      for (int j = 0; j < kStores; ++j) {
        Vec<T> v;
#pragma unroll
        for (int r = 0; r < V; ++r) {
          float x = acc[i][(j * V + r) / 4][r & 3];
          if (biased) x += to_f(extra[j].v[r]);
          v.v[r] = (T)x;
        }
        store_vec(out + at + j * V, v, left - j * V);
      }
    }
  }
  if (sums && lane < 16) {
#pragma unroll
    for (int i = 0; i < FS; ++i) {
      const int m = wm + (mine * FS + i) * 16 + lane;
      if (mine * FS + i >= FM || m >= job.rows) continue;
      if (job.parted)
        p.part_sums[job.out_row + m] = sum[i][0];
      else
        reinterpret_cast<T*>(p.sums)[job.out_row + m] = (T)sum[i][0];
    }
  }
}

// Ends a dweight over parts: the sums of the groups that have several, in
// their order, and zeros for groups without rows.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(Product p) {
  const int g = blockIdx.x;
  const int start = edge(p.offsets, g, p.G, p.C);
  const int end = edge(p.offsets, g + 1, p.G, p.C);
  const int count = ska::part_count(start, end, p.shift);
  if (count == 1) return;
  const long size = (long)p.M * p.N;
  const long unit = part_place(start, p.shift);
  T* out = reinterpret_cast<T*>(p.out) + g * size;
  for (long e = (long)blockIdx.y * 256 + threadIdx.x; p.out && e < size;
       e += (long)gridDim.y * 256) {
    float sum = 0.f;
#pragma unroll 8
    for (int u = 0; u < count; ++u) sum += p.part[(unit + u) * size + e];
    out[e] = (T)sum;
  }
  if (p.sums && blockIdx.y == 0)
    for (int m = threadIdx.x; m < p.M; m += 256) {
      float sum = 0.f;
#pragma unroll 8
      for (int u = 0; u < count; ++u) sum += p.part_sums[(unit + u) * p.M + m];
      reinterpret_cast<T*>(p.sums)[(long)g * p.M + m] = (T)sum;
    }
}

// ---------------------------------------------------------------------------
// Narrow forward products: few outputs (a keyed model's classes) or few rows a
// group (single rows of a serving step).  Bound by reading the larger operand,
// once: 8 rows x 2048 x 2048 bfloat16 in 12.4 us (5.4 TB/s), 10^6 x 256
// float32 with 10 outputs in 218 us (4.9).  It goes straight from memory into
// fragments: a lane takes 16 bytes of row lane & 15 at the contraction's step
// (lane >> 4) * V, and both operands agree on which steps these are, so their
// order in the instruction does not matter. KW of the 4 waves share the
// contraction, the others lie along the rows.
// ---------------------------------------------------------------------------
template <typename T>
struct Wide {
  typedef typename Mma<T>::Frag Frag;
  static __device__ __forceinline__ Frag load(const T* p) {
    return get(p).v;
  }
  static __device__ __forceinline__ Frag load(const T* p, int n) {
    Frag v;
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i)
      v[i] = i < n ? p[i] : (T)0.f;
    return v;
  }
};

template <typename T, int MF, int NF, int KW>
__global__ __launch_bounds__(256) void narrow_kernel(Product p, bool by_row) {
  constexpr int V = 16 / sizeof(T), kChunk = 4 * V;
  constexpr int BM = 4 / KW * MF * 16, BN = NF * 16;
  const Segment seg =
      by_row ? find_segment_at(p.offsets, p.G, p.M, blockIdx.x, log2_of(BM))
             : find_segment(p.offsets, p.G, p.M, blockIdx.x, log2_of(BM));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int part = wave % KW;
  const int row0 = seg.first + wave / KW * MF * 16;
  const int n0 = blockIdx.y * BN;
  if (KW == 1 ? row0 >= seg.end : seg.first >= seg.end) return;
  f32x4 acc[MF][NF] = {};
  if (seg.group < p.G) {
    // rows and outputs past the end read the last one's values, and are not
    // stored
    const T *a[MF], *b[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
      a[i] = reinterpret_cast<const T*>(p.a) +
             min(row0 + i * 16 + r, seg.end - 1) * p.a_pitch + q * V;
#pragma unroll
    for (int j = 0; j < NF; ++j)
      b[j] = reinterpret_cast<const T*>(p.b) +
             ((long)seg.group * p.N + min(n0 + j * 16 + r, p.N - 1)) * p.C +
             q * V;
    const int whole = p.C / kChunk * kChunk;
    int c = part * kChunk;
    auto chunks = [&](auto n) {
      constexpr int U = decltype(n)::value;
      typename Wide<T>::Frag fa[U][MF], fb[U][NF];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = c + u * KW * kChunk;
#pragma unroll
        for (int i = 0; i < MF; ++i) fa[u][i] = Wide<T>::load(a[i] + at);
#pragma unroll
        for (int j = 0; j < NF; ++j) fb[u][j] = Wide<T>::load(b[j] + at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
          for (int j = 0; j < NF; ++j)
            acc[i][j] = Mma<T>::go(fb[u][j], fa[u][i], acc[i][j]);
    };
    constexpr int U = MF + NF > 4 ? 2 : 4;
    for (; c + (U - 1) * KW * kChunk < whole; c += U * KW * kChunk)
      chunks(Count<U>{});
    for (; c < whole; c += KW * kChunk) chunks(Count<1>{});
    if (c == whole && whole < p.C) {
      const int left = p.C - whole - q * V;
      typename Wide<T>::Frag fa[MF], fb[NF];
#pragma unroll
      for (int i = 0; i < MF; ++i) fa[i] = Wide<T>::load(a[i] + c, left);
#pragma unroll
      for (int j = 0; j < NF; ++j) fb[j] = Wide<T>::load(b[j] + c, left);
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
          acc[i][j] = Mma<T>::go(fb[j], fa[i], acc[i][j]);
    }
  }
  if constexpr (KW > 1) {
    __shared__ f32x4 sums[4][MF * NF][64];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) sums[wave][i * NF + j][lane] = acc[i][j];
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int w = 1; w < KW; ++w)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
          acc[i][j] += sums[wave + w][i * NF + j][lane];
  }
  const T* bias = reinterpret_cast<const T*>(p.bias);
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int n = n0 + j * 16 + q * 4;
    const int left = p.N - n;
    if (left <= 0) continue;
    float add[4] = {};
    if (bias && seg.group < p.G) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) add[e] = to_f(bias[(long)seg.group * p.N + n + e]);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int m = row0 + i * 16 + r;
      if (m >= seg.end) continue;
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(acc[i][j][e] + add[e]);
      T* to = reinterpret_cast<T*>(p.out) + (long)m * p.N + n;
      if (left >= 4) {
        __builtin_memcpy(to, v, sizeof(v));
      } else {
        for (int e = 0; e < left; ++e) to[e] = v[e];
      }
    }
  }
}

// float32 dweight with few outputs: dw[g, n, f] for 16 outputs.  A lane takes
// 4 columns f = 4 * (lane & 15) + e of the row (lane >> 4) * 4 + i, which are
// four fragments' values at once.  KW of the 4 waves share the rows, the
// others lie along f.  Bound by reading the rows: 400000 x 256 with 3 outputs
// in 512 groups take 86 us (4.8 TB/s; 64^2 tiles 171).  No accumulator takes
// more than 512 rows: a term passes the additions of its own 512, then one for
// each 512 rows of its wave's share, KW - 1, and one for each part of the group
// (2048 at most).
template <int KW>
__global__ __launch_bounds__(256) void narrow_dweight_kernel(Product p) {
  constexpr int BF = 4 / KW * 64;
  const Segment seg = find_segment(p.offsets, p.G, p.C, blockIdx.x, p.shift);
  if (seg.first >= seg.end || seg.group >= p.G) return;
  const int end = ska::part_end(seg.first, seg.end, p.shift);
  const bool parted = seg.end - seg.start > (1 << p.shift);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int part = wave % KW;
  const int f = blockIdx.y * BF + wave / KW * 64 + r * 4;
  const int left = p.N - f;
  const bool sums = p.sums && blockIdx.y == 0 && wave / KW == 0;
  const float* a = reinterpret_cast<const float*>(p.a);
  const float* b = reinterpret_cast<const float*>(p.b) + f;
  const int n = min(r, p.M - 1);
  f32x4 acc[4] = {}, sum = {};
  int s = seg.first + part * 16;
  while (s < end) {
    const int stop = ska::part_end(s, end, log2_of(KW * 512));
    f32x4 now[4] = {}, now_sum = {};
#pragma unroll 2
    for (; s < stop; s += KW * 16) {
      float fa[4];
      f32x4 fb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = s + q * 4 + i;
        const bool in = row < end;
        const long at = in ? row : end - 1;
        const float d = a[at * p.a_pitch + n];
        fa[i] = in ? d : 0.f;
        f32x4 v = {};
        if (left >= 4) {
          __builtin_memcpy(&v, b + at * p.b_pitch, 16);
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (e < left) v[e] = b[at * p.b_pitch + e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) fb[i][e] = in ? v[e] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          now[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i][e],
                                                        now[e], 0, 0, 0);
        if (sums)
          now_sum = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], 1.f, now_sum,
                                                         0, 0, 0);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += now[e];
    sum += now_sum;
  }
  if constexpr (KW > 1) {
    __shared__ f32x4 all[4][5][64];
#pragma unroll
    for (int e = 0; e < 4; ++e) all[wave][e][lane] = acc[e];
    all[wave][4][lane] = sum;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int w = 1; w < KW; ++w) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += all[wave + w][e][lane];
      sum += all[wave + w][4][lane];
    }
  }
  const long out_row =
      (parted ? part_place(seg.start, p.shift) +
                    ((seg.first - seg.start) >> p.shift)
              : (long)seg.group) *
      p.M;
  float* out = parted && p.out ? p.part : reinterpret_cast<float*>(p.out);
  float* out_sums = parted ? p.part_sums : reinterpret_cast<float*>(p.sums);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = q * 4 + i;
    if (m >= p.M) continue;
    float* to = out + (out_row + m) * p.N + f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (p.out && e < left) to[e] = acc[e][i];
    if (sums && r == 0) out_sums[out_row + m] = sum[i];
  }
}

// drows with a short contraction (the classes of a keyed model, C <= NB):
// bound by writing the rows.  A lane holds its columns' weights, the rows' dy
// are in LDS in 32 bits, and a wave writes 32 rows in whole vectors; `lanes`
// lanes (a power of two) share a row.
template <typename T, int NB>
__global__ __launch_bounds__(256) void narrow_drows_kernel(Product p,
                                                           int lanes) {
  constexpr int V = 16 / sizeof(T), BM = 128;
  const Segment seg =
      find_segment(p.offsets, p.G, p.M, blockIdx.x, log2_of(BM));
  if (seg.first >= seg.end) return;
  __shared__ __align__(16) float d[BM][NB];
  const int rows = min(BM, seg.end - seg.first);
  const bool any = seg.group < p.G;
  const T* a = reinterpret_cast<const T*>(p.a) + seg.first * p.a_pitch;
  for (int i = threadIdx.x; i < BM * NB; i += 256) {
    const int row = i / NB, n = i % NB;
    d[row][n] = any && row < rows && n < p.C ? to_f(a[row * p.a_pitch + n])
                                             : 0.f;
  }
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int per = 64 / lanes;
  const int end = min(rows, wave * 32 + 32);
  const T* b = reinterpret_cast<const T*>(p.b) +
               (long)min(seg.group, p.G - 1) * p.C * p.N;
  T* out = reinterpret_cast<T*>(p.out) + (long)seg.first * p.N;
  for (int f = (blockIdx.y * lanes + lane % lanes) * V; f < p.N;
       f += gridDim.y * lanes * V) {
    const int left = p.N - f;
    float w[NB][V];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      Vec<T> v = {};
      if (any && n < p.C) v = load_vec(b + (long)n * p.N + f, left);
#pragma unroll
      for (int i = 0; i < V; ++i) w[n][i] = to_f(v.v[i]);
    }
    for (int row = wave * 32 + lane / lanes; row < end; row += per) {
      float acc[V] = {};
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float x = d[row][n];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += x * w[n][i];
      }
      Vec<T> v;
#pragma unroll
      for (int i = 0; i < V; ++i) v.v[i] = (T)acc[i];
      store_vec(out + (long)row * p.N + f, v, left);
    }
  }
}

// Buffer loads to LDS take addresses of whole words.
template <typename T>
bool whole_words(const T* p, long pitch) {
  return (reinterpret_cast<uintptr_t>(p) & 3) == 0 && (pitch & 1) == 0;
}

unsigned grid_of(long blocks, int threads) {
  TORCH_CHECK(blocks * threads < (1ll << 32), "too many output tiles");
  return (unsigned)blocks;
}

template <typename T>
bool narrow_launch(const Product& p) {
  const long rows = p.M / std::min(p.G, p.M);
  auto go = [&](auto kern, int bm, int bn) {
    const bool by_row = p.M < p.M / bm + p.G + 1;
    const long tiles = by_row ? p.M : p.M / bm + p.G + 1;
    dim3 grid(grid_of(tiles, 256), (p.N + bn - 1) / bn);
    if (grid.y > 65535) return false;  // more than a launch takes
    kern<<<grid, 256, 0, stream_now()>>>(p, by_row);
    check_launch();
    return true;
  };
  // Measured against the tile kernels, us (type, rows, groups, outputs,
  // columns; the kernels by rows x outputs of a wave, k: its share of c):
  //   float32       8,   64, 2048, 2048: 16 x 32 k 34, tiles  83
  //   float32    2000,  200,  512,  512: 16 x 32 k 45, tiles  69
  //   float32    3000,   64, 1024, 1024: 16 x 32 k 203, tiles 110
  //   bfloat16      8,   64, 2048, 2048: 16 x 16 k 12, tiles  20
  //   bfloat16   2000,  200,  512,  512: 16 x 16 k 28, tiles  22
  //   float32 1000000, 1000,  10,  256: 64 x 16 225, 32 x 16 k 247, tiles 355
  //   float32  200000, 1000,   3,  250: 64 x 16  56, 32 x 16 k  42, tiles  88
  //   float32  400000, 1000,  32,  256: 32 x 32 127, tiles 149
  //   float32  400000, 1000,  64,  256: 32 x 32 244, tiles 164
  //   bfloat16 200000, 1000,   3,  250: 64 x 16  31, 32 x 16 k  23, tiles  35
  //   bfloat16 400000, 1000,  32,  256: 64 x 32  51, tiles  49
  constexpr bool kWide = sizeof(T) == 4;
  if (rows <= (kWide ? 16 : 8))
    return kWide ? go(narrow_kernel<T, 1, 2, 4>, 16, 32)
                 : go(narrow_kernel<T, 1, 1, 4>, 16, 16);
  if (p.N <= 16)
    return rows >= 512 && p.C < 512 ? go(narrow_kernel<T, 4, 1, 1>, 256, 16)
                                    : go(narrow_kernel<T, 2, 1, 4>, 32, 16);
  if constexpr (kWide)
    if (p.N <= 32) return go(narrow_kernel<T, 2, 2, 1>, 128, 32);
  return false;
}

// Parts of a group's rows, so that `tiles` outputs a group make about `want`
// blocks of work that are alike.
int part_shift(long rows, long tiles, long want) {
  int shift = 8;
  while (shift < 30 && (rows * tiles >> shift) > want) ++shift;
  return shift;
}

struct Parts {
  at::Tensor part, sums;
};

Parts take_parts(Product& p, at::TensorOptions opt) {
  Parts parts;
  const int64_t units = 2 * (((int64_t)p.C >> p.shift) + 1);
  if (p.out) {
    parts.part = at::empty({units, p.M, p.N}, opt.dtype(at::kFloat));
    p.part = ptr<float>(parts.part);
  }
  if (p.sums) {
    parts.sums = at::empty({units, p.M}, opt.dtype(at::kFloat));
    p.part_sums = ptr<float>(parts.sums);
  }
  return parts;
}

template <typename T>
void finish_launch(const Product& p) {
  const long size = (long)p.M * p.N;
  dim3 grid(grid_of(p.G, 256), std::min(1024l, (size + 255) / 256));
  finish_kernel<T><<<grid, 256, 0, stream_now()>>>(p);
  check_launch();
}

template <typename T, int MODE>
void product_launch(Product p, at::TensorOptions opt) {
  if (MODE == kForward && narrow_launch<T>(p)) return;
  const bool async =
      sizeof(T) == 4 ||
      (whole_words((const T*)p.a, p.a_pitch) &&
       whole_words((const T*)p.b, p.b_pitch) &&
       // the weights of a group may begin at an odd value
       (MODE == kDWeight || ((long)p.N * p.C) % 2 == 0));
  auto tiles = [&](long b) { return (p.M + b - 1) / b * ((p.N + b - 1) / b); };
  auto go = [&](auto kern, int bm, int bn, int threads) {
    const long m_tiles = (p.M + bm - 1) / bm;
    long mt = (long)p.M / bm + p.G + 1;
    Parts parts;
    if (MODE == kDWeight) {
      mt = p.G * m_tiles;
      const long all = m_tiles * ((p.N + bn - 1) / bn);
      if (bm == 64 && all * p.G < 512) {
        p.shift = part_shift(p.C, all, 512);
        parts = take_parts(p, opt);
        mt = ((p.C >> p.shift) + p.G + 1) * m_tiles;
      }
    }
    const long nt = p.out ? (p.N + bn - 1) / bn : 1;
    grid_of(mt * nt + 512, threads);
    p.tiles = (int)(mt * nt);
    // One run an XCD shares most; shorter ones spread large groups.  us for
    // one run / 16 tiles: forward 65536, 64, 1024, 2048: 345 / 305, but 65536,
    // 32, 4096, 1024: 593 / 634; dweight of the latter 696 / 598, and with more
    // skewed groups 894 / 653, but 8198, 48, 768, 768 (9 tiles a group): 32 / 39
    const long each = m_tiles * nt;
    long most = p.tiles;
    if (MODE == kDWeight)
      most = each > 16 ? 16 : each * std::max(1l, 8 / each);
    else if (bm == 256 && nt <= 4)
      most = 16;
    p.run = (int)std::min(most, (p.tiles + 7l) / 8);
    const long round = 8 * p.run;
    const unsigned blocks = (unsigned)((p.tiles + round - 1) / round * round);
    kern<<<blocks, threads, 0, stream_now()>>>(p);
    check_launch();
    if (MODE == kDWeight && p.shift) finish_launch<T>(p);
  };
  // Larger tiles read less and fill the matrix units better; smaller ones
  // waste less of the groups' last tiles and leave more blocks to hide the
  // loads behind.  Measured on bfloat16, us for 256^2 / 128^2 / 64 x 128 /
  // 64^2 tiles (rows, groups, outputs, columns):
  //   forward  65536, 32, 4096, 1024:  625 / 754 /  879 / 1018
  //            14420, 132, 3330, 904:  300 / 284 /  325 /  374
  //            16384, 64, 1024, 1024:   57 /  58 /   62 /   76
  //             8198, 48,  768,  768:   25 /  28 /   25 /   27
  //             3000, 64, 1024, 1024:   53 /  37 /   26 /   32
  //             8192,  8,  256,  256:   12 /   8 /    8 /    7
  //   dweight  65536, 32, 4096, 1024:  693 / 959 / 1324 / 1397
  //            65536, 64,  256, 1024:   99 /  78 /   70 /   79
  //            28273, 179, 2072,  84:   84 /  59 /   59 /   61
  //            60000, 300,  720,  40:   60 /  45 /   42 /   31
  //             8198, 48,  768,  768:   29 /  27 /      /   31
  //            16384, 64, 1024, 1024:   81 /  75 /      /   92
  //            32768, 64, 1024, 1024:  116 / 116 /      /  151
  //
  // One tile of c at a time, where enough blocks share a CU (us with two / one
  // at 128^2): forward 28273, 179, 2072, 84: 93 / 71; 8192, 8, 1024, 1024:
  // 37 / 32; but 2048, 16, 2048, 2048: 40 / 48.
  constexpr bool kWide = sizeof(T) == 4;  // float32 has no larger ones
  constexpr long KS = 128 / sizeof(T);
  auto tile128 = [&](bool ahead) {
    if (!async)
      go(product_kernel<T, 128, 128, 2, 2, MODE, kWide>, 128, 128, 256);
    else if (ahead)
      go(product_kernel<T, 128, 128, 2, 2, MODE, true>, 128, 128, 256);
    else
      go(product_kernel<T, 128, 128, 2, 2, MODE, true, false>, 128, 128, 256);
  };
  auto tile64 = [&](bool ahead) {
    if (!async)
      go(product_kernel<T, 64, 64, 2, 2, MODE, kWide>, 64, 64, 256);
    else if (ahead)
      go(product_kernel<T, 64, 64, 2, 2, MODE, true>, 64, 64, 256);
    else
      go(product_kernel<T, 64, 64, 2, 2, MODE, true, false>, 64, 64, 256);
  };
  const long each =  // rows a group
      MODE == kDWeight ? p.C / p.G : p.M / std::min(p.G, p.M);
  auto ahead = [&](long blocks, long enough) {
    // (the float32 instructions take eight times as long: always worth it)
    return (kWide || blocks < enough) &&
           (MODE == kDWeight ? each : p.C) > 2 * KS;
  };
  if constexpr (MODE == kDWeight) {
    // 256^2 where that fills the card, its edges waste less than a third and
    // the rows of a group outlast a block's first loads
    const bool large = each >= 512 && p.G * tiles(256) >= 400 &&
                       tiles(256) * 65536 * 3 <= 4l * p.M * p.N;
    const bool middle = p.M > 64 && p.N > 64 && p.G * tiles(128) >= 256;
    if (large && async && !kWide) {
      if constexpr (!kWide)
        go(product_kernel<T, 256, 256, 2, 4, MODE, true>, 256, 256, 512);
    } else if (large || middle) {
      tile128(ahead(p.G * tiles(128), 512));
    } else {
      tile64(ahead(p.G * tiles(64), 1024));
    }
  } else {
    auto row_tiles = [&](long bm, long bn) {
      return (p.M / bm + std::min(p.G, p.M) / 2 + 1) * ((p.N + bn - 1) / bn);
    };
    const bool large = each >= 768 && p.N > 128 && row_tiles(256, 256) >= 512;
    const bool middle =
        p.N > 64 && ((each >= 192 && row_tiles(128, 128) >= 256) ||
                     (each >= 96 && row_tiles(128, 128) >= 1024));
    if (large && async && !kWide) {
      if constexpr (!kWide)
        go(product_kernel<T, 256, 256, 2, 4, MODE, true>, 256, 256, 512);
    } else if (large || middle) {
      tile128(ahead(row_tiles(128, 128), 512));
    } else if (async && p.N > 64 && row_tiles(64, 128) >= 256) {
      if (ahead(row_tiles(64, 128), 768))
        go(product_kernel<T, 64, 128, 1, 4, MODE, true>, 64, 128, 256);
      else
        go(product_kernel<T, 64, 128, 1, 4, MODE, true, false>, 64, 128, 256);
    } else {
      tile64(ahead(row_tiles(64, 64), 1024));
    }
  }
}

void narrow_dweight_launch(Product p, at::TensorOptions opt) {
  const int kw = p.N <= 64 ? 4 : 1, bf = 4 / kw * 64;
  const long tiles = (p.N + bf - 1) / bf;
  p.shift = part_shift(p.C, tiles, 2048);
  Parts parts = take_parts(p, opt);
  dim3 grid(grid_of(((long)p.C >> p.shift) + p.G + 1, 256), p.out ? tiles : 1);
  if (kw == 4)
    narrow_dweight_kernel<4><<<grid, 256, 0, stream_now()>>>(p);
  else
    narrow_dweight_kernel<1><<<grid, 256, 0, stream_now()>>>(p);
  check_launch();
  finish_launch<float>(p);
}

template <typename T>
void narrow_drows_launch(const Product& p) {
  const int lanes = lanes_for(p.N, 16 / sizeof(T));
  const long blocks = (long)p.M / 128 + p.G + 1;
  // the columns are shared among blocks where there are few row tiles
  const long parts = (p.N * sizeof(T) + 16 * lanes - 1) / (16 * lanes);
  dim3 grid(grid_of(blocks, 256),
            std::max(1l, std::min({parts, 2048 / blocks, 1024l})));
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream_now()>>>(p, lanes);
    check_launch();
  };
  if (p.C <= 4)
    go(narrow_drows_kernel<T, 4>);
  else if (p.C <= 8)
    go(narrow_drows_kernel<T, 8>);
  else
    go(narrow_drows_kernel<T, 16>);
}

at::Tensor product(const at::Tensor& a_in, const at::Tensor& weight,
                   const at::Tensor& offsets,
                   const c10::optional<at::Tensor>& bias, bool transposed) {
  const int G = (int)weight.size(0);
  const int N = (int)weight.size(transposed ? 2 : 1);
  const int C = (int)weight.size(transposed ? 1 : 2);
  c10::cuda::CUDAGuard guard(a_in.device());
  at::Tensor a = packed_rows(a_in);
  const int M = (int)a.size(0);
  at::Tensor out = at::empty({M, N}, a.options());
  if (out.numel() == 0) return out;
  Product p{ptr<void>(a), ptr<void>(weight),
            bias ? ptr<void>(*bias) : nullptr, ptr<void>(out), nullptr,
            ptr<int>(offsets), a.stride(0), transposed ? N : C, G, M, N,
            C, 0, nullptr, nullptr, 0, 0};
  SKA_TYPES(a.scalar_type(), [&] {
    if (transposed && C <= 16)
      narrow_drows_launch<T>(p);
    else if (transposed)
      product_launch<T, kDRows>(p, a.options());
    else
      product_launch<T, kForward>(p, a.options());
  });
  return out;
}

at::Tensor grouped_linear(const at::Tensor& rows, const at::Tensor& weight,
                          const at::Tensor& offsets,
                          const c10::optional<at::Tensor>& bias) {
  return product(rows, weight, offsets, bias, false);
}

at::Tensor grouped_linear_drows(const at::Tensor& dy,
                                const at::Tensor& weight,
                                const at::Tensor& offsets) {
  return product(dy, weight, offsets, c10::nullopt, true);
}

// (dweight, dbias); one that is not asked for comes back undefined.  The bias
// alone is summed in the same order as together with the weights.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>>
grouped_linear_dweight(const at::Tensor& dy_in, const at::Tensor& rows_in,
                       const at::Tensor& offsets, bool need_weight,
                       bool need_bias) {
  c10::cuda::CUDAGuard guard(dy_in.device());
  at::Tensor dy = packed_rows(dy_in), x = packed_rows(rows_in);
  const int G = (int)offsets.numel() - 1, M = (int)dy.size(0);
  const int N = (int)dy.size(1), F = (int)x.size(1);
  c10::optional<at::Tensor> dw, db;
  if (need_weight) dw = at::empty({G, N, F}, dy.options());
  if (need_bias) db = at::empty({G, N}, dy.options());
  if (N == 0 || (!need_weight && !need_bias)) return {dw, db};
  if (M == 0) {
    if (dw) dw->zero_();
    if (db) db->zero_();
    return {dw, db};
  }
  if (F == 0 && !need_bias) return {dw, db};
  // rows of no width leave the bias: any other operand does for its sums
  const at::Tensor& b = F ? x : dy;
  Product p{ptr<void>(dy), ptr<void>(b), nullptr,
            F && dw ? ptr<void>(*dw) : nullptr, db ? ptr<void>(*db) : nullptr,
            ptr<int>(offsets), dy.stride(0), b.stride(0), G, N,
            F ? F : N, M, 0, nullptr, nullptr, 0, 0};
  SKA_TYPES(dy.scalar_type(), [&] {
    if (sizeof(T) == 4 && N <= 16)
      narrow_dweight_launch(p, dy.options());
    else
      product_launch<T, kDWeight>(p, dy.options());
  });
  return {dw, db};
}

// ---------------------------------------------------------------------------
// Autograd.  In C++ because small calls are otherwise bound by the
// interpreter: sort, gather and gradient of 12289 x 2 rows took 95 us with
// autograd functions in Python, and 62 with these.
// ---------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<at::Tensor> Maybe;

bool wants(const at::Tensor& t) {
  return at::GradMode::is_enabled() && t.requires_grad();
}
bool wants(const Maybe& t) { return t && wants(*t); }

at::Tensor defined_or_none(const Maybe& t) { return t ? *t : at::Tensor(); }

// The kernels' gradients have no gradients of their own.  Where a graph of the
// backward pass is asked for, a gradient gets a node between itself and the two
// tensors it is a product of, the incoming gradient and a saved operand: a
// second differentiation that comes through it is an error, whatever else the
// loss holds, and one that does not is none of its business.
template <typename Make>
struct OnceFunction : torch::autograd::Function<OnceFunction<Make>> {
  static at::Tensor forward(AutogradContext*, const Make& make,
                            const at::Tensor&, const at::Tensor&) {
    return make();
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false,
                "grouped-row operators can be differentiated once only");
  }
};

template <typename Make>
at::Tensor once(const at::Tensor& grad, const at::Tensor& operand,
                const Make& make) {
  if (!at::GradMode::is_enabled()) return make();
  return OnceFunction<Make>::apply(make, grad,
                                   operand.defined() ? operand : grad);
}

struct GatherFunction : torch::autograd::Function<GatherFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& offsets,
                            const at::Tensor& slots) {
    ctx->save_for_backward({offsets, slots});
    return gather_rows(x, offsets, slots);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain("the gradient", grads[0]);
    auto saved = ctx->get_saved_variables();
    // a row's gradient is the sum over its places
    auto dx = once(grads[0], at::Tensor(), [&] {
      return combine_rows(grads[0], saved[0], saved[1], c10::nullopt);
    });
    return {dx, at::Tensor(), at::Tensor()};
  }
};

struct CombineFunction : torch::autograd::Function<CombineFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows,
                            const at::Tensor& offsets,
                            const at::Tensor& slots, const Maybe& weights,
                            bool need_rows, bool need_weights) {
    ctx->saved_data["rows"] = need_rows;
    ctx->saved_data["weights"] = need_weights;
    ctx->save_for_backward({need_weights ? rows : at::Tensor(), offsets,
                            slots, defined_or_none(weights)});
    return combine_rows(rows, offsets, slots, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain("the gradient", grads[0]);
    auto saved = ctx->get_saved_variables();
    const bool need_rows =
        ctx->saved_data["rows"].toBool() && ctx->needs_input_grad(0);
    const bool need_weights =
        ctx->saved_data["weights"].toBool() && ctx->needs_input_grad(3);
    const Maybe weights = saved[3].defined() ? Maybe(saved[3]) : Maybe();
    auto both = [&](bool rows, bool dots) {
      return combine_rows_backward(grads[0], dots ? saved[0] : grads[0],
                                   saved[1], saved[2], weights, rows, dots);
    };
    at::Tensor drows, dw;
    if (!at::GradMode::is_enabled()) {  // in one pass
      auto got = both(need_rows, need_weights);
      drows = defined_or_none(std::get<0>(got));
      dw = defined_or_none(std::get<1>(got));
    } else {
      if (need_rows)
        drows = once(grads[0], saved[3],
                     [&] { return *std::get<0>(both(true, false)); });
      if (need_weights)
        dw = once(grads[0], saved[0],
                  [&] { return *std::get<1>(both(false, true)); });
    }
    return {drows, at::Tensor(), at::Tensor(), dw, at::Tensor(),
            at::Tensor()};
  }
};

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows,
                            const at::Tensor& weight,
                            const at::Tensor& offsets, const Maybe& bias,
                            bool need_rows, bool need_weight,
                            bool need_bias) {
    ctx->saved_data["rows"] = need_rows;
    ctx->saved_data["weight"] = need_weight;
    ctx->saved_data["bias"] = need_bias;
    ctx->save_for_backward(
        {need_weight || need_bias ? rows : at::Tensor(),
         need_rows ? weight : at::Tensor(), offsets});
    return grouped_linear(rows, weight, offsets, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain("the gradient", grads[0]);
    auto saved = ctx->get_saved_variables();
    at::Tensor drows, dweight, dbias;
    if (ctx->saved_data["rows"].toBool() && ctx->needs_input_grad(0))
      drows = once(grads[0], saved[1], [&] {
        return grouped_linear_drows(grads[0], saved[1], saved[2]);
      });
    const bool need_weight =
        ctx->saved_data["weight"].toBool() && ctx->needs_input_grad(1);
    const bool need_bias =
        ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
    auto both = [&](bool weight, bool bias) {
      return grouped_linear_dweight(grads[0], saved[0], saved[2], weight,
                                    bias);
    };
    if (!at::GradMode::is_enabled()) {  // in one pass
      std::tuple<Maybe, Maybe> got;
      if (need_weight || need_bias) got = both(need_weight, need_bias);
      dweight = defined_or_none(std::get<0>(got));
      dbias = defined_or_none(std::get<1>(got));
    } else {
      if (need_weight)
        dweight = once(grads[0], saved[0],
                       [&] { return *std::get<0>(both(true, false)); });
      if (need_bias)
        dbias = once(grads[0], at::Tensor(),
                     [&] { return *std::get<1>(both(false, true)); });
    }
    return {drows,        dweight,      at::Tensor(), dbias,
            at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// The entry points: checks, then with or without a place in the graph.
at::Tensor gather_rows_checked(const at::Tensor& x, const at::Tensor& offsets,
                               const at::Tensor& slots) {
  check_not_traced();
  check_rows("x", x);
  const Plan plan = check_plan(x, offsets, slots);
  TORCH_CHECK_VALUE(plan.slots.size(0) == x.size(0), "x has ", x.size(0),
                    " rows, the plan ", plan.slots.size(0));
  if (!wants(x)) return gather_rows(x, plan.offsets, plan.slots);
  return GatherFunction::apply(x, plan.offsets, plan.slots);
}

at::Tensor combine_rows_checked(const at::Tensor& rows,
                                const at::Tensor& offsets,
                                const at::Tensor& slots, Maybe weights) {
  check_not_traced();
  check_rows("rows", rows);
  const Plan plan = check_plan(rows, offsets, slots);
  TORCH_CHECK_VALUE(plan.slots.numel() == rows.size(0), "rows has ",
                    rows.size(0), " rows, the plan ", plan.slots.numel());
  if (weights) {
    check_plain("weights", *weights);
    TORCH_CHECK_TYPE(
        weights->dtype() == at::kFloat || weights->dtype() == rows.dtype(),
        "weights must be float32 or ", rows.dtype(), ", got ",
        weights->dtype());
    TORCH_CHECK_VALUE(weights->device() == rows.device(), "weights are on ",
                      weights->device(), ", the rows on ", rows.device());
    TORCH_CHECK_VALUE(weights->sizes() == slots.sizes(),
                      "weights must have the ids' shape ", slots.sizes(),
                      ", got ", weights->sizes());
    if (weights->dim() == 1) weights = weights->unsqueeze(1);
    weights = whole(*weights);
  }
  if (!wants(rows) && !wants(weights))
    return combine_rows(rows, plan.offsets, plan.slots, weights);
  return CombineFunction::apply(rows, plan.offsets, plan.slots, weights,
                                wants(rows), wants(weights));
}

at::Tensor grouped_linear_checked(const at::Tensor& rows,
                                  const at::Tensor& weight_in,
                                  const at::Tensor& offsets_in, Maybe bias) {
  check_not_traced();
  check_rows("rows", rows);
  check_ints("offsets", offsets_in, rows);
  TORCH_CHECK_VALUE(weight_in.dim() == 3,
                    "weight must be [G, N, F], got shape ",
                    weight_in.sizes());
  const int64_t G = weight_in.size(0), N = weight_in.size(1);
  TORCH_CHECK_VALUE(G >= 1 && G <= kMaxGroups, "between 1 and ", kMaxGroups,
                    " groups, got ", G);
  TORCH_CHECK_VALUE(N <= kMaxWidth, "at most ", kMaxWidth, " outputs, got ",
                    N);
  TORCH_CHECK_VALUE(weight_in.size(2) == rows.size(1), "rows have ",
                    rows.size(1), " columns, weight takes ",
                    weight_in.size(2));
  TORCH_CHECK_VALUE(offsets_in.dim() == 1 && offsets_in.numel() == G + 1,
                    "offsets must have ", G + 1, " values, got shape ",
                    offsets_in.sizes());
  check_same("weight", weight_in, rows);
  if (bias) {
    check_same("bias", *bias, rows);
    TORCH_CHECK_VALUE(bias->dim() == 2 && bias->size(0) == G &&
                          bias->size(1) == N,
                      "bias must be [", G, ", ", N, "], got ",
                      bias->sizes());
    bias = whole(*bias);
  }
  const at::Tensor weight = whole(weight_in);
  const at::Tensor offsets = whole(offsets_in);
  if (!wants(rows) && !wants(weight) && !wants(bias))
    return grouped_linear(rows, weight, offsets, bias);
  return LinearFunction::apply(rows, weight, offsets, bias, wants(rows),
                               wants(weight), wants(bias));
}

// The gradients of weight and bias alone, for a solver that has dy in hand.
std::tuple<Maybe, Maybe> grouped_linear_dweight_checked(
    const at::Tensor& dy, const at::Tensor& rows, const at::Tensor& offsets,
    bool need_weight, bool need_bias) {
  check_not_traced();
  check_rows("dy", dy);
  check_rows("rows", rows);
  check_same("dy", dy, rows);
  check_ints("offsets", offsets, rows);
  TORCH_CHECK_VALUE(dy.size(0) == rows.size(0),
                    "dy and rows differ in length");
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 2 &&
                        offsets.numel() <= kMaxGroups + 1,
                    "offsets must have n_groups + 1 values");
  return grouped_linear_dweight(dy, rows, whole(offsets), need_weight,
                                need_bias);
}

}  // namespace

void bind_grouped(pybind11::module_& m) {
  m.def("group_rows", &group_rows, "stable sort of rows by group");
  m.def("gather_rows", &gather_rows_checked, "rows into group order");
  m.def("combine_rows", &combine_rows_checked,
        "weighted rows back into row order");
  m.def("grouped_linear", &grouped_linear_checked,
        "each group's rows times its weights");
  m.def("grouped_linear_dweight", &grouped_linear_dweight_checked,
        "gradients of the weights and the bias");
}
