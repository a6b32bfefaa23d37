// C-ABI implementation (include/jppgpu_lm.h): the language-model operators.  Checks of the arguments, the choice of the
// kernel, the launches; nothing is allocated and nothing is waited for.  Part of libjppgpu.so beside jppgpu_api.cc, and
// built against the fiber emulator by tests/emu like it.
#include "../../include/jppgpu_lm.h"

#include <initializer_list>
#include <tuple>
#include <utility>

#include "jpp_api.h"
#include "jpp_lm.h"
#include "k_lm_embed.h"
#include "k_lm_nce.h"
#include "k_lm_scan.h"

using namespace jpp;
using jpp_api::fail;

namespace {

// ---- launches ----------------------------------------------------------------------
// The device of the call for as long as it lasts; the caller's current device is his own (torch, a host with several GPUs).
class DeviceScope {
 public:
#if defined(JPP_EMU)
  explicit DeviceScope(int32_t device) : rc_(device == 0 ? JPPGPU_OK : fail(JPPGPU_INVALID_PARAMETER, "bad device ordinal")) {}
#else
  explicit DeviceScope(int32_t device) {
    if (hipGetDevice(&before_) != hipSuccess) {
      rc_ = fail(JPPGPU_NO_DEVICE, "jppgpu: no HIP device available (the operators have no CPU fallback)");
      return;
    }
    if (before_ == device) return;
    int count = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || device < 0 || device >= count) {
      rc_ = fail(JPPGPU_INVALID_PARAMETER, "bad device ordinal");
      return;
    }
    moved_ = hipSetDevice(device) == hipSuccess;
    if (!moved_) rc_ = fail(JPPGPU_NO_DEVICE, "hipSetDevice failed");
  }
  ~DeviceScope() {
    if (moved_) (void)hipSetDevice(before_);
  }
#endif
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  int rc() const { return rc_; }

 private:
  int rc_ = JPPGPU_OK;
#if !defined(JPP_EMU)
  int before_ = 0;
  bool moved_ = false;
#endif
};

struct Launcher {
  jpp_stream_t stream;
  int rc = JPPGPU_OK;

  template <class... P, class... A>
  void operator()(void (*kernel)(P...), u64 blocks, u32 threads, A&&... args) {
    if (rc != JPPGPU_OK || blocks == 0) return;
    const u32 grid = blocks < kLmMaxBlocks ? (u32)blocks : kLmMaxBlocks;
#if defined(JPP_EMU)
    std::tuple<P...> t(std::forward<A>(args)...);
    hip_emu::launch(dim3(grid), dim3(threads), [&] { std::apply(kernel, t); });
#else
    std::tuple<P...> t(std::forward<A>(args)...);
    void* ptrs[sizeof...(P)];
    point(t, ptrs, std::index_sequence_for<P...>());
    if (hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(threads), ptrs, 0, stream) != hipSuccess) {
      (void)hipGetLastError();
      rc = fail(JPPGPU_INVALID_STATE, "jppgpu: a kernel of a language-model operator could not be launched");
    }
#endif
  }

 private:
  template <class Tuple, size_t... I>
  static void point(Tuple& t, void** ptrs, std::index_sequence<I...>) {
    ((ptrs[I] = &std::get<I>(t)), ...);
  }
};

// Results of more bytes than this leave with the non-temporal hint: 2 031 616 rows of 128 columns looked up in 101 us, without
// it 162; the recurrence over 65 536 rows of 1 024 columns 134 us and 152, over 40 001 of 1 000 with its gradient 220 and 236.  Smaller
// ones stay where their reader finds them.
constexpr u64 kStreamBytes = u64{64} << 20;
bool streamed(u64 bytes) { return bytes > kStreamBytes; }

u64 div_up(u64 a, u64 b) { return (a + b - 1) / b; }

// ---- checks --------------------------------------------------------------------------
constexpr int64_t kMaxDim = 1 << 24, kMaxRows = int64_t{1} << 40, kMaxStride = 0xffffffff;
constexpr int64_t kMaxIndex = 0x7fffffff;   // words, packed rows, sentences, entries of a sum by word

int bytes_of(int32_t type) { return type == JPPGPU_LM_F32 ? 4 : 2; }

int32_t type_of(const jppgpu_lm_matrix* m) { return m->type & ~JPPGPU_LM_CLEAR_REST; }
bool cleared(const jppgpu_lm_matrix* m) { return (m->type & JPPGPU_LM_CLEAR_REST) != 0; }

enum Need { kNeeded, kOptional, kBatchResult };   // (kBatchResult: needed, and may have its other rows cleared)

// nullptr, or what is wrong with the matrix
const char* bad_matrix(const jppgpu_lm_matrix* m, int64_t rows, int64_t dim, Need need) {
  if (m == nullptr) return need == kOptional ? nullptr : "a matrix is missing";
  if (m->reserved != 0) return "jppgpu_lm_matrix::reserved is not 0";
  const int32_t type = need == kBatchResult ? type_of(m) : m->type;
  if (type != JPPGPU_LM_F32 && type != JPPGPU_LM_BF16 && type != JPPGPU_LM_F16) return "unknown element type";
  if (m->data == nullptr) return need == kOptional || rows == 0 ? nullptr : "a matrix has no data";
  if (reinterpret_cast<uintptr_t>(m->data) % (uintptr_t)bytes_of(type) != 0) return "a matrix does not start on an element";
  if (m->stride < dim || m->stride > kMaxStride) return "the stride of a matrix is shorter than its rows, or beyond 2^32 - 1";
  return nullptr;
}

bool given(const jppgpu_lm_matrix* m) { return m != nullptr && m->data != nullptr; }

const char* bad_ids(const jppgpu_lm_ids* ids, int64_t n) {
  if (ids == nullptr) return "the ids are missing";
  if (ids->reserved != 0) return "jppgpu_lm_ids::reserved is not 0";
  if (ids->bytes != 4 && ids->bytes != 8) return "ids are int32 or int64";
  if (n > 0 && ids->data == nullptr) return "the ids are missing";
  if (reinterpret_cast<uintptr_t>(ids->data) % (uintptr_t)ids->bytes != 0) return "the ids do not start on an id";
  return nullptr;
}

const char* bad_f32(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 != 0 ? "an array of floats does not start on a float" : nullptr; }

LmIds ids_of(const jppgpu_lm_ids* ids) { return LmIds{ids->data, ids->bytes == 8 ? 1u : 0u}; }

// one of the inputs is this very matrix
bool same_start(const void* out, std::initializer_list<const void*> others) {
  for (const void* o : others)
    if (out != nullptr && out == o) return true;
  return false;
}

#define JPP_LM_REFUSE_IF(what)                                        \
  do {                                                                \
    if (const char* why = (what)) return fail(JPPGPU_INVALID_PARAMETER, why); \
  } while (0)
#define JPP_LM_CHECK(ok, why)                                   \
  do {                                                          \
    if (!(ok)) return fail(JPPGPU_INVALID_PARAMETER, why);      \
  } while (0)

// ---- workspaces ------------------------------------------------------------------------
constexpr u64 kAlign = 256;

struct Carver {
  char* base;
  u64 used = 0;
  template <class E>
  E* take(u64 count) {
    E* p = reinterpret_cast<E*>(base + used);
    used += div_up(count * sizeof(E), kAlign) * kAlign;
    return p;
  }
};

int bad_workspace(const void* p, uint64_t bytes, uint64_t need) {
  if (need == 0) return JPPGPU_OK;
  if (p == nullptr || bytes < need) return fail(JPPGPU_INVALID_PARAMETER, "the workspace is smaller than the operator's ..._workspace() says");
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return fail(JPPGPU_INVALID_PARAMETER, "the workspace does not start on 16 bytes");
  return JPPGPU_OK;
}

// ---- sums by word --------------------------------------------------------------------
constexpr u64 kL2Bytes = u64{4} << 20;   // of an XCD

struct SumPlan {
  u32 n, dim, keyBits, passes, sortRounds, sortTiles, pack, lanes, part, tile, tiles, colBlocks;
  bool one, weighted;
  char *a, *b;           // entries
  u32 *counts, *totals, *spanCount, *span;
  float *head, *tail;

  // n entries, `perToken` of them read one row of src.  The tiles, and with them the workspace, follow from the sizes
  // alone, not from the type of src.
  SumPlan(u64 n_, u64 vocab, u64 dim_, u64 perToken, bool weighted_, i32 type = JPPGPU_LM_F32) : n((u32)n_), dim((u32)dim_), weighted(weighted_) {
    keyBits = 1;
    while ((vocab >> keyBits) != 0) ++keyBits;   // (keys 0 .. vocab)
    passes = (keyBits + 7) / 8;
    one = n <= kLmSortOne;   // (1 003 rows, 100 columns, 30 000 words: 16 us, 25 with the kernels for many)
    // entries of a thread: two as long as that makes no more tiles than a workgroup looks back on by itself (37 us for the
    // loss of 1 021 tokens, 50 with eight), eight where that leaves two workgroups a compute unit (2.2 M entries: 5 us more
    // with four, 24 with two; in workgroups of 1 024 threads half as long again), four between (507 904 ids: 5 us less than
    // with eight)
    sortRounds = n <= kLmSortOwn * kLmThreads * 2 ? 2 : n <= 512u * kLmThreads * 8 ? 4 : 8;
    sortTiles = (u32)div_up(n, kLmThreads * sortRounds);
    // rows that are read again and do not fit one L2: cache lines of 128 bytes spread over the XCDs (k_lm_seg_sum; the step on
    // 65 536 tokens: 300 us, 39 more without)
    const bool sliced = perToken > 1 && dim >= 64 && n / perToken * dim * 2 > kL2Bytes;
    pack = dim < 4 ? 1 : sliced && bytes_of(type) == 2 ? 8 : 4;
    lanes = sliced || dim <= 32 ? 8 : dim <= 64 ? 16 : dim <= 128 ? 32 : 64;
    colBlocks = (u32)div_up(div_up(dim, pack), lanes);
    // parts long enough that words rarely cross them, short enough that some eight thousand wavefronts share the work
    // (507 904 rows: a third longer in parts of 8; 1 003 rows: 16 us, 27 in parts of 64)
    part = 8;
    while (part < 64 && (u64)n * div_up(dim, 256) / (part * 2) >= 8192) part *= 2;
    tile = part * (kLmThreads / lanes);
    tiles = (u32)div_up(n, tile);
  }
  u64 carve(void* ws) {
    Carver c{static_cast<char*>(ws)};
    const u64 bytes = (u64)n * (weighted ? sizeof(LmEntry) : sizeof(LmPair));
    a = c.take<char>(bytes);
    b = passes > 1 && !one ? c.take<char>(bytes) : nullptr;
    counts = one ? nullptr : c.take<u32>((u64)kLmBins * sortTiles);
    totals = one ? nullptr : c.take<u32>(kLmBins);
    spanCount = c.take<u32>(2);
    span = c.take<u32>(tiles);
    head = c.take<float>((u64)tiles * dim);
    tail = c.take<float>((u64)tiles * dim);
    return c.used;
  }
};

LmZero zero_of(float* data, i64 stride, u64 rows, u64 cols) {
  constexpr u64 kPiece = 4096;
  const u64 total = rows * cols;
  if (stride != (i64)cols || total == 0) return LmZero{data, stride, rows, (u32)cols, (u32)cols};
  const u64 pieces = div_up(total, kPiece);
  return LmZero{data, (i64)kPiece, pieces, (u32)kPiece, (u32)(total - (pieces - 1) * kPiece)};
}
u64 zero_blocks(const LmZero& z) { return z.rows < 2048 ? z.rows : 2048; }

template <class T, class E>
void launch_seg_sum(Launcher& go, const LmSeg<E>& q, u32 pack, u32 lanes, const void* src) {
  const u64 blocks = (u64)q.tiles * q.colBlocks;
  const typename T::store* s = static_cast<const typename T::store*>(src);
  if (pack == 1) {
    go(k_lm_seg_sum<T, 1, 8, E>, blocks, kLmThreads, q, s);
    return;
  }
  if constexpr (sizeof(typename T::store) == 2 && E::kWeighted) {
    if (pack == 8) {
      go(k_lm_seg_sum<T, 8, 8, E>, blocks, kLmThreads, q, s);
      return;
    }
  }
  switch (lanes) {
    case 8: go(k_lm_seg_sum<T, 4, 8, E>, blocks, kLmThreads, q, s); break;
    case 16: go(k_lm_seg_sum<T, 4, 16, E>, blocks, kLmThreads, q, s); break;
    case 32: go(k_lm_seg_sum<T, 4, 32, E>, blocks, kLmThreads, q, s); break;
    default: go(k_lm_seg_sum<T, 4, 64, E>, blocks, kLmThreads, q, s); break;
  }
}

// what sum_by_word sums
struct SumSource {
  const jppgpu_lm_ids* ids;
  u32 vocab, perToken;
  float scale;
  const float* weights;   // or null
  const jppgpu_lm_matrix* src;
  float* grad;
  i64 gradStride;
};

template <class E, class Keys>
void sort_pass(Launcher& go, const SumPlan& p, const Keys& keys, u32 shift, u32 bits, const LmZero& zero, E* to) {
  const u64 zeroBlocks = zero_blocks(zero);
  const u32 mask = (1u << bits) - 1;
  auto pass = [&](auto rounds) {
    constexpr int R = decltype(rounds)::value;
    go(k_lm_sort_count<R, Keys>, p.sortTiles + zeroBlocks, kLmThreads, keys, p.n, shift, mask, p.counts, p.sortTiles, p.spanCount, zero);
    if (p.sortTiles > kLmSortOwn) go(k_lm_sort_scan, kLmBins, kLmThreads, p.counts, p.sortTiles, p.totals);
    go(k_lm_sort_scatter<R, E, Keys>, p.sortTiles, kLmThreads, keys, p.n, shift, bits, p.counts, p.sortTiles, p.totals, to);
  };
  if (p.sortRounds == 2) pass(LmConst<2>());
  else if (p.sortRounds == 4) pass(LmConst<4>());
  else pass(LmConst<8>());
}

template <class E>
void sum_entries(Launcher& go, SumPlan& p, const SumSource& x) {
  const LmZero zero = zero_of(x.grad, x.gradStride, x.vocab, p.dim);
  const LmKeysOfIds<E> keys{ids_of(x.ids), x.vocab, x.perToken, LmDiv::by(x.perToken), x.weights};
  E *a = reinterpret_cast<E*>(p.a), *b = reinterpret_cast<E*>(p.b), *sorted = a;
  if (p.one) {
    go(k_lm_sort_one<E>, 1 + zero_blocks(zero), (u32)kLmOneThreads, keys, p.n, p.keyBits, p.passes, a, p.spanCount, zero);
  } else {
    const u32 digit = (p.keyBits + p.passes - 1) / p.passes;
    const LmZero none{nullptr, 0, 0, 0, 0};
    E *from = nullptr, *to = a;
    for (u32 pass = 0; pass < p.passes; ++pass) {
      const u32 shift = pass * digit;
      if (pass == 0) sort_pass(go, p, keys, shift, digit, zero, to);
      else sort_pass(go, p, LmKeysOfPass<E>{from}, shift, digit, none, to);
      sorted = from = to;
      to = to == a ? b : a;
    }
  }
  LmSeg<E> q{};
  q.entries = sorted;
  q.n = p.n;
  q.part = p.part;
  q.tile = p.tile;
  q.tiles = p.tiles;
  q.vocab = x.vocab;
  q.dim = p.dim;
  q.colBlocks = p.colBlocks;
  q.scale = x.scale;
  q.srcStride = (u32)x.src->stride;
  q.grad = x.grad;
  q.gradStride = x.gradStride;
  q.head = p.head;
  q.tail = p.tail;
  q.span = p.span;
  q.spanCount = p.spanCount;
  switch (x.src->type) {
    case JPPGPU_LM_F32: launch_seg_sum<LmF32, E>(go, q, p.pack, p.lanes, x.src->data); break;
    case JPPGPU_LM_BF16: launch_seg_sum<LmBf16, E>(go, q, p.pack, p.lanes, x.src->data); break;
    default: launch_seg_sum<LmF16, E>(go, q, p.pack, p.lanes, x.src->data); break;
  }
  if (p.tiles > 1) {
    const u32 pack = p.dim < 4 ? 1 : 4;
    const u64 most = (u64)p.tiles * div_up(p.dim, 64 * pack), blocks = most < 2048 ? most : 2048;
    if (pack == 4) go(k_lm_seg_join<4, E>, blocks, 64u * kLmJoinWaves, q);
    else go(k_lm_seg_join<1, E>, blocks, 64u * kLmJoinWaves, q);
  }
}

// grad = the sums by word of the weighted rows of src (jppgpu_lm.h); n > 0
void sum_by_word(Launcher& go, SumPlan& p, const SumSource& x) {
  if (p.weighted) sum_entries<LmEntry>(go, p, x);
  else sum_entries<LmPair>(go, p, x);
}

// the gradient of a table that nothing reads
void clear_matrix(Launcher& go, const jppgpu_lm_matrix* m, u64 rows, u64 cols) {
  const LmZero z = zero_of(static_cast<float*>(m->data), m->stride, rows, cols);
  go(k_lm_zero, zero_blocks(z), kLmThreads, z);
}

template <class Tin, class Tout, int V, int PER, bool STREAM>
void launch_embed_packs(Launcher& go, const jppgpu_lm_matrix* table, u32 vocab, u32 dim, LmIds ids, u64 n, float scale, const jppgpu_lm_matrix* out) {
  const u32 packs = (u32)div_up(dim, V), per = PER * kLmThreads;
  const u32 rows = packs >= per ? 1 : per / packs;
  go(k_lm_embed<Tin, Tout, V, PER, STREAM>, div_up(n, rows), kLmThreads, static_cast<const typename Tin::store*>(table->data), table->stride,
     vocab, dim, ids, n, scale, static_cast<typename Tout::store*>(out->data), out->stride, rows);
}

template <class Tin, class Tout>
void launch_embed(Launcher& go, const jppgpu_lm_matrix* table, u32 vocab, u32 dim, LmIds ids, u64 n, float scale, const jppgpu_lm_matrix* out) {
  constexpr int V = 16 / sizeof(typename Tout::store);   // a 16-byte store a lane
  // four packs a thread once that still fills the chip's wavefront slots (2 031 616 rows of 128 columns: 101 us, 182 with one)
  if (dim < (u32)V) launch_embed_packs<Tin, Tout, 1, 1, false>(go, table, vocab, dim, ids, n, scale, out);
  else if (n * div_up(dim, V) < (u64)4 * 256 * 2048) launch_embed_packs<Tin, Tout, V, 1, false>(go, table, vocab, dim, ids, n, scale, out);
  else if (!streamed(n * dim * sizeof(typename Tout::store))) launch_embed_packs<Tin, Tout, V, 4, false>(go, table, vocab, dim, ids, n, scale, out);
  else launch_embed_packs<Tin, Tout, V, 4, true>(go, table, vocab, dim, ids, n, scale, out);
}

// ---- the recurrence --------------------------------------------------------------------
// Columns of a wavefront: a lane takes 4 of a long row, fewer where that leaves lanes idle (128 columns of floats with the
// gradient: 464 us with two, 479 with one, 467 with four; 1 024 of bfloat16: 134 us with four, 163 with one).  The gradient
// holds eight rows of five values an element in registers, so a lane takes 8 bytes a row there.
u32 scan_pack(u32 dim, i32 type, bool grad) {
  const u32 most = grad && type == JPPGPU_LM_F32 ? 2 : 4;
  const u32 v = dim <= 64 ? 1u : dim <= 128 ? 2u : 4u;
  return v < most ? v : most;
}

// Whether the rows are walked in chunks, and of how many rows (0: a wavefront per sentence and column block).  Decided from
// the sizes alone, not from the type, so that one workspace rule serves all.  Sentences of up to 256 rows are walked, and
// longer ones where there are enough of about one length to fill the chip: a step of 64 sentences takes 10 us, 46 in chunks;
// 16 384 sentences of 31 rows of 128 floats with the gradient 464, 520 in chunks.  Five documents of 40 001 rows of
// 1 000 columns with the gradient: 220 us in chunks, 8.1 ms walked.  4 096 wavefronts: 6 144 and 8 192 took 8 and 4 % longer over 65 536
// rows of 1 024 columns.
u32 scan_chunk(u64 rows, u64 n, u64 dim, u64 maxLen) {
  const u64 longest = maxLen == 0 || maxLen > rows ? rows : maxLen;
  const u64 blocks = div_up(dim, 256);
  if (longest <= 256) return 0;
  if (n * blocks >= 2048 && longest <= 4 * (rows / n)) return 0;
  const u64 chunk = div_up(div_up(rows * blocks, 4096), kLmSave) * kLmSave;
  return (u32)(chunk < 32 ? 32 : chunk < (1u << 30) ? chunk : 1u << 30);
}

// Workgroups of a kernel that walks sentences: a wavefront each and column block, and where rows of no sentence are to be cleared,
// of which the host does not know how many there are, one for 64 KB of all rows, up to four a compute unit.
template <class T>
u64 scan_blocks(const LmScan<T>& q) {
  const u64 blocks = div_up((u64)q.n * q.colBlocks, kLmThreads / 64), rest = div_up((u64)q.rows * q.dim * sizeof(typename T::store), 1 << 16);
  return q.clear == 0 || rest <= blocks ? blocks : blocks > 1024 ? blocks : rest < 1024 ? rest : 1024;
}

template <class T, int V, bool STREAM>
void launch_scan(Launcher& go, const LmScan<T>& q) {
  const u64 waves = kLmThreads / 64;
  if (q.chunk == 0) {
    const u64 blocks = scan_blocks(q);
    if (q.saved != nullptr) go(k_lm_scan_seq<T, V, true, STREAM>, blocks, kLmThreads, q);
    else go(k_lm_scan_seq<T, V, false, STREAM>, blocks, kLmThreads, q);
    return;
  }
  const u64 blocks = div_up((u64)q.chunks * q.colBlocks, waves), groups = div_up(q.chunks, kLmGroup) * q.colBlocks;
  go(k_lm_scan_agg<T, V>, groups, kLmThreads, q);
  go(k_lm_scan_carry<false>, div_up(q.dim, kLmCarryCols), kLmCarryCols * kLmCarryRuns, q.groupW, q.groupB, (u32)div_up(q.chunks, kLmGroup), q.dim);
  if (q.saved != nullptr) go(k_lm_scan_chunk<T, V, true, STREAM>, blocks, kLmThreads, q);
  else go(k_lm_scan_chunk<T, V, false, STREAM>, blocks, kLmThreads, q);
}

template <class T, int V, bool STREAM>
void launch_scan_grad(Launcher& go, const LmScan<T>& q) {
  const u64 waves = kLmThreads / 64;
  if (q.chunk == 0) {
    go(k_lm_scan_grad_seq<T, V, STREAM>, scan_blocks(q), kLmThreads, q);
    return;
  }
  const u64 blocks = div_up((u64)q.chunks * q.colBlocks, waves), groups = div_up(q.chunks, kLmGroup) * q.colBlocks;
  go(k_lm_scan_grad_agg<T, V>, groups, kLmThreads, q);
  go(k_lm_scan_carry<true>, div_up(q.dim, kLmCarryCols), kLmCarryCols * kLmCarryRuns, q.groupW, q.groupB, (u32)div_up(q.chunks, kLmGroup), q.dim);
  go(k_lm_scan_grad_chunk<T, V, STREAM>, blocks, kLmThreads, q);
}

template <class T, int V>
void launch_scan_any(Launcher& go, const LmScan<T>& q, bool grad) {
  const bool stream = streamed((u64)q.rows * q.dim * sizeof(typename T::store));
  if (!grad) {
    if (stream) launch_scan<T, V, true>(go, q);
    else launch_scan<T, V, false>(go, q);
  } else if constexpr (V * sizeof(typename T::store) <= 8) {
    if (stream) launch_scan_grad<T, V, true>(go, q);
    else launch_scan_grad<T, V, false>(go, q);
  }
}

void carve_maps(Carver& c, u64 chunks, u64 dim, float** aggW, float** aggB, float** groupW, float** groupB) {
  *aggW = c.take<float>(chunks * dim);
  *aggB = c.take<float>(chunks * dim);
  *groupW = c.take<float>(div_up(chunks, kLmGroup) * dim);
  *groupB = c.take<float>(div_up(chunks, kLmGroup) * dim);
}

struct ScanArgs {
  const jppgpu_lm_matrix *gate, *x, *state, *h, *last, *dh, *dlast, *dgate, *dx, *dstate;
  const int32_t* offsets;
  int64_t n, rows, dim, maxLen;
  float* saved;
  void* workspace;
};

template <class T>
void run_scan(Launcher& go, const ScanArgs& s, bool grad) {
  typedef typename T::store S;
  LmScan<T> q{};
  q.gate = static_cast<const S*>(s.gate->data);
  q.gateStride = s.gate->stride;
  q.x = static_cast<const S*>(s.x->data);
  q.xStride = s.x->stride;
  q.offsets = s.offsets;
  q.n = (u32)s.n;
  q.rows = (u32)s.rows;
  q.dim = (u32)s.dim;
  if (given(s.state)) {
    q.state = static_cast<const float*>(s.state->data);
    q.stateStride = s.state->stride;
  }
  q.saved = s.saved;
  if (!grad) {
    q.clear = cleared(s.h) ? kLmClearRows : 0;
    q.h = static_cast<S*>(s.h->data);
    q.hStride = s.h->stride;
    if (given(s.last)) {
      q.last = static_cast<float*>(s.last->data);
      q.lastStride = s.last->stride;
    }
  } else {
    q.clear = (cleared(s.dgate) ? kLmClearDgate : 0) | (cleared(s.dx) ? kLmClearDx : 0);
    q.dh = static_cast<const S*>(s.dh->data);
    q.dhStride = s.dh->stride;
    q.dgate = static_cast<S*>(s.dgate->data);
    q.dgateStride = s.dgate->stride;
    q.dx = static_cast<S*>(s.dx->data);
    q.dxStride = s.dx->stride;
    if (given(s.dlast)) {
      q.dlast = static_cast<const float*>(s.dlast->data);
      q.dlastStride = s.dlast->stride;
    }
    if (given(s.dstate)) {
      q.dstate = static_cast<float*>(s.dstate->data);
      q.dstateStride = s.dstate->stride;
    }
  }
  const u32 v = scan_pack(q.dim, s.x->type, grad);
  q.colBlocks = (u32)div_up(div_up(q.dim, v), 64);
  q.chunk = s.n == 0 ? 0 : scan_chunk((u64)s.rows, (u64)s.n, (u64)s.dim, (u64)s.maxLen);
  if (q.chunk != 0) {
    q.chunks = (u32)div_up(q.rows, q.chunk);
    Carver c{static_cast<char*>(s.workspace)};
    carve_maps(c, q.chunks, q.dim, &q.aggW, &q.aggB, &q.groupW, &q.groupB);
  }
  if (v == 1) launch_scan_any<T, 1>(go, q, grad);
  else if (v == 2) launch_scan_any<T, 2>(go, q, grad);
  else launch_scan_any<T, 4>(go, q, grad);
}

int check_scan(const ScanArgs& s) {
  JPP_LM_CHECK(s.dim >= 1 && s.dim <= kMaxDim, "dim outside 1 .. 2^24");
  JPP_LM_CHECK(s.n >= 0 && s.n <= kMaxIndex - 1 && s.rows >= 0 && s.rows <= kMaxIndex, "n or rows outside 0 .. 2^31 - 1");
  JPP_LM_CHECK(s.maxLen >= 0, "max_len < 0");
  JPP_LM_CHECK(s.n == 0 || s.offsets != nullptr, "the offsets are missing");
  JPP_LM_CHECK(reinterpret_cast<uintptr_t>(s.offsets) % 4 == 0, "the offsets do not start on an int32");
  JPP_LM_REFUSE_IF(bad_matrix(s.gate, s.rows, s.dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_matrix(s.x, s.rows, s.dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_matrix(s.state, s.n, s.dim, kOptional));
  JPP_LM_CHECK(s.gate->type == s.x->type, "gate and x are of one type");
  JPP_LM_CHECK(!given(s.state) || s.state->type == JPPGPU_LM_F32, "states are 32-bit");
  return JPPGPU_OK;
}

uint64_t scan_workspace(int64_t rows, int64_t n, int64_t dim, int64_t max_len) {
  if (rows == 0 || n == 0) return 0;
  const u32 chunk = scan_chunk((u64)rows, (u64)n, (u64)dim, (u64)max_len);
  if (chunk == 0) return 0;
  Carver c{nullptr};
  float* none;
  carve_maps(c, div_up((u64)rows, chunk), (u64)dim, &none, &none, &none, &none);
  return c.used;
}

// ---- noise-contrastive score and loss ------------------------------------------------------
template <class T, int G, int NV, LmRowKind KIND>
void launch_nce(Launcher& go, const LmNce& q, const void* h, const void* table, LmIds ids, void* dh, bool loss) {
  constexpr int V = 16 / (int)sizeof(typename T::store);
  auto hp = static_cast<const typename T::store*>(h);
  auto tp = static_cast<const typename T::store*>(table);
  auto dp = static_cast<typename T::store*>(dh);
  if (!loss) {
    go(k_lm_nce_score<T, V, G, NV, KIND>, div_up(q.n * div_up(q.cands, kLmScoreCands), kLmThreads / G), kLmThreads, q, hp, tp, ids);
    return;
  }
  // at most kLmChipBlocks workgroups: a wavefront that goes from token to token has the next one's data ahead.  (These kernels
  // have 82 to 181 registers a lane, so that a compute unit holds five to two of the eight workgroups at a time.)
  const u64 blocks = div_up(q.n, kLmThreads / 64), most = blocks < kLmChipBlocks ? blocks : kLmChipBlocks;
  if (dp != nullptr) go(k_lm_nce_loss<T, V, G, NV, KIND, true>, most, kLmThreads, q, hp, tp, ids, dp);
  else go(k_lm_nce_loss<T, V, G, NV, KIND, false>, most, kLmThreads, q, hp, tp, ids, dp);
}

template <class T, int G, int NV>
void launch_nce_row(Launcher& go, const LmNce& q, const void* h, const void* table, LmIds ids, void* dh, bool loss) {
  if (q.dim == G * NV * (16 / sizeof(typename T::store))) launch_nce<T, G, NV, kLmFull>(go, q, h, table, ids, dh, loss);
  else launch_nce<T, G, NV, kLmPart>(go, q, h, table, ids, dh, loss);
}

// packs of 16 bytes of the longest row that a wavefront holds in registers; longer ones are walked in blocks
constexpr u32 kNcePacks = 256;
u32 nce_packs(u32 dim, i32 type) { return dim / (16 / (u32)bytes_of(type)); }

template <class T>
void run_nce(Launcher& go, const LmNce& q, const void* h, const void* table, LmIds ids, void* dh, bool loss) {
  const u32 packs = q.dim / (16 / (u32)sizeof(typename T::store));
  if (packs <= 16) launch_nce_row<T, 16, 1>(go, q, h, table, ids, dh, loss);
  else if (packs <= 32) launch_nce_row<T, 16, 2>(go, q, h, table, ids, dh, loss);
  else if (packs <= 64) launch_nce_row<T, 16, 4>(go, q, h, table, ids, dh, loss);
  else if (packs <= 128) launch_nce_row<T, 64, 2>(go, q, h, table, ids, dh, loss);
  else if (packs <= kNcePacks) launch_nce_row<T, 64, 4>(go, q, h, table, ids, dh, loss);
  else launch_nce<T, 64, 4, kLmBlocks>(go, q, h, table, ids, dh, loss);
}

void dispatch_nce(Launcher& go, const LmNce& q, const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* table, LmIds ids, void* dh, bool loss) {
  switch (h->type) {
    case JPPGPU_LM_F32: run_nce<LmF32>(go, q, h->data, table->data, ids, dh, loss); break;
    case JPPGPU_LM_BF16: run_nce<LmBf16>(go, q, h->data, table->data, ids, dh, loss); break;
    default: run_nce<LmF16>(go, q, h->data, table->data, ids, dh, loss); break;
  }
}

int check_nce(const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim, const jppgpu_lm_ids* ids, int64_t n, int64_t cands) {
  JPP_LM_CHECK(dim >= 1 && dim <= kMaxDim, "dim outside 1 .. 2^24");
  JPP_LM_CHECK(vocab >= 0 && vocab < kMaxIndex, "vocab outside 0 .. 2^31 - 2");
  JPP_LM_CHECK(n >= 0 && n < kMaxRows, "n outside 0 .. 2^40 - 1");
  JPP_LM_CHECK(cands >= 1 && cands <= kMaxIndex, "cands outside 1 .. 2^31 - 1");
  JPP_LM_CHECK(n <= kMaxRows / cands, "more than 2^40 candidates");
  JPP_LM_REFUSE_IF(bad_matrix(h, n, dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_matrix(table, vocab, dim, kNeeded));
  JPP_LM_CHECK(h->type == table->type, "h and the table are of one type");
  JPP_LM_REFUSE_IF(bad_ids(ids, n));
  return JPPGPU_OK;
}

// the loss's scratch: the gradients of the scores, then the sum by word
uint64_t nce_workspace(int64_t n, int64_t cands, int64_t vocab, int64_t dim) {
  if (n == 0) return 0;
  const u64 entries = (u64)n * (u64)cands;
  Carver c{nullptr};
  c.take<float>(entries);
  SumPlan p(entries, (u64)vocab, (u64)dim, (u64)cands, true);
  return c.used + p.carve(nullptr);
}

}  // namespace

// ---- entry points ----------------------------------------------------------------------------
extern "C" int jppgpu_lm_embed(const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim, const jppgpu_lm_ids* ids, int64_t n, float scale,
                               const jppgpu_lm_matrix* out, int32_t device, void* stream) {
  JPP_LM_CHECK(dim >= 1 && dim <= kMaxDim, "dim outside 1 .. 2^24");
  JPP_LM_CHECK(vocab >= 0 && vocab < kMaxIndex, "vocab outside 0 .. 2^31 - 2");
  JPP_LM_CHECK(n >= 0 && n < kMaxRows, "n outside 0 .. 2^40 - 1");
  JPP_LM_REFUSE_IF(bad_matrix(table, vocab, dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_matrix(out, n, dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_ids(ids, n));
  JPP_LM_CHECK(out->type == table->type || table->type == JPPGPU_LM_F32, "the rows are of the table's type, or 16-bit from a 32-bit table");
  JPP_LM_CHECK(!same_start(out->data, {table->data, ids->data}), "the output overlaps an input");
  DeviceScope scope(device);
  if (scope.rc() != JPPGPU_OK) return scope.rc();
  if (n == 0) return JPPGPU_OK;
  Launcher go{static_cast<jpp_stream_t>(stream)};
  const LmIds id = ids_of(ids);
  if (out->type == JPPGPU_LM_F32) launch_embed<LmF32, LmF32>(go, table, (u32)vocab, (u32)dim, id, (u64)n, scale, out);
  else if (out->type == JPPGPU_LM_BF16 && table->type == JPPGPU_LM_F32) launch_embed<LmF32, LmBf16>(go, table, (u32)vocab, (u32)dim, id, (u64)n, scale, out);
  else if (out->type == JPPGPU_LM_BF16) launch_embed<LmBf16, LmBf16>(go, table, (u32)vocab, (u32)dim, id, (u64)n, scale, out);
  else if (table->type == JPPGPU_LM_F32) launch_embed<LmF32, LmF16>(go, table, (u32)vocab, (u32)dim, id, (u64)n, scale, out);
  else launch_embed<LmF16, LmF16>(go, table, (u32)vocab, (u32)dim, id, (u64)n, scale, out);
  return go.rc;
}

extern "C" int jppgpu_lm_embed_grad_workspace(int64_t n, int64_t vocab, int64_t dim, uint64_t* bytes) {
  JPP_LM_CHECK(bytes != nullptr, "null argument");
  JPP_LM_CHECK(dim >= 1 && dim <= kMaxDim, "dim outside 1 .. 2^24");
  JPP_LM_CHECK(vocab >= 0 && vocab < kMaxIndex, "vocab outside 0 .. 2^31 - 2");
  JPP_LM_CHECK(n >= 0 && n <= kMaxIndex, "n outside 0 .. 2^31 - 1");
  *bytes = 0;
  if (n > 0) {
    SumPlan p((u64)n, (u64)vocab, (u64)dim, 1, false);
    *bytes = p.carve(nullptr);
  }
  return JPPGPU_OK;
}

extern "C" int jppgpu_lm_embed_grad(const jppgpu_lm_matrix* dy, const jppgpu_lm_ids* ids, int64_t n, int64_t vocab, int64_t dim, float scale,
                                    const jppgpu_lm_matrix* grad, void* workspace, uint64_t workspace_bytes, int32_t device, void* stream) {
  uint64_t need = 0;
  if (int rc = jppgpu_lm_embed_grad_workspace(n, vocab, dim, &need)) return rc;
  JPP_LM_REFUSE_IF(bad_matrix(dy, n, dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_matrix(grad, vocab, dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_ids(ids, n));
  JPP_LM_CHECK(grad->type == JPPGPU_LM_F32, "the gradient of a table is 32-bit");
  JPP_LM_CHECK(!same_start(grad->data, {dy->data, ids->data, workspace}), "the output overlaps an input");
  if (int rc = bad_workspace(workspace, workspace_bytes, need)) return rc;
  DeviceScope scope(device);
  if (scope.rc() != JPPGPU_OK) return scope.rc();
  if (vocab == 0) return JPPGPU_OK;
  Launcher go{static_cast<jpp_stream_t>(stream)};
  if (n == 0) {
    clear_matrix(go, grad, (u64)vocab, (u64)dim);
    return go.rc;
  }
  SumPlan p((u64)n, (u64)vocab, (u64)dim, 1, false, dy->type);
  p.carve(workspace);
  sum_by_word(go, p, SumSource{ids, (u32)vocab, 1, scale, nullptr, dy, static_cast<float*>(grad->data), grad->stride});
  return go.rc;
}

extern "C" int64_t jppgpu_lm_scan_saved(int64_t rows) { return rows > 0 ? (int64_t)div_up((u64)rows, kLmSave) : 0; }

extern "C" int jppgpu_lm_scan_workspace(int64_t rows, int64_t n, int64_t dim, int64_t max_len, uint64_t* bytes) {
  JPP_LM_CHECK(bytes != nullptr, "null argument");
  JPP_LM_CHECK(dim >= 1 && dim <= kMaxDim, "dim outside 1 .. 2^24");
  JPP_LM_CHECK(n >= 0 && n <= kMaxIndex - 1 && rows >= 0 && rows <= kMaxIndex, "n or rows outside 0 .. 2^31 - 1");
  JPP_LM_CHECK(max_len >= 0, "max_len < 0");
  *bytes = scan_workspace(rows, n, dim, max_len);
  return JPPGPU_OK;
}

extern "C" int jppgpu_lm_scan(const jppgpu_lm_matrix* gate, const jppgpu_lm_matrix* x, const int32_t* offsets, int64_t n, int64_t rows, int64_t dim,
                              int64_t max_len, const jppgpu_lm_matrix* state, const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* last,
                              float* saved, void* workspace, uint64_t workspace_bytes, int32_t device, void* stream) {
  ScanArgs s{};
  s.gate = gate;
  s.x = x;
  s.state = state;
  s.h = h;
  s.last = last;
  s.offsets = offsets;
  s.n = n;
  s.rows = rows;
  s.dim = dim;
  s.maxLen = max_len;
  s.saved = saved;
  s.workspace = workspace;
  if (int rc = check_scan(s)) return rc;
  JPP_LM_REFUSE_IF(bad_matrix(h, rows, dim, kBatchResult));
  JPP_LM_REFUSE_IF(bad_matrix(last, n, dim, kOptional));
  JPP_LM_REFUSE_IF(bad_f32(saved));
  JPP_LM_CHECK(type_of(h) == x->type, "h is of the type of x");
  JPP_LM_CHECK(!given(last) || last->type == JPPGPU_LM_F32, "states are 32-bit");
  JPP_LM_CHECK(!same_start(h->data, {gate->data, x->data, given(state) ? state->data : nullptr}) &&
                   !same_start(given(last) ? last->data : nullptr, {gate->data, x->data, h->data, given(state) ? state->data : nullptr}),
               "the output overlaps an input");
  if (int rc = bad_workspace(workspace, workspace_bytes, scan_workspace(rows, n, dim, max_len))) return rc;
  DeviceScope scope(device);
  if (scope.rc() != JPPGPU_OK) return scope.rc();
  if (n == 0 && !cleared(h)) return JPPGPU_OK;
  Launcher go{static_cast<jpp_stream_t>(stream)};
  switch (x->type) {
    case JPPGPU_LM_F32: run_scan<LmF32>(go, s, false); break;
    case JPPGPU_LM_BF16: run_scan<LmBf16>(go, s, false); break;
    default: run_scan<LmF16>(go, s, false); break;
  }
  return go.rc;
}

extern "C" int jppgpu_lm_scan_grad(const jppgpu_lm_matrix* gate, const jppgpu_lm_matrix* x, const int32_t* offsets, int64_t n, int64_t rows,
                                   int64_t dim, int64_t max_len, const jppgpu_lm_matrix* state, const float* saved, const jppgpu_lm_matrix* dh,
                                   const jppgpu_lm_matrix* dlast, const jppgpu_lm_matrix* dgate, const jppgpu_lm_matrix* dx,
                                   const jppgpu_lm_matrix* dstate, void* workspace, uint64_t workspace_bytes, int32_t device, void* stream) {
  ScanArgs s{};
  s.gate = gate;
  s.x = x;
  s.state = state;
  s.dh = dh;
  s.dlast = dlast;
  s.dgate = dgate;
  s.dx = dx;
  s.dstate = dstate;
  s.offsets = offsets;
  s.n = n;
  s.rows = rows;
  s.dim = dim;
  s.maxLen = max_len;
  s.saved = const_cast<float*>(saved);
  s.workspace = workspace;
  if (int rc = check_scan(s)) return rc;
  JPP_LM_REFUSE_IF(bad_matrix(dh, rows, dim, kNeeded));
  JPP_LM_REFUSE_IF(bad_matrix(dgate, rows, dim, kBatchResult));
  JPP_LM_REFUSE_IF(bad_matrix(dx, rows, dim, kBatchResult));
  JPP_LM_REFUSE_IF(bad_matrix(dlast, n, dim, kOptional));
  JPP_LM_REFUSE_IF(bad_matrix(dstate, n, dim, kOptional));
  JPP_LM_REFUSE_IF(bad_f32(saved));
  JPP_LM_CHECK(rows == 0 || saved != nullptr, "the saved states are missing");
  JPP_LM_CHECK(dh->type == x->type && type_of(dgate) == x->type && type_of(dx) == x->type, "the gradients of rows are of the type of x");
  JPP_LM_CHECK((!given(dlast) || dlast->type == JPPGPU_LM_F32) && (!given(dstate) || dstate->type == JPPGPU_LM_F32),
               "the gradients of states are 32-bit");
  const void* st = given(state) ? state->data : nullptr;
  const void* dl = given(dlast) ? dlast->data : nullptr;
  JPP_LM_CHECK(!same_start(dgate->data, {gate->data, x->data, st, dh->data, dl, saved}) &&
                   !same_start(dx->data, {gate->data, x->data, st, dh->data, dl, saved, dgate->data}) &&
                   !same_start(given(dstate) ? dstate->data : nullptr, {gate->data, x->data, st, dh->data, dl, saved, dgate->data, dx->data}),
               "the output overlaps an input");
  if (int rc = bad_workspace(workspace, workspace_bytes, scan_workspace(rows, n, dim, max_len))) return rc;
  DeviceScope scope(device);
  if (scope.rc() != JPPGPU_OK) return scope.rc();
  if (n == 0 && !cleared(dgate) && !cleared(dx)) return JPPGPU_OK;
  Launcher go{static_cast<jpp_stream_t>(stream)};
  switch (x->type) {
    case JPPGPU_LM_F32: run_scan<LmF32>(go, s, true); break;
    case JPPGPU_LM_BF16: run_scan<LmBf16>(go, s, true); break;
    default: run_scan<LmF16>(go, s, true); break;
  }
  return go.rc;
}

extern "C" int jppgpu_lm_nce_score(const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim, const jppgpu_lm_ids* ids,
                                   int64_t n, int64_t cands, float constant, float* scores, int32_t device, void* stream) {
  if (int rc = check_nce(h, table, vocab, dim, ids, n, cands)) return rc;
  JPP_LM_CHECK(n == 0 || scores != nullptr, "the scores are missing");
  JPP_LM_REFUSE_IF(bad_f32(scores));
  JPP_LM_CHECK(!same_start(scores, {h->data, table->data, ids->data}), "the output overlaps an input");
  DeviceScope scope(device);
  if (scope.rc() != JPPGPU_OK) return scope.rc();
  if (n == 0) return JPPGPU_OK;
  LmNce q{};
  q.vocab = (u32)vocab;
  q.dim = (u32)dim;
  q.n = (u64)n;
  q.cands = (u32)cands;
  q.hStride = h->stride;
  q.tableStride = table->stride;
  q.constant = constant;
  q.out = scores;
  Launcher go{static_cast<jpp_stream_t>(stream)};
  dispatch_nce(go, q, h, table, ids_of(ids), nullptr, false);
  return go.rc;
}

extern "C" int jppgpu_lm_nce_loss_workspace(int64_t n, int64_t cands, int64_t vocab, int64_t dim, uint64_t* bytes) {
  JPP_LM_CHECK(bytes != nullptr, "null argument");
  JPP_LM_CHECK(dim >= 1 && dim <= kMaxDim, "dim outside 1 .. 2^24");
  JPP_LM_CHECK(vocab >= 0 && vocab < kMaxIndex, "vocab outside 0 .. 2^31 - 2");
  JPP_LM_CHECK(cands >= 1 && cands <= kMaxIndex && n >= 0 && n <= kMaxIndex / cands, "n * cands outside 0 .. 2^31 - 1");
  *bytes = nce_workspace(n, cands, vocab, dim);
  return JPPGPU_OK;
}

extern "C" int jppgpu_lm_nce_loss(const jppgpu_lm_matrix* h, const jppgpu_lm_matrix* table, int64_t vocab, int64_t dim, const jppgpu_lm_ids* ids,
                                  int64_t n, int64_t cands, const float* log_noise, float constant, const float* weight, float* loss,
                                  const jppgpu_lm_matrix* dh, const jppgpu_lm_matrix* dtable, void* workspace, uint64_t workspace_bytes,
                                  int32_t device, void* stream) {
  if (int rc = check_nce(h, table, vocab, dim, ids, n, cands)) return rc;
  JPP_LM_CHECK(n <= kMaxIndex / cands, "n * cands outside 0 .. 2^31 - 1");
  JPP_LM_REFUSE_IF(bad_matrix(dh, n, dim, kOptional));
  JPP_LM_REFUSE_IF(bad_matrix(dtable, vocab, dim, kOptional));
  JPP_LM_CHECK(vocab == 0 || log_noise != nullptr, "the logarithms of the noise are missing");
  JPP_LM_CHECK(n == 0 || loss != nullptr, "the loss is missing");
  JPP_LM_REFUSE_IF(bad_f32(log_noise));
  JPP_LM_REFUSE_IF(bad_f32(weight));
  JPP_LM_REFUSE_IF(bad_f32(loss));
  JPP_LM_CHECK(!given(dh) || dh->type == h->type, "the gradient of h is of its type");
  JPP_LM_CHECK(!given(dtable) || dtable->type == JPPGPU_LM_F32, "the gradient of a table is 32-bit");
  const void* dhp = given(dh) ? dh->data : nullptr;
  JPP_LM_CHECK(!same_start(loss, {h->data, table->data, ids->data, log_noise, weight}) &&
                   !same_start(dhp, {h->data, table->data, ids->data, log_noise, weight, loss}) &&
                   !same_start(given(dtable) ? dtable->data : nullptr, {h->data, table->data, ids->data, log_noise, weight, loss, dhp}),
               "the output overlaps an input");
  const bool grads = n > 0 && (given(dh) || given(dtable));
  if (grads)
    if (int rc = bad_workspace(workspace, workspace_bytes, nce_workspace(n, cands, vocab, dim))) return rc;
  DeviceScope scope(device);
  if (scope.rc() != JPPGPU_OK) return scope.rc();
  Launcher go{static_cast<jpp_stream_t>(stream)};
  if (n == 0) {
    if (given(dtable) && vocab > 0) clear_matrix(go, dtable, (u64)vocab, (u64)dim);
    return go.rc;
  }
  LmNce q{};
  q.vocab = (u32)vocab;
  q.dim = (u32)dim;
  q.n = (u64)n;
  q.cands = (u32)cands;
  q.hStride = h->stride;
  q.tableStride = table->stride;
  q.dhStride = given(dh) ? dh->stride : 0;
  q.constant = constant;
  q.logNoise = log_noise;
  q.weight = weight;
  q.out = loss;
  const u64 entries = (u64)n * (u64)cands;
  Carver c{static_cast<char*>(workspace)};
  if (grads) {
    // read by the sums by word, and for dh where rows are walked in blocks
    float* g = c.take<float>(entries);
    if (given(dtable) || nce_packs((u32)dim, h->type) > kNcePacks) q.g = g;
  }
  dispatch_nce(go, q, h, table, ids_of(ids), const_cast<void*>(dhp), true);
  if (given(dtable) && vocab > 0) {
    SumPlan p(entries, (u64)vocab, (u64)dim, (u64)cands, true, h->type);
    p.carve(static_cast<char*>(workspace) + c.used);
    sum_by_word(go, p, SumSource{ids, (u32)vocab, (u32)cands, 1.f, q.g, h, static_cast<float*>(dtable->data), dtable->stride});
  }
  return go.rc;
}
