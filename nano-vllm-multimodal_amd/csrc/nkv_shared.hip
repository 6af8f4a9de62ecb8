// Decode attention of a batch whose sequences share prefixes: one query
// token per sequence over its paged context, as nkv_attention.hip computes
// it, but the prefix that a group of consecutive sequences has in common is
// read once for all of the group's query rows.
//
// Group g (sequences [cu_groups[g], cu_groups[g+1])) shares the first P_g
// rows of its contexts.  For the (sequence, query head) rows of one kv head
//   o = (sum_prefix w v + sum_rest w v) / (sum_prefix w + sum_rest w),
//   w = exp(scale q k - m),
// the prefix sums of all rows of the group are one product of the rows with
// the prefix's keys and one with its values; the sums over the rest of each
// context are a sequence's own.  Both are cut into pieces of keys whose
// partials (m, weight sum, 128 output sums, all fp32) a merge adds up.
//
// One launch holds both kinds of items, the prefix's first: they are bound
// by the matrix cores, the others by HBM, so they run side by side on a CU.
//   A prefix item is one workgroup of four wavefronts: up to 128 query rows of
//     a kv head over 64-key tiles that all four read.  RW of them split the
//     rows (32 each), 4 / RW the keys of a tile; up to 32 rows split keys
//     only, and every wavefront reads only the keys it copied itself, with no
//     barrier in its loop.
//   A rest's item is one wavefront (attend_solo), four to a workgroup.
// K and V go from the cache straight into rings of tiles in LDS
// (global_load_lds), copies ahead of the products.
//   S^T = K Q^T    16x16x32 MFMAs: a lane's scores belong to one query row
//   O^T += V^T P^T the weights, rounded to the element type, straight from
//                  the score registers; V^T from the transposing LDS read;
//                  a product with ones sums the same rounded weights, so the
//                  rounding of a weight (at most half a step of the type)
//                  enters numerator and denominator alike.
// Sequences shorter than their group's prefix share nothing and are read
// from row 0 through their own table, so no row is masked inside a tile; nor
// does a group whose first sequence is, as its table would not hold the rows.
// Keys in a block outside the cache or past the table are dropped: they copy
// a row of zeros and their scores become -inf.
//
// 256 sequences of 16 query and 8 kv heads behind 16,384 shared keys, 16 to
// 2,048 of their own (bf16, 533 MB, 35 GFLOP): 114 us; the rests alone 94 us,
// 5.0 TB/s, the prefix alone 60 us.  Reading the prefix once per sequence
// instead is 17.7 GB.  32 sequences of 28 and 4 heads behind 12,001 keys: 27
// us, of which 21 are the attention; 8 sequences, 12 us, two launches' latency.
#include <algorithm>
#include <cmath>

#include "nkv_common.h"
#include "nkv_mfma.h"

namespace nkv {
namespace {

constexpr int kDim = 128;
constexpr int kThreads = 256;
constexpr int kTileKeys = 64;
constexpr int kChunk = 16;        // keys a wavefront copies per tile
constexpr uint32_t kTileBytes = kTileKeys * 256;
constexpr int kMaxGroup = 16;     // query heads per kv head
constexpr int kTileRows = 128;    // query rows of a prefix tile at most
constexpr int kPlanThreads = 1024;
constexpr int kSlots = 512;       // workgroups resident on the chip: two per CU
// The rests' entries: about so many rounds of wavefronts over the chip, so
// that the last round is a small part (the rests of 256 sequences 94.5 us; of
// 8 rounds 98.2, of 2 94.6, and 124.7 instead of 124.0 beside a prefix), but
// none shorter than kMinRestChunks chunks (13 groups of 96 sequences 46.3 us;
// from 2 chunks on 50.3, from 8 on 47.0).
constexpr int kRestRounds = 4;
constexpr int kMinRestChunks = 4;
// Pieces of a prefix, in 64-key tiles.  Those that could all run at once at
// two workgroups per CU are cut for one per CU instead, up to kWidePieceTiles:
// a piece of few tiles costs as much to start, to store its 128 rows of
// partials and to merge them as to walk (28 heads over 12,001 keys 28.8 us,
// cut for two 32.0; up to 12 and 16 tiles the same).  8 sequences behind
// 1,511 keys take 12.6 us from 1 or 2 tiles on, 14.5 from 4.  Longer ones pay
// for the second workgroup: it takes its weights while the first multiplies
// (16,384 keys alone 60 us, cut for one 71).  Beside long rests, more than
// kRestsPerTile chunks per tile, the rests take that second place, and a cut
// for one leaves no CU with two pieces while others have one (256 sequences of
// 32 heads behind 4,096 keys, 16 to 256 of their own: 50 us instead of 56;
// 1,024 of them 160 instead of 175; at 1.5 chunks per tile 45.3 instead of 43.6).
constexpr int kMinPieceTiles = 2;
constexpr int kRestsPerTile = 2;
constexpr int kWidePieceTiles = 8;
constexpr int32_t kMaxLength = 0x7FFFFF00;
constexpr float kRescaleLog2 = 8.f;  // the reference max moves only past this

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(4))) const int32_t const_i32;

// ------------------------------------------------------------------ the plan
//
// int4s:
//   [0]  {prefix entries, rest entries, num_seqs, num_groups}
//   [1]  {num_kv_heads, query heads per kv head, 0, 0}
//   [2, 18)  256 bytes of zeros, the row that dropped keys copy
//   two per sequence  {rest's first row, context length, first rest entry, rest entries}
//                     {first entry of its group's first tile, pieces per tile, member, 0}
//   two per prefix entry  {first sequence, first query row, query rows, piece}
//                         {first key, past the last, 0, 0}
//   one per rest entry  {sequence, first row, past the last, 0}
// Entries past the last of their kind are empty, so that a workgroup finds
// its own at a fixed place, without the counts.
// The query rows of a group and kv head are member-major, (member, head).
constexpr int kPlanSeqs = 18;
struct PlanShape {
  int64_t seqs, prefix, rest;  // sequences and entries to allocate
  int64_t prefix_rows;         // partial rows of the prefix entries, per kv head
  __host__ __device__ int64_t prefix_at() const { return kPlanSeqs + 2 * seqs; }
  __host__ __device__ int64_t rest_at() const { return prefix_at() + 2 * prefix; }
  __host__ __device__ int64_t int4s() const { return rest_at() + rest; }
  __host__ __device__ int64_t rows(int64_t kv_heads, int64_t group) const {
    return kv_heads * (prefix_rows + rest * group);
  }
};
__host__ __device__ constexpr int64_t slots_per_head(int64_t kv_heads) {
  return kSlots / kv_heads > 0 ? kSlots / kv_heads : 1;
}
// All pieces but a tile's last are full and a slot's share or longer: at most
// slots + tiles prefix entries, and at most sharing + rows / kTileRows tiles.
PlanShape plan_shape(int64_t num_seqs, int64_t num_groups, int64_t kv_heads, int64_t group,
                     int64_t rest_tokens) {
  PlanShape p{num_seqs, 0, 0, 0};
  const int64_t sharing = std::min(num_groups, num_seqs / 2);
  if (sharing > 0) {
    p.prefix = slots_per_head(kv_heads) + sharing + num_seqs * group / kTileRows;
    p.prefix_rows = (slots_per_head(kv_heads) + sharing) * kTileRows + num_seqs * group;
  }
  p.rest = 4 * slots_per_head(kv_heads) * kRestRounds;
  if (rest_tokens >= 0) p.rest = std::min(p.rest, rest_tokens / kChunk + 1);
  p.rest += num_seqs;
  return p;
}

__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* s_sum) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) s_sum[threadIdx.x / kWave] = v;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kPlanThreads / kWave; ++w) total += s_sum[w];
  return total;
}

struct GroupOf {
  const int32_t* cu_seqlens_k;
  const int32_t* cu;
  const int32_t* prefix;
  int32_t num_groups, num_seqs;
  // (A key past the bound lies in no table; tile ends stay below 2^31.)
  __device__ __forceinline__ int32_t length_of(int32_t i) const {
    return min(max(0, cu_seqlens_k[i + 1] - cu_seqlens_k[i]), kMaxLength);
  }
  // A group that shares something: at least two sequences of the batch, the
  // first of which, whose table the prefix is read through, has all of it.
  __device__ __forceinline__ bool shares(int32_t g, int32_t* first, int32_t* n, int32_t* rows) const {
    const int32_t s0 = cu[g], s1 = cu[g + 1];
    *first = s0;
    *n = s1 - s0;
    *rows = prefix[g];
    return s0 >= 0 && s1 <= num_seqs && s1 - s0 >= 2 && *rows > 0 && *rows <= length_of(s0);
  }
  // The group of sequence i, -1 for none.
  __device__ __forceinline__ int32_t of(int32_t i) const {
    int32_t lo = 0, hi = num_groups;
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (cu[mid] <= i) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    // Empty groups at the same place: the last one that starts at or before i.
    return num_groups > 0 && cu[lo] <= i && i < cu[lo + 1] ? lo : -1;
  }
};

__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(
    GroupOf groups, int32_t num_kv_heads, int32_t group, PlanShape shape, int4* __restrict__ plan) {
  extern __shared__ int32_t s_mem[];
  __shared__ int64_t s_sum[kPlanThreads / kWave];
  __shared__ int32_t s_tmp[kPlanThreads / kWave + 1];
  const int32_t t = threadIdx.x;
  const int32_t num_seqs = groups.num_seqs;
  const int32_t num_groups = groups.num_groups;
  // Where sequence i's own part begins: its group's prefix, when it has all of it.
  auto rest_of = [&](int32_t i, int32_t* length) {
    *length = groups.length_of(i);
    const int32_t g = groups.of(i);
    int32_t first, n, rows;
    return g >= 0 && groups.shares(g, &first, &n, &rows) && *length >= rows ? rows : 0;
  };

  int64_t prefix_units = 0, rest_units = 0;  // 64-key tiles and 16-key chunks to walk, per kv head
  for (int32_t g = t; g < num_groups; g += kPlanThreads) {
    int32_t first, n, rows;
    if (groups.shares(g, &first, &n, &rows)) {
      const int64_t q_rows = static_cast<int64_t>(n) * group;
      const int64_t tiles = (q_rows + kTileRows - 1) / kTileRows;
      prefix_units += tiles * ((static_cast<int64_t>(rows) + kTileKeys - 1) / kTileKeys);
    }
  }
  for (int32_t i = t; i < num_seqs; i += kPlanThreads) {
    int32_t length;
    const int32_t start = rest_of(i, &length);
    if (length > start) rest_units += (static_cast<int64_t>(length) - (start & -kChunk) + kChunk - 1) / kChunk;
  }
  prefix_units = block_sum(prefix_units, s_sum);
  rest_units = block_sum(rest_units, s_sum);
  // Prefixes: all items together one round of workgroups.  Rests: about
  // kRestRounds rounds of wavefronts, within the plan's room for them.
  const int64_t slots = slots_per_head(num_kv_heads);
  const int64_t share = (prefix_units + rest_units / 4 + slots - 1) / slots;
  const int64_t half = (2 * prefix_units + slots - 1) / slots;  // a workgroup per CU
  const bool wide = rest_units > kRestsPerTile * prefix_units;
  const int64_t prefix_tiles = max(max(static_cast<int64_t>(kMinPieceTiles), share),
                                   wide ? half : min(half, static_cast<int64_t>(kWidePieceTiles)));
  const int64_t room = max(static_cast<int64_t>(1), shape.rest - num_seqs);
  const int64_t rest_chunks =
      max(max(static_cast<int64_t>(kMinRestChunks), rest_units / (4 * slots * kRestRounds) + 1),
          (rest_units + room - 1) / room);
  const int32_t piece_keys = static_cast<int32_t>(min(prefix_tiles, static_cast<int64_t>(1) << 24) * kTileKeys);
  const int32_t entry_keys = static_cast<int32_t>(min(rest_chunks, static_cast<int64_t>(1) << 26) * kChunk);

  // Prefix entries: a group's tiles of query rows, each cut into pieces.
  lds_exclusive_scan<kPlanThreads>(
      num_groups,
      [&](int32_t g) {
        int32_t first, n, rows;
        if (!groups.shares(g, &first, &n, &rows)) return 0;
        const int32_t tiles = (n * group + kTileRows - 1) / kTileRows;
        return tiles * ((rows - 1) / piece_keys + 1);
      },
      s_mem, s_tmp);
  const int32_t prefix_entries = static_cast<int32_t>(min(static_cast<int64_t>(s_mem[num_groups]), shape.prefix));
  for (int32_t e = t; e < prefix_entries; e += kPlanThreads) {
    const int32_t g = owner_of(s_mem, num_groups, e);
    int32_t first, n, rows;
    groups.shares(g, &first, &n, &rows);
    const int32_t pieces = (rows - 1) / piece_keys + 1;
    const int32_t tile = (e - s_mem[g]) / pieces, piece = (e - s_mem[g]) % pieces;
    const int32_t tile_q = min(kTileRows, n * group - tile * kTileRows);
    // Pieces of equal length, in whole tiles.
    const int32_t key_tiles = (rows - 1) / kTileKeys + 1;
    const int32_t k0 = static_cast<int32_t>(static_cast<int64_t>(key_tiles) * piece / pieces) * kTileKeys;
    const int32_t k1 = min(rows, static_cast<int32_t>(static_cast<int64_t>(key_tiles) * (piece + 1) / pieces) * kTileKeys);
    plan[shape.prefix_at() + 2 * e] = make_int4(first, tile * kTileRows, tile_q, piece);
    plan[shape.prefix_at() + 2 * e + 1] = make_int4(k0, k1, 0, 0);
  }
  for (int32_t e = prefix_entries + t; e < shape.prefix; e += kPlanThreads) {
    plan[shape.prefix_at() + 2 * e] = make_int4(0, 0, 0, 0);
    plan[shape.prefix_at() + 2 * e + 1] = make_int4(0, 0, 0, 0);
  }
  for (int32_t i = t; i < num_seqs; i += kPlanThreads) {
    const int32_t g = groups.of(i);
    int32_t first, n, rows, length;
    int4 record = make_int4(0, 0, 0, 0);
    if (rest_of(i, &length) > 0) {
      groups.shares(g, &first, &n, &rows);
      record = make_int4(s_mem[g], (rows - 1) / piece_keys + 1, i - first, 0);
    }
    plan[kPlanSeqs + 2 * i + 1] = record;
  }
  __syncthreads();
  // The rests.
  lds_exclusive_scan<kPlanThreads>(
      num_seqs,
      [&](int32_t i) {
        int32_t length;
        const int32_t start = rest_of(i, &length);
        return length > start ? (length - (start & -kChunk) - 1) / entry_keys + 1 : 0;
      },
      s_mem, s_tmp);
  const int32_t rest_entries = static_cast<int32_t>(min(static_cast<int64_t>(s_mem[num_seqs]), shape.rest));
  for (int32_t i = t; i < num_seqs; i += kPlanThreads) {
    int32_t length;
    const int32_t start = rest_of(i, &length);
    plan[kPlanSeqs + 2 * i] = make_int4(start, length, s_mem[i], s_mem[i + 1] - s_mem[i]);
  }
  for (int32_t e = t; e < rest_entries; e += kPlanThreads) {
    const int32_t i = owner_of(s_mem, num_seqs, e);
    int32_t length;
    const int32_t start = rest_of(i, &length);
    const int32_t row0 = (start & -kChunk) + (e - s_mem[i]) * entry_keys;  // cuts at whole chunks
    plan[shape.rest_at() + e] =
        make_int4(i, max(start, row0), length - row0 > entry_keys ? row0 + entry_keys : length, 0);
  }
  for (int32_t e = rest_entries + t; e < shape.rest; e += kPlanThreads) {
    plan[shape.rest_at() + e] = make_int4(0, 0, 0, 0);
  }
  if (t < 16) plan[2 + t] = make_int4(0, 0, 0, 0);
  if (t == 0) {
    plan[0] = make_int4(prefix_entries, rest_entries, num_seqs, num_groups);
    plan[1] = make_int4(num_kv_heads, group, 0, 0);
  }
}

// ------------------------------------------------------------- the attention

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lgkmcnt0() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// A wave-uniform address, in scalar registers.
__device__ __forceinline__ const uint8_t* scalar_pointer(const uint8_t* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
  const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(high) << 32 | low);
}

// A ring of three K tiles and two V tiles: 80 KiB, two workgroups per CU.
// The key waves' partial sums take its place at the end, 16 KiB each, their
// maxima and weight sums behind them.
struct TileShared {
  u32x4 k[3][kTileKeys * 16];
  u32x4 v[2][kTileKeys * 16];
};
static_assert(sizeof(TileShared) == 80 * 1024, "two workgroups per CU");

// The cache as one item sees it: a kv head of the rows of one block table.
struct KeySource {
  const uint8_t* k_head;
  const uint8_t* v_head;
  const const_i32* table;
  const uint8_t* zeros;
  int64_t table_stride;
  uint32_t row_bytes;
  int32_t block_size, block_shift, num_blocks;
  int32_t begin, end;  // context rows; tiles start at begin rounded down to a chunk
};

// The item's query rows [row0, row0 + rows): row r is head r % group of the
// sequence first + r / group.
struct RowSource {
  const uint16_t* q;  // of the kv head's first query head
  int64_t seq_stride;
  int32_t first, row0, rows, group;
};

// Blocks [first, first + 64) of an item's table, one id per lane, -1 outside
// the cache or the table: keys find their rows by lane reads, with no memory
// access in the loop but where an item outgrows the window (blocks of 16
// keys: every 1,024 keys).
template <bool kChunked>
struct BlockWindow {
  const KeySource& src;
  int32_t last, first, ids;
  bool ok;  // every block of the item in the window is there
  __device__ __forceinline__ explicit BlockWindow(const KeySource& s) : src(s), first(0), ids(-1), ok(false) {
    last = block_at(src.end - 1);
  }
  __device__ __forceinline__ int32_t block_at(int32_t t) const {
    return kChunked ? t >> src.block_shift : t / src.block_size;
  }
  __device__ __forceinline__ void load(int32_t block) {
    first = block;
    const int32_t logical = block + static_cast<int32_t>(threadIdx.x & (kWave - 1));
    ids = -1;
    if (logical <= last && logical < src.table_stride) {
      ids = src.table[logical];
      if (ids >= src.num_blocks) ids = -1;
    }
    ok = !__any(logical <= last && ids < 0);
  }
  // Makes the window hold the blocks of keys [t, t + keys).
  __device__ __forceinline__ void cover(int32_t t, int32_t keys) {
    if (min(block_at(t + keys - 1), last) - first >= kWave) load(block_at(t));
  }
  // The cache row of the lane's key, -1 if it is not there.
  __device__ __forceinline__ int32_t row_of(int32_t key) const {
    const int32_t block = block_at(key);
    const int32_t id = __shfl(ids, (block - first) & (kWave - 1), kWave);
    return key >= src.begin && key < src.end && id >= 0 ? id * src.block_size + (key - block * src.block_size) : -1;
  }
};

// Four copies of a 16-key chunk of K or V into LDS: lane l copies 16 bytes of
// key 4 i + l / 16 to position l % 16 of its row.  Keys that are not there
// (their bit in `there` is 0) copy zeros.  row: the cache row of the chunk's
// first key, or, without whole chunks, of the lane's four keys.
// kStream: no other item reads these rows, the copies pass the caches by.
template <bool kChunked, bool kStream>
struct ChunkCopy {
  const KeySource& src;
  int c16, g4;
  uint32_t off_k[4], off_v[4];
  __device__ __forceinline__ ChunkCopy(const KeySource& s, int lane) : src(s), c16(lane & 15), g4(lane >> 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 4 * i + g4;
      off_k[i] = key * src.row_bytes + 16u * static_cast<uint32_t>(c16 ^ key);
      off_v[i] = key * src.row_bytes + 16u * static_cast<uint32_t>(c16 ^ ((key & 7) << 1));
    }
  }
  __device__ __forceinline__ void run(const uint8_t* head, const uint32_t* off, uint32_t dst, uint32_t there,
                                      const int32_t* row) const {
    if (kChunked && there == 0xFFFFu) {
      const uint8_t* const base =
          scalar_pointer(head + static_cast<uint64_t>(static_cast<uint32_t>(row[0])) * src.row_bytes);
#pragma unroll
      for (int i = 0; i < 4; ++i) lds_copy16<kStream>(base, off[i], dst + i * 1024u);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 4 * i + g4;
        const uint32_t place = off[i] - key * src.row_bytes;  // inside the key's row
        const int32_t at = kChunked ? row[0] + key : row[kChunked ? 0 : i];
        const uint8_t* const from =
            (there >> key) & 1u ? head + static_cast<uint64_t>(static_cast<uint32_t>(at)) * src.row_bytes : src.zeros;
        lds_copy16<kStream>(from + place, dst + i * 1024u);
      }
    }
  }
  __device__ __forceinline__ void k(uint32_t dst, uint32_t there, const int32_t* row) const {
    run(src.k_head, off_k, dst, there, row);
  }
  __device__ __forceinline__ void v(uint32_t dst, uint32_t there, const int32_t* row) const {
    run(src.v_head, off_v, dst, there, row);
  }
};

// kChunked: blocks are a power of two of keys, whole chunks (one block id per
// chunk); otherwise every key looks up its own.
template <int RW, int NMB, bool kChunked, bool kHalf>
__device__ __forceinline__ void attend(TileShared& sh, const KeySource& src, const RowSource& rows,
                                       float scale_log2, float* __restrict__ part_acc,
                                       f32x2* __restrict__ part_ml) {
  typedef Elem<kHalf> E;
  typedef typename E::T T;
  typedef typename E::X8 X8;
  typedef typename E::X4 X4;
  constexpr int KW = 4 / RW;
  constexpr int NKB = RW;  // 16-key blocks a wavefront computes per tile
  static_assert(RW == 1 || NMB == 2, "row waves hold 32 rows");
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int c16 = lane & 15;
  const int g4 = lane >> 4;
  const int rw = wave % RW;   // which 32 rows
  const int kw = wave / RW;   // which keys of a tile
  const int chunk = kw * NKB + rw;  // the 16 keys this wavefront copies

  // Q^T operands: row 16 mb + c16 of the wavefront's, dims 32 dc + 8 g4 .. +8.
  X8 qb[NMB][4];
#pragma unroll
  for (int mb = 0; mb < NMB; ++mb) {
    const int32_t r = rows.row0 + rw * 32 + mb * 16 + c16;
    const bool ok = rw * 32 + mb * 16 + c16 < rows.rows;
    const int32_t member = ok ? r / rows.group : 0;
    const int32_t head = ok ? r - member * rows.group : 0;
    const uint16_t* row = rows.q + static_cast<int64_t>(rows.first + member) * rows.seq_stride + head * kDim;
#pragma unroll
    for (int dc = 0; dc < 4; ++dc) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (ok) v = *reinterpret_cast<const u32x4*>(row + 32 * dc + 8 * g4);
      qb[mb][dc] = __builtin_bit_cast(X8, v);
    }
  }

  BlockWindow<kChunked> window(src);
  // What is known of a tile from the copies of its K to its products: its
  // keys that are there (bit = key) and where this wavefront's chunk lies (a
  // cache row for its first key; without whole chunks a row for each of the
  // lane's four keys).
  struct Tile {
    uint64_t there;
    int32_t row[kChunked ? 1 : 4];
  };
  auto find = [&](int32_t tile_t) -> Tile {
    Tile tile;
    window.cover(tile_t, kTileKeys);
    if constexpr (kChunked) {
      const int32_t t = tile_t + chunk * kChunk;
      const int32_t block = window.block_at(t);
      const int32_t id = __builtin_amdgcn_readlane(window.ids, (block - window.first) & (kWave - 1));
      tile.row[0] = (id << src.block_shift) + (t & (src.block_size - 1));
      tile.there = ~uint64_t{0};
      if (tile_t < src.begin || tile_t + kTileKeys > src.end || !window.ok) {
        tile.there = __ballot(window.row_of(tile_t + lane) >= 0);
      }
    } else {
      const int32_t row = window.row_of(tile_t + lane);
      tile.there = __ballot(row >= 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) tile.row[i] = __shfl(row, chunk * kChunk + 4 * i + g4, kWave);
    }
    return tile;
  };
  // (Up to 64 rows are a whole group, whose keys nothing else reads, or the
  // last of its tiles, behind those that keep them in the caches.)
  const ChunkCopy<kChunked, RW != 4> copy(src, lane);
  const uint32_t lds_k = lds_address(&sh.k[0][0]) + chunk * 4096u;
  const uint32_t lds_v = lds_address(&sh.v[0][0]) + chunk * 4096u;

  float row_max[NMB];
  f32x4 acc[9][NMB];  // dims 16 db + 4 g4 + i of row c16; block 8: the weight sum (g4 == 0, i == 0)
#pragma unroll
  for (int mb = 0; mb < NMB; ++mb) {
    row_max[mb] = -INFINITY;
#pragma unroll
    for (int db = 0; db < 9; ++db) acc[db][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const T one = c16 == 0 ? static_cast<T>(1.f) : static_cast<T>(0.f);
  const int tr_key = 4 * g4 + ((lane >> 2) & 3);
  const int tr_dim = 4 * (lane & 3);

  const int32_t first_key = src.begin & ~(kChunk - 1);
  const int32_t num_tiles = (src.end - first_key + kTileKeys - 1) / kTileKeys;
  auto tile_key = [&](int32_t tile) { return first_key + tile * kTileKeys; };
  window.load(window.block_at(first_key));
  __builtin_amdgcn_s_waitcnt(0);  // q and ids have landed: only the copies are in flight below
  // S^T of the tile in K slot `slot`: block (kb, mb) holds keys 16 kb + 4 g4 + i
  // (of the wavefront's keys) of row 16 mb + c16.
  auto scores = [&](int slot, f32x4 (&st)[NKB][NMB]) {
    const u32x4* const k_tile = sh.k[slot];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb) st[kb][mb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dc = 0; dc < 4; ++dc) {
        const X8 a = __builtin_bit_cast(X8, k_tile[k_index(16 * (kw * NKB + kb) + c16, 4 * dc + g4)]);
#pragma unroll
        for (int mb = 0; mb < NMB; ++mb) st[kb][mb] = E::mfma(a, qb[mb][dc], st[kb][mb]);
      }
    }
  };
  // Scores to weights: -inf for the keys that are not there, the row's
  // reference max, which moves only past kRescaleLog2, and exp2.
  auto weights = [&](uint64_t tile_there, f32x4 (&st)[NKB][NMB]) {
    if (tile_there != ~uint64_t{0}) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const uint32_t there = static_cast<uint32_t>(tile_there >> ((kw * NKB + kb) * kChunk)) >> (4 * g4);
#pragma unroll
        for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[kb][mb][i] = (there >> i) & 1u ? st[kb][mb][i] : -INFINITY;
      }
    }
    float ref[NMB];
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
      float local = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) local = fmaxf(local, st[kb][mb][i]);
      local = row4_max(local) * scale_log2;  // scale > 0: the max commutes with it
      const bool move = local > row_max[mb] + kRescaleLog2;
      if (__any(move)) {
        const float m_new = move ? local : row_max[mb];
        const float alpha = move ? __builtin_amdgcn_exp2f(row_max[mb] - m_new) : 1.f;
#pragma unroll
        for (int db = 0; db < 9; ++db) acc[db][mb] *= alpha;
        row_max[mb] = m_new;
      }
      ref[mb] = row_max[mb] == -INFINITY ? INFINITY : row_max[mb];  // nothing yet: weights 0
    }
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          st[kb][mb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kb][mb][i], scale_log2, -ref[mb]));
        }
  };

  // Tile t's K is copied ahead of its V; within a step V goes first, so that a
  // step waits for what it reads while the K behind it is still in flight.
  Tile now{}, ahead1{}, ahead2{}, ahead3{};  // tiles t, t + 1, ...
  auto copy_k = [&](int slot, const Tile& tile) {
    copy.k(lds_k + slot * kTileBytes, static_cast<uint32_t>(tile.there >> (chunk * kChunk)) & 0xFFFFu, tile.row);
  };
  auto copy_v = [&](int32_t t, const Tile& tile) {
    copy.v(lds_v + (t & 1) * kTileBytes, static_cast<uint32_t>(tile.there >> (chunk * kChunk)) & 0xFFFFu, tile.row);
  };
  now = find(first_key);
  copy_k(0, now);
  copy_v(0, now);
  if (num_tiles > 1) {
    ahead1 = find(tile_key(1));
    copy_k(1, ahead1);
  }
  f32x4 st[NKB][NMB];
  if constexpr (RW == 1) {
    // Every wavefront reads what it copied itself: counted waits, no barrier.
    const X4 ones = {one, one, one, one};
    int slot = 0;  // tile % 3
    for (int32_t tile = 0; tile < num_tiles; ++tile) {
      const int32_t left = num_tiles - 1 - tile;  // tiles behind this one
      if (left > 0) {
        wait_vmcnt<8>();  // K(tile): V(tile) and K(tile + 1) may be in flight
      } else {
        wait_vmcnt<4>();
      }
      wait_lgkmcnt0();  // the slots filled next have been read
      if (left > 0) copy_v(tile + 1, ahead1);
      if (left > 1) {
        ahead2 = find(tile_key(tile + 2));
        copy_k(slot == 0 ? 2 : slot - 1, ahead2);  // (tile + 2) % 3
      }
      scores(slot, st);
      weights(now.there, st);
      if (left > 1) {  // V(tile): what was issued behind it may be in flight
        wait_vmcnt<12>();
      } else if (left == 1) {
        wait_vmcnt<8>();
      } else {
        wait_vmcnt<0>();
      }
      X4 pb[NMB];
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) pb[mb][i] = static_cast<T>(st[0][mb][i]);
      const u32x4* const v_tile = sh.v[tile & 1];
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        const X4 a = __builtin_bit_cast(X4, v_tr_read(v_tile, 16 * kw + tr_key, 16 * db + tr_dim));
#pragma unroll
        for (int mb = 0; mb < NMB; ++mb) acc[db][mb] = E::mfma16(a, pb[mb], acc[db][mb]);
      }
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb) acc[8][mb] = E::mfma16(ones, pb[mb], acc[8][mb]);
      now = ahead1;
      ahead1 = ahead2;
      slot = slot == 2 ? 0 : slot + 1;
    }
  } else {
    // A step takes tile t's weights, then, in one run of matrix instructions,
    // the scores of tile t + 1 and tile t's product with V: while one
    // wavefront of a SIMD is in that run, the other takes its weights.
    const X8 ones = {one, one, one, one, one, one, one, one};
    if (num_tiles > 2) {
      ahead2 = find(tile_key(2));
      copy_k(2, ahead2);
      wait_vmcnt<12>();  // K(0)
    } else {
      wait_vmcnt<0>();
    }
    __syncthreads();
    scores(0, st);
    int slot = 0;  // tile % 3
    for (int32_t tile = 0; tile < num_tiles; ++tile) {
      const int32_t left = num_tiles - 1 - tile;
      const int next = slot == 2 ? 0 : slot + 1;
      if (left > 1) {
        wait_vmcnt<4>();  // V(tile) and K(tile + 1): K(tile + 2) may be in flight
      } else {
        wait_vmcnt<0>();
      }
      wait_lgkmcnt0();
      __syncthreads();  // everyone's copies have landed, the slots filled next have been read
      if (left > 0) copy_v(tile + 1, ahead1);
      if (left > 2) {
        ahead3 = find(tile_key(tile + 3));
        copy_k(slot, ahead3);
      }
      weights(now.there, st);
      X8 pb[NKB / 2][NMB];
#pragma unroll
      for (int mb = 0; mb < NMB; ++mb)
#pragma unroll
        for (int c = 0; c < NKB / 2; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            pb[c][mb][i] = static_cast<T>(st[2 * c][mb][i]);
            pb[c][mb][4 + i] = static_cast<T>(st[2 * c + 1][mb][i]);
          }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      __builtin_amdgcn_sched_barrier(0);
      scores(next, st);  // (behind the last tile: of an older one, dropped)
      // Four K operand reads ahead, then each read's products with the next read.
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < 4 * NKB; ++i) {
        if (i < 4 * NKB - 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, NMB, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      const u32x4* const v_tile = sh.v[tile & 1];
#pragma unroll
      for (int db = 0; db < 8; ++db) {
#pragma unroll
        for (int c = 0; c < NKB / 2; ++c) {
          const int key = 16 * kw * NKB + 32 * c + tr_key;
          const u32x2 lo = v_tr_read(v_tile, key, 16 * db + tr_dim);
          const u32x2 hi = v_tr_read(v_tile, key + 16, 16 * db + tr_dim);
          const X8 a = __builtin_bit_cast(X8, u32x4{lo.x, lo.y, hi.x, hi.y});
#pragma unroll
          for (int mb = 0; mb < NMB; ++mb) acc[db][mb] = E::mfma(a, pb[c][mb], acc[db][mb]);
        }
      }
#pragma unroll
      for (int c = 0; c < NKB / 2; ++c)
#pragma unroll
        for (int mb = 0; mb < NMB; ++mb) acc[8][mb] = E::mfma(ones, pb[c][mb], acc[8][mb]);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      now = ahead1;
      ahead1 = ahead2;
      ahead2 = ahead3;
      slot = next;
    }
  }

  if constexpr (KW == 1) {
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
      const int r = rw * 32 + mb * 16 + c16;
      if (r >= rows.rows) continue;
      float* dst = part_acc + static_cast<int64_t>(r) * kDim + 4 * g4;
#pragma unroll
      for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db) = acc[db][mb];
      if (g4 == 0) part_ml[r] = f32x2{row_max[mb], acc[8][mb][0]};
    }
  } else {
    // The key waves add up through LDS: wavefront (rw, kw) leaves its rows in
    // the buffers (16 KiB per wavefront, 16-byte pieces swizzled by row).
    __syncthreads();  // every wavefront has read its last tile
    u32x4* const buffers = reinterpret_cast<u32x4*>(&sh);  // k and v: 64 KiB in a row
    u32x4* const buffer = buffers + wave * 1024;
    f32x2* const s_ml = reinterpret_cast<f32x2*>(buffers + 4 * 1024);  // [wavefront][row]
#pragma unroll
    for (int mb = 0; mb < NMB; ++mb) {
      const int r = mb * 16 + c16;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        buffer[r * 32 + ((4 * db + g4) ^ c16)] = __builtin_bit_cast(u32x4, acc[db][mb]);
      }
      if (g4 == 0) s_ml[wave * 32 + r] = f32x2{row_max[mb], acc[8][mb][0]};
    }
    __syncthreads();
#pragma unroll 4
    for (int step = 0; step < RW * NMB * 16 * 32 / kThreads; ++step) {
      const int row = (step * kThreads + tid) >> 5, piece = tid & 31;
      if (row >= rows.rows) continue;
      const int from = row / 32, r = row & 31;  // row wave and its row
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < KW; ++k) top = fmaxf(top, s_ml[(k * RW + from) * 32 + r].x);
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const int w = k * RW + from;
        const float mw = s_ml[w * 32 + r].x, lw = s_ml[w * 32 + r].y;
        // A wavefront without keys has (-inf, 0); -inf with another sum is
        // NaN scores, which go on.
        const float f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mw - top);
        const f32x4 v = __builtin_bit_cast(f32x4, buffers[w * 1024 + r * 32 + (piece ^ (r & 15))]);
        if (f != 0.f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(v[i], f, sum[i]);
          l = __builtin_fmaf(lw, f, l);
        }
      }
      *reinterpret_cast<f32x4*>(part_acc + static_cast<int64_t>(row) * kDim + 4 * piece) = sum;
      if (piece == 0) part_ml[row] = f32x2{top, l};
    }
  }
}

// A sequence's rest, by one wavefront on its own: the group's query heads (at
// most 16 rows) over [begin, end) in 16-key chunks, K two chunks ahead and V
// one in a ring of its own (20 KiB).  A rest is short next to what starting an
// item costs (its entry, block ids, q and first chunk, one after another,
// 2.5 us, and its partial 1.2): four wavefronts that each walk an item overlap
// these where one workgroup per item waited for them (2,640 items of 5.7
// 64-key tiles took 10 us each, 4.3 of them so).
constexpr int kSoloBytes = 20 * 1024;
template <bool kChunked, bool kHalf>
__device__ __forceinline__ void attend_solo(TileShared& sh, const KeySource& src, const uint16_t* q,
                                            int32_t group, float scale_log2, float* __restrict__ part_acc,
                                            f32x2* __restrict__ part_ml) {
  typedef Elem<kHalf> E;
  typedef typename E::T T;
  typedef typename E::X8 X8;
  typedef typename E::X4 X4;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c16 = lane & 15;
  const int g4 = lane >> 4;
  X8 qb[4];
  {
    const uint16_t* row = q + (c16 < group ? c16 : 0) * kDim;
#pragma unroll
    for (int dc = 0; dc < 4; ++dc) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (c16 < group) v = *reinterpret_cast<const u32x4*>(row + 32 * dc + 8 * g4);
      qb[dc] = __builtin_bit_cast(X8, v);
    }
  }
  BlockWindow<kChunked> window(src);
  const int32_t first_key = src.begin & ~(kChunk - 1);
  const int32_t chunks = (src.end - first_key + kChunk - 1) / kChunk;
  window.load(window.block_at(first_key));
  struct Chunk {
    uint32_t there;
    int32_t row[kChunked ? 1 : 4];
  };
  auto find = [&](int32_t t) -> Chunk {
    Chunk c;
    window.cover(t, kChunk);
    if constexpr (kChunked) {
      const int32_t block = window.block_at(t);
      const int32_t id = __builtin_amdgcn_readlane(window.ids, (block - window.first) & (kWave - 1));
      const int32_t low = max(0, src.begin - t), high = min(kChunk, src.end - t);
      c.there = id >= 0 ? ((1u << high) - 1u) & ~((1u << low) - 1u) : 0u;
      c.row[0] = (id << src.block_shift) + (t & (src.block_size - 1));
    } else {
      const int32_t key = t + c16;
      const int32_t row = window.row_of(key);
      c.there = static_cast<uint32_t>(__ballot(row >= 0)) & 0xFFFFu;  // lanes 0-15
#pragma unroll
      for (int i = 0; i < 4; ++i) c.row[i] = __shfl(row, 4 * i + g4, kWave);
    }
    return c;
  };
  const ChunkCopy<kChunked, true> copy(src, lane);
  const uint32_t lds_k = lds_address(reinterpret_cast<const u32x4*>(&sh)) + wave * kSoloBytes;
  const uint32_t lds_v = lds_k + 3 * 4096u;
  const u32x4* const ring = reinterpret_cast<const u32x4*>(&sh) + wave * (kSoloBytes / 16);

  float row_max = -INFINITY;
  f32x4 acc[9];
#pragma unroll
  for (int db = 0; db < 9; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T one = c16 == 0 ? static_cast<T>(1.f) : static_cast<T>(0.f);
  const X4 ones = {one, one, one, one};
  const int tr_key = 4 * g4 + ((lane >> 2) & 3);
  const int tr_dim = 4 * (lane & 3);

  __builtin_amdgcn_s_waitcnt(0);  // q and ids have landed: only the copies are in flight below
  Chunk now = find(first_key), ahead1{}, ahead2{};
  copy.k(lds_k, now.there, now.row);
  copy.v(lds_v, now.there, now.row);
  if (chunks > 1) {
    ahead1 = find(first_key + kChunk);
    copy.k(lds_k + 4096u, ahead1.there, ahead1.row);
  }
  int slot = 0;  // chunk % 3
  for (int32_t c = 0; c < chunks; ++c) {
    const int32_t left = chunks - 1 - c;
    if (left > 0) {
      wait_vmcnt<8>();  // K(c): V(c) and K(c + 1) may be in flight
    } else {
      wait_vmcnt<4>();
    }
    wait_lgkmcnt0();  // the slots filled next have been read
    if (left > 0) copy.v(lds_v + ((c + 1) & 1) * 4096u, ahead1.there, ahead1.row);
    if (left > 1) {
      ahead2 = find(first_key + (c + 2) * kChunk);
      copy.k(lds_k + (slot == 0 ? 2 : slot - 1) * 4096u, ahead2.there, ahead2.row);  // (c + 2) % 3
    }
    const u32x4* const k_tile = ring + slot * 256;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dc = 0; dc < 4; ++dc) {
      s = E::mfma(__builtin_bit_cast(X8, k_tile[k_index(c16, 4 * dc + g4)]), qb[dc], s);
    }
    if (now.there != 0xFFFFu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = (now.there >> (4 * g4 + i)) & 1u ? s[i] : -INFINITY;
    }
    float local = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    local = row4_max(local) * scale_log2;  // scale > 0: the max commutes with it
    const bool move = local > row_max + kRescaleLog2;
    if (__any(move)) {
      const float m_new = move ? local : row_max;
      const float alpha = move ? __builtin_amdgcn_exp2f(row_max - m_new) : 1.f;
#pragma unroll
      for (int db = 0; db < 9; ++db) acc[db] *= alpha;
      row_max = m_new;
    }
    const float ref = row_max == -INFINITY ? INFINITY : row_max;  // nothing yet: weights 0
    X4 pb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pb[i] = static_cast<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale_log2, -ref)));
    }
    if (left > 1) {  // V(c): what was issued behind it may be in flight
      wait_vmcnt<12>();
    } else if (left == 1) {
      wait_vmcnt<8>();
    } else {
      wait_vmcnt<0>();
    }
    const u32x4* const v_tile = ring + (3 + (c & 1)) * 256;
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      acc[db] = E::mfma16(__builtin_bit_cast(X4, v_tr_read(v_tile, tr_key, 16 * db + tr_dim)), pb, acc[db]);
    }
    acc[8] = E::mfma16(ones, pb, acc[8]);
    now = ahead1;
    ahead1 = ahead2;
    slot = slot == 2 ? 0 : slot + 1;
  }
  if (c16 < group) {
    float* dst = part_acc + c16 * kDim + 4 * g4;
#pragma unroll
    for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db) = acc[db];
    if (g4 == 0) part_ml[c16] = f32x2{row_max, acc[8][0]};
  }
}

struct SharedArgs {
  const uint16_t* q;
  const uint8_t* key_cache;
  const uint8_t* value_cache;
  const int32_t* tables;
  const int4* plan;
  float* part_acc;
  f32x2* part_ml;
  int64_t q_seq_stride, table_stride;
  PlanShape shape;
  int32_t block_size, block_shift, num_blocks, num_kv_heads, group, num_seqs, num_groups;
  float scale_log2;
};

// Whether the plan was built for this batch.
__device__ __forceinline__ bool plan_fits(const const_i32* plan, int32_t num_seqs, int32_t num_groups,
                                          int32_t num_kv_heads, int32_t group) {
  return ((plan[2] ^ num_seqs) | (plan[3] ^ num_groups) | (plan[4] ^ num_kv_heads) | (plan[5] ^ group)) == 0;
}

template <bool kChunked, bool kHalf>
__global__ __launch_bounds__(kThreads, 2) void shared_attention_kernel(SharedArgs a) {
  __shared__ TileShared sh;
  const const_i32* const plan = (const const_i32*)a.plan;
  // Another batch's plan leaves at the first use of an entry, below: the entry
  // is on its way by then.
  const bool fits = plan_fits(plan, a.num_seqs, a.num_groups, a.num_kv_heads, a.group);
  // Workgroups of the prefix's entries, one per kv head each; then one per
  // four (rest entry, kv head) items.  The kv head rotates with the entry, so
  // that no XCD (workgroup id % 8) stays on one byte offset of the rows; with
  // the piece of a prefix, so that the tiles that read the same keys, a whole
  // number of 8 workgroups apart from 8 kv heads on, share an L2 (256 sequences
  // of 16 heads behind 16,384 keys 121.2 us; turned with the entry 124.2).
  const int64_t prefix_groups = a.shape.prefix * a.num_kv_heads;
  const bool is_prefix = blockIdx.x < prefix_groups;
  int64_t item = blockIdx.x;
  if (!is_prefix) {
    item = 4 * (item - prefix_groups) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  }
  const int32_t entry = static_cast<int32_t>(item / a.num_kv_heads);
  const int32_t turn = static_cast<int32_t>(item - static_cast<int64_t>(entry) * a.num_kv_heads);
  const const_i32* const prefix_record = plan + 4 * (a.shape.prefix_at() + 2 * static_cast<int64_t>(entry));
  const int32_t turned = is_prefix ? max(0, prefix_record[3]) : 4 * (entry & 0xFFFF);
  const int32_t kh = static_cast<int32_t>((static_cast<uint32_t>(turn) + turned) % a.num_kv_heads);
  KeySource src;
  src.k_head = a.key_cache + static_cast<int64_t>(kh) * (kDim * 2);
  src.v_head = a.value_cache + static_cast<int64_t>(kh) * (kDim * 2);
  src.zeros = reinterpret_cast<const uint8_t*>(a.plan + 2);
  src.table_stride = a.table_stride;
  src.row_bytes = static_cast<uint32_t>(a.num_kv_heads) * (kDim * 2);
  src.block_size = a.block_size;
  src.block_shift = a.block_shift;
  src.num_blocks = a.num_blocks;
  RowSource rows;
  rows.q = a.q + static_cast<int64_t>(kh) * a.group * kDim;
  rows.seq_stride = a.q_seq_stride;
  rows.group = a.group;
  if (is_prefix) {
    const const_i32* const e = prefix_record;
    rows.first = e[0];
    rows.row0 = e[1];
    rows.rows = e[2];
    src.begin = e[4];
    src.end = e[5];
    // Uniform exits for entries that name rows outside the batch.
    const int64_t row = static_cast<int64_t>(entry) * kTileRows;
    if (!fits || rows.first < 0 || rows.row0 < 0 || rows.rows <= 0 || rows.rows > kTileRows || src.begin < 0 ||
        src.end <= src.begin || row + rows.rows > a.shape.prefix_rows ||
        rows.first + (static_cast<int64_t>(rows.row0) + rows.rows - 1) / a.group >= a.num_seqs) {
      return;
    }
    src.table = (const const_i32*)(a.tables + static_cast<int64_t>(rows.first) * a.table_stride);
    float* const acc = a.part_acc + (kh * a.shape.prefix_rows + row) * kDim;
    f32x2* const ml = a.part_ml + kh * a.shape.prefix_rows + row;
    if (rows.rows > 64) {
      attend<4, 2, kChunked, kHalf>(sh, src, rows, a.scale_log2, acc, ml);
    } else if (rows.rows > 32) {
      attend<2, 2, kChunked, kHalf>(sh, src, rows, a.scale_log2, acc, ml);
    } else if (rows.rows > 16) {
      attend<1, 2, kChunked, kHalf>(sh, src, rows, a.scale_log2, acc, ml);
    } else {
      attend<1, 1, kChunked, kHalf>(sh, src, rows, a.scale_log2, acc, ml);
    }
    return;
  }
  if (entry >= a.shape.rest) return;
  const const_i32* const e = plan + 4 * (a.shape.rest_at() + entry);
  const int32_t seq = e[0];
  src.begin = e[1];
  src.end = e[2];
  if (!fits || seq < 0 || seq >= a.num_seqs || src.begin < 0 || src.end <= src.begin) return;
  src.table = (const const_i32*)(a.tables + static_cast<int64_t>(seq) * a.table_stride);
  const int64_t row = a.num_kv_heads * a.shape.prefix_rows +
                      (static_cast<int64_t>(entry) * a.num_kv_heads + kh) * a.group;
  attend_solo<kChunked, kHalf>(sh, src, rows.q + seq * a.q_seq_stride, a.group, a.scale_log2,
                               a.part_acc + row * kDim, a.part_ml + row);
}

// Adds up the partials of (sequence, query head) pairs: those of the prefix's
// pieces, then the rest's.  kWaves wavefronts per pair, each every kWaves-th
// batch; a lane holds two dims.  Few pairs leave the chip to the latency of a
// wavefront's chain of batches: four share a pair then (call of 896 pairs 28.1
// instead of 31.1 us, of 4,096 127.5 instead of 128.0; of 8,192 60.4 instead of
// 56.0, of 32,768 190 instead of 181: there one wavefront each).
constexpr int kMergePairs = 4096;  // up to so many pairs, four wavefronts each
template <bool kHalf, int kWaves>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a, uint16_t* __restrict__ out,
                                                           int64_t out_seq_stride) {
  constexpr int kPairs = 4 / kWaves;
  constexpr int kMergeBatch = kWaves == 1 ? 8 : 4;
  const int lane = threadIdx.x & (kWave - 1);
  const int w4 = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int part_wave = w4 % kWaves;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * kPairs + w4 / kWaves;
  const int32_t num_q_heads = a.num_kv_heads * a.group;
  const bool there = pair < static_cast<int64_t>(a.num_seqs) * num_q_heads;
  if (kWaves == 1 && !there) return;  // (with more waves a workgroup is one pair)
  const int32_t seq = static_cast<int32_t>(pair / num_q_heads);
  const int32_t qh = static_cast<int32_t>(pair % num_q_heads);
  const int32_t kh = qh / a.group, head = qh % a.group;
  uint32_t* const dst = reinterpret_cast<uint32_t*>(out + seq * out_seq_stride + qh * kDim + 2 * lane);
  const const_i32* const plan = (const const_i32*)a.plan;
  const const_i32* const record = plan + 4 * (kPlanSeqs + 2 * static_cast<int64_t>(seq));
  const int32_t rest_first = record[2], rest_count = record[3];
  const int32_t prefix_entry = record[4], pieces = record[5], member = record[6];
  if (!plan_fits(plan, a.num_seqs, a.num_groups, a.num_kv_heads, a.group)) {
    // Another batch's plan: no partial was written.  NaN, not stale values.
    if (part_wave == 0) *dst = kHalf ? 0x7E007E00u : 0x7FC07FC0u;
    return;
  }
  const int32_t row = member * a.group + head;
  const int32_t tile = row / kTileRows;
  // The row's first partial; its pieces lie kTileRows apart.
  const int64_t prefix_row = kh * a.shape.prefix_rows +
                             (prefix_entry + static_cast<int64_t>(tile) * pieces) * kTileRows + row % kTileRows;
  const int64_t prefix_most = a.num_kv_heads * a.shape.prefix_rows - 1;
  const int64_t rest_row = a.num_kv_heads * a.shape.prefix_rows;
  const int32_t parts = pieces + rest_count;
  auto row_of = [&](int32_t p) -> int64_t {
    if (p < pieces) return min(prefix_row + static_cast<int64_t>(p) * kTileRows, prefix_most);
    const int64_t e = min(static_cast<int64_t>(rest_first) + p - pieces, a.shape.rest - 1);
    return rest_row + (e * a.num_kv_heads + kh) * a.group + head;
  };
  float run_max = -INFINITY, total = 0.f;
  f32x2 sum = {0.f, 0.f};
  for (int32_t p0 = part_wave * kMergeBatch; p0 < parts; p0 += kWaves * kMergeBatch) {
    f32x2 ml[kMergeBatch], v[kMergeBatch];
#pragma unroll
    for (int i = 0; i < kMergeBatch; ++i) {
      const int64_t at = row_of(min(p0 + i, parts - 1));
      ml[i] = a.part_ml[at];
      v[i] = *reinterpret_cast<const f32x2*>(a.part_acc + at * kDim + 2 * lane);
    }
    float top = run_max;
#pragma unroll
    for (int i = 0; i < kMergeBatch; ++i) {
      if (p0 + i >= parts) ml[i] = f32x2{-INFINITY, 0.f};  // a repeat of the last one
      top = fmaxf(top, ml[i].x);
    }
    const float keep = run_max == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(run_max - top);
    sum *= keep;
    total *= keep;
#pragma unroll
    for (int i = 0; i < kMergeBatch; ++i) {
      if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;
      const float f = ml[i].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[i].x - top);
      sum.x = __builtin_fmaf(v[i].x, f, sum.x);
      sum.y = __builtin_fmaf(v[i].y, f, sum.y);
      total = __builtin_fmaf(ml[i].y, f, total);
    }
    run_max = top;
  }
  if constexpr (kWaves > 1) {
    __shared__ f32x2 s_sum[kWaves][kWave];
    __shared__ f32x2 s_ml[kWaves];
    s_sum[part_wave][lane] = sum;
    if (lane == 0) s_ml[part_wave] = f32x2{run_max, total};
    __syncthreads();
    if (part_wave != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_ml[w].x);
    sum = f32x2{0.f, 0.f};
    total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const f32x2 ml = s_ml[w], v = s_sum[w][lane];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;
      const float f = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
      sum.x = __builtin_fmaf(v.x, f, sum.x);
      sum.y = __builtin_fmaf(v.y, f, sum.y);
      total = __builtin_fmaf(ml.y, f, total);
    }
  }
  typedef typename Elem<kHalf>::T T;
  const bool empty = total == 0.f;  // no key at all (a NaN sum is not empty)
  const T x = static_cast<T>(empty ? 0.f : sum.x / total), y = static_cast<T>(empty ? 0.f : sum.y / total);
  *dst = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, x)) |
         (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, y)) << 16);
}

bool layout_ok(int64_t num_seqs, int64_t num_groups, int64_t num_kv_heads, int64_t num_q_heads) {
  return num_seqs >= 0 && num_seqs <= NKV_MAX_PLAN_SEQS && num_groups >= 0 &&
         num_groups <= NKV_MAX_PLAN_SEQS && num_kv_heads > 0 && num_kv_heads <= 4096 &&
         num_q_heads > 0 && num_q_heads % num_kv_heads == 0 && num_q_heads / num_kv_heads <= kMaxGroup;
}

}  // namespace
}  // namespace nkv

extern "C" int64_t nkv_shared_plan_bytes(int64_t num_seqs, int64_t num_groups, int64_t num_kv_heads,
                                         int64_t num_q_heads, int64_t rest_tokens) {
  using namespace nkv;
  if (!layout_ok(num_seqs, num_groups, num_kv_heads, num_q_heads)) return 0;
  return 16 * plan_shape(num_seqs, num_groups, num_kv_heads, num_q_heads / num_kv_heads, rest_tokens).int4s();
}

extern "C" int64_t nkv_shared_workspace_bytes(int64_t num_seqs, int64_t num_groups, int64_t num_kv_heads,
                                              int64_t num_q_heads, int64_t rest_tokens) {
  using namespace nkv;
  if (!layout_ok(num_seqs, num_groups, num_kv_heads, num_q_heads)) return 0;
  const int64_t group = num_q_heads / num_kv_heads;
  return plan_shape(num_seqs, num_groups, num_kv_heads, group, rest_tokens).rows(num_kv_heads, group) *
         (kDim * 4 + 8);
}

extern "C" int nkv_build_shared_plan(const int32_t* cu_seqlens_k, int64_t num_seqs, const int32_t* cu_groups,
                                     const int32_t* prefix_lens, int64_t num_groups, int64_t num_kv_heads,
                                     int64_t num_q_heads, int64_t rest_tokens, void* plan,
                                     int64_t plan_bytes, void* stream) {
  using namespace nkv;
  if (!layout_ok(num_seqs, num_groups, num_kv_heads, num_q_heads)) {
    return nkv_fail(NKV_E_INVALID,
                    "nkv_build_shared_plan: need at most %d sequences and groups, and at most %d query "
                    "heads per kv head",
                    NKV_MAX_PLAN_SEQS, kMaxGroup);
  }
  const int64_t group = num_q_heads / num_kv_heads;
  const PlanShape shape = plan_shape(num_seqs, num_groups, num_kv_heads, group, rest_tokens);
  if (plan_bytes != 16 * shape.int4s()) {
    return nkv_fail(NKV_E_CAPACITY, "nkv_build_shared_plan: a plan of %lld bytes, exactly %lld are laid out",
                    static_cast<long long>(plan_bytes), static_cast<long long>(16 * shape.int4s()));
  }
  if (!plan || !cu_seqlens_k || (num_groups > 0 && (!cu_groups || !prefix_lens))) {
    return nkv_fail(NKV_E_INVALID, "nkv_build_shared_plan: null pointer");
  }
  if (reinterpret_cast<uint64_t>(plan) % 16 != 0) {
    return nkv_fail(NKV_E_INVALID, "nkv_build_shared_plan: plan must be 16-byte aligned");
  }
  const GroupOf groups{cu_seqlens_k, cu_groups, prefix_lens, static_cast<int32_t>(num_groups),
                       static_cast<int32_t>(num_seqs)};
  const size_t lds = (static_cast<size_t>(std::max(num_seqs, num_groups)) + 1) * sizeof(int32_t);
  shared_plan_kernel<<<dim3(1), dim3(kPlanThreads), lds, static_cast<hipStream_t>(stream)>>>(
      groups, static_cast<int32_t>(num_kv_heads), static_cast<int32_t>(group), shape, static_cast<int4*>(plan));
  return nkv_check_launch("nkv_build_shared_plan");
}

extern "C" int nkv_shared_prefix_attention_decode(
    const void* q, int64_t q_seq_stride, const void* key_cache, const void* value_cache,
    const int32_t* block_tables, int64_t table_stride, const void* plan, int64_t plan_bytes,
    int64_t num_seqs, int64_t num_groups, int64_t num_kv_heads, int64_t num_q_heads, int64_t head_dim,
    int64_t block_size, int64_t num_blocks, int64_t rest_tokens, float scale, int32_t dtype,
    void* workspace, int64_t workspace_bytes, void* out, int64_t out_seq_stride, void* stream) {
  using namespace nkv;
  const char* const what = "nkv_shared_prefix_attention_decode";
  if (dtype != NKV_DTYPE_BFLOAT16 && dtype != NKV_DTYPE_FLOAT16) {
    return nkv_fail(NKV_E_INVALID, "%s: only bfloat16 and float16 are supported", what);
  }
  if (head_dim != kDim) return nkv_fail(NKV_E_INVALID, "%s: head_dim must be %d", what, kDim);
  if (!layout_ok(num_seqs, num_groups, num_kv_heads, num_q_heads)) {
    return nkv_fail(NKV_E_INVALID,
                    "%s: need at most %d sequences and groups, and 1 to %d query heads per kv head", what,
                    NKV_MAX_PLAN_SEQS, kMaxGroup);
  }
  if (block_size <= 0 || num_blocks < 0 || num_blocks > INT32_MAX || block_size > INT32_MAX ||
      num_blocks * block_size > INT32_MAX || table_stride < 0 || q_seq_stride < num_q_heads * head_dim ||
      out_seq_stride < num_q_heads * head_dim) {
    return nkv_fail(NKV_E_INVALID, "%s: bad sizes or strides", what);
  }
  // The chunk max is taken of the raw scores: it commutes with scale > 0 only.
  if (!std::isfinite(scale) || !(scale > 0.f)) {
    return nkv_fail(NKV_E_INVALID, "%s: scale must be finite and positive", what);
  }
  if (num_seqs == 0) return NKV_OK;
  const int64_t group = num_q_heads / num_kv_heads;
  const PlanShape shape = plan_shape(num_seqs, num_groups, num_kv_heads, group, rest_tokens);
  if (plan_bytes != 16 * shape.int4s()) {
    return nkv_fail(NKV_E_CAPACITY, "%s: a plan of %lld bytes, exactly %lld are laid out", what,
                    static_cast<long long>(plan_bytes), static_cast<long long>(16 * shape.int4s()));
  }
  const int64_t rows = shape.rows(num_kv_heads, group);
  if (workspace_bytes < rows * (kDim * 4 + 8)) {
    return nkv_fail(NKV_E_CAPACITY, "%s: workspace of %lld bytes < %lld needed", what,
                    static_cast<long long>(workspace_bytes), static_cast<long long>(rows * (kDim * 4 + 8)));
  }
  if (!q || !key_cache || !value_cache || !plan || !workspace || !out || (table_stride > 0 && !block_tables)) {
    return nkv_fail(NKV_E_INVALID, "%s: null pointer", what);
  }
  if ((reinterpret_cast<uint64_t>(q) | reinterpret_cast<uint64_t>(key_cache) |
       reinterpret_cast<uint64_t>(value_cache) | reinterpret_cast<uint64_t>(plan) |
       reinterpret_cast<uint64_t>(workspace) | static_cast<uint64_t>(q_seq_stride * 2)) % 16 != 0 ||
      (reinterpret_cast<uint64_t>(out) | static_cast<uint64_t>(out_seq_stride * 2)) % 4 != 0) {
    return nkv_fail(NKV_E_INVALID,
                    "%s: q/caches/plan/workspace must be 16-byte aligned and out rows 4-byte aligned", what);
  }
  const int64_t items = shape.prefix * num_kv_heads + (shape.rest * num_kv_heads + 3) / 4;
  const int64_t pairs = num_seqs * num_q_heads;
  const bool four = pairs <= kMergePairs;
  const int64_t merges = four ? pairs : (pairs + 3) / 4;
  if (items > UINT32_MAX / kThreads || merges > UINT32_MAX / kThreads) {
    return nkv_fail(NKV_E_INVALID, "%s: too many sequences and heads for one launch", what);
  }
  SharedArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.key_cache = static_cast<const uint8_t*>(key_cache);
  a.value_cache = static_cast<const uint8_t*>(value_cache);
  a.tables = block_tables;
  a.plan = static_cast<const int4*>(plan);
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<f32x2*>(a.part_acc + rows * kDim);
  a.q_seq_stride = q_seq_stride;
  a.table_stride = table_stride;
  a.shape = shape;
  a.block_size = static_cast<int32_t>(block_size);
  a.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctzll(static_cast<uint64_t>(block_size)) : -1;
  a.num_blocks = static_cast<int32_t>(num_blocks);
  a.num_kv_heads = static_cast<int32_t>(num_kv_heads);
  a.group = static_cast<int32_t>(group);
  a.num_seqs = static_cast<int32_t>(num_seqs);
  a.num_groups = static_cast<int32_t>(num_groups);
  a.scale_log2 = scale * 1.4426950408889634f;  // log2(e)
  const bool half = dtype == NKV_DTYPE_FLOAT16;
  const bool chunked = block_size % kChunk == 0 && a.block_shift >= 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  void (*kernel)(SharedArgs) =
      chunked ? (half ? shared_attention_kernel<true, true> : shared_attention_kernel<true, false>)
              : (half ? shared_attention_kernel<false, true> : shared_attention_kernel<false, false>);
  kernel<<<dim3(static_cast<unsigned>(items)), dim3(kThreads), 0, s>>>(a);
  if (int rc = nkv_check_launch(what)) return rc;
  void (*merge)(SharedArgs, uint16_t*, int64_t) =
      four ? (half ? shared_merge_kernel<true, 4> : shared_merge_kernel<false, 4>)
           : (half ? shared_merge_kernel<true, 1> : shared_merge_kernel<false, 1>);
  merge<<<dim3(static_cast<unsigned>(merges)), dim3(256), 0, s>>>(
      a, static_cast<uint16_t*>(out), out_seq_stride);
  return nkv_check_launch(what);
}
