// Attention over a paged cache for sequences of many rows (more than 16 packed rows: rows times query heads per kv
// head), on the tensor cores: 4 d flops per visible pair of row and key.
//
// A CTA takes a unit of up to 256 packed rows of one kv head of one sequence, as one or two tiles of 128, and tiles of
// 128 keys. Two streams keep the tensor core busy while softmax runs: with two row tiles each stream has one and both
// see every key tile; with one row tile (128 rows or fewer) the streams take the key tiles in turn and their results are
// joined at the end. Per stream and key tile
//     S[128, 128] = Q K^T     tcgen05.mma, both operands in shared memory, S in tensor memory;
//     P = 2^(S scale - m)     a thread per row: S from tensor memory, P (16 bit) back over S's own columns;
//     O[128, d] += P V        tcgen05.mma, P from tensor memory, V [key][d] as a transposed operand.
// A thread for each stream issues its P V and the next Q K', so one stream's two products (4 x 128 x 128 x d flops) run
// under the other one's softmax. Products of one thread execute in order, so S may be overwritten as soon as the product
// that reads P has been issued.
//
// Roles: warps 0-3 and 4-7 do the softmax of stream 0 and 1, warps 8-11 fetch keys and values (16-bit pages by 16-byte
// asynchronous copies, e4m3 codes through registers, exactly to f16), a thread each of warps 12 and 13 issues the products
// of stream 0 and 1. Operands lie in 128-byte rows with the 128-byte swizzle, d = 128 in two panels. Every wait is bounded.
//
// What bounds it: the chain of a stream, Q K (650 clocks from the first issue to the last product accepted, 250 more to
// the waiting warps), softmax (2300: 128 exponentials a thread at 8 clocks a warp are 1024 of them), P V (620), commits
// and barriers (700), 4.8 thousand for 128 keys of 16-bit pages against the 2130 clocks that the four products of two
// streams take. With e4m3 pages it is 7 thousand: softmax goes in two short loops, and the fetching warps bring codes to
// f16 on the same schedulers. The first tile is in softmax 7 thousand clocks after the CTA starts, the output takes 6, so
// the tensor core is busy 30 % of a call. With one row tile the rings of two hold one key tile for each stream, whose next
// one is fetched late: 4 us a key tile and CTA (16 heads, 56 rows: 17 us over 256 keys, 33 over 4152, 72 over 16440).
// Measured: 2048 rows, 16 heads, over 6000 + 2048 e4m3 keys 236 us (501 TFLOP/s, 31 % of a large bf16 product's rate);
// 8191 rows, 16 heads over 4, window 1024, 139 us (465 TFLOP/s of visible pairs).
//
// Softmax: base 2, lazy maximum (O is rescaled only when a score passes m by more than 2^15), scales of e4m3 pages kept
// out of 16-bit numbers and queries in bf16 brought to f16 exactly, as cache_decode.cu describes.
//
// With too few units for the GPU, several CTAs split a unit's keys; their parts go to the workspace and join_parts_kernel
// adds them up in order.
//
// Masked tiles: see cache_decode.cu. Non-finite values of tiles that not every row sees are replaced by 0 on the way into
// shared memory; the CTA then reads those tiles' values again at the end and adds the non-finite ones to the rows that
// see them.
#include "cache_attention.cuh"

namespace plm {
namespace {

constexpr int kTile = 128;  // rows of a stream, and keys
constexpr int kUnit = 2 * kTile;
constexpr int kRoleThreads = 128;
constexpr int kPrefillThreads = 3 * kRoleThreads + 64;
constexpr int kScaleSlots = 4;
constexpr uint32_t kTmemColumns = 512;
constexpr float kGuess = -4.f;  // a row's maximum, in units of log2, before it has seen a key

constexpr int kFetchBytes = 3328;

template <int HD>
struct PrefillSmem {
  static constexpr int TILE = kTile * HD * 2;  // a tile of 128 rows, keys or values
  static constexpr int Q = 0;
  static constexpr int K = 2 * TILE;
  static constexpr int V = 4 * TILE;
  static constexpr int SCALES = 6 * TILE;      // [slot] TileScales
  static constexpr int FETCH = SCALES + kScaleSlots * 3 * kTile * 4;  // FetchRows
  static constexpr int BARRIERS = FETCH + kFetchBytes;
  static constexpr int UNIT = BARRIERS + 256;
  static constexpr int BYTES = UNIT + 256 + 1024;  // and the alignment's slack
};

struct PrefillBarriers {
  uint64_t q_ready, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], pv_done[2],
      scales_full[kScaleSlots];
  int one[kScaleSlots];  // 0: the tile has more than one scale; otherwise 1 + spread of its values'
  uint32_t tmem;
  int issuing;  // held by the stream that issues products
  int odd;  // a value that is no number was met in a masked tile
};
static_assert(sizeof(PrefillBarriers) <= 256, "barriers");

// What a unit's parts are joined from.
struct SplitUnit {
  int row0, i0, rows, head;
};
constexpr size_t split_unit_bytes(int64_t units) { return (size_t(units) * sizeof(SplitUnit) + 127) & ~size_t(127); }
// Whether all lanes' waits came to an end in time: the warp goes on, or gives up, together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

template <int HD>
constexpr size_t part_floats() {
  return size_t(kUnit) * (HD + 2);
}

// D(tmem) (+)= A(tmem) B(smem)
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A tile of [k][m or n] rows of 128 bytes with the 128-byte swizzle as a transposed operand: 64 elements along m or n to
// a row, panels of 64 `panel` bytes apart, groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc_transposed(uint32_t smem_addr, uint32_t panel) {
  uint64_t d = 0;
  d |= uint64_t((smem_addr >> 4) & 0x3FFF);
  d |= uint64_t((panel >> 4) & 0x3FFF) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
// 16 words of every lane into 16 columns of tensor memory.
__device__ __forceinline__ void tmem_st_16cols(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 32 columns of every lane, to be waited for with tmem_wait_ld.
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Byte offset of 16-byte vector `vec` of row `row` in a tile of 128 rows of d 16-bit elements.
__device__ __forceinline__ int tile_at(int row, int vec) {
  return (vec >> 3) * (kTile * 128) + row * 128 + (((vec & 7) ^ (row & 7)) << 4);
}

// Which key tiles of a CTA each stream works on: with one row tile every second one; with two row tiles the sinks' and
// those that some of its rows see.
struct Turns {
  int two;             // row tiles: 1 for two
  int t_begin, t_end;  // the CTA's key tiles
  int sinks0, begin0, end0, sinks1, begin1, end1;
  // (Fields by stream, not arrays: an index known only at run time would put them into local memory.)
  // The stream's first tile from t on (t_end or more: none).
  __device__ __forceinline__ int next(int s, int t) const {
    if (!two) return t + (((t - t_begin) ^ s) & 1);
    if (t < (s ? sinks1 : sinks0)) return t;
    t = max(t, s ? begin1 : begin0);
    return t < (s ? end1 : end0) ? t : t_end;
  }
};

// What a CTA works on.
struct Unit {
  SeqRange r;
  int seq, head, i0, rows;   // packed rows [i0, i0 + rows); rows 0: nothing
  TileKeys keys;             // of all its rows, in tiles of 128 keys
  TileKeys stream_keys[2];   // of a stream's rows
  Turns turns;
};
static_assert(sizeof(Unit) <= 256, "unit");

// Unit `index` of the call's rows, or false past the last one. All threads of a warp together.
__device__ __forceinline__ bool find_unit(const CacheAttnArgs& a, int index, int head, int split, Unit* u) {
  const int lane = threadIdx.x & 31;
  int before = 0, unit = 0;
  bool found = false;
  for (int base = 0; base < a.s.n_seqs && !found; base += 32) {
    SeqRange r = {0, 0, 0};
    if (base + lane < a.s.n_seqs) r = sequence_range(a.s, base + lane, a.err);
    const int count = (r.n * a.group + kUnit - 1) / kUnit;
    int upto = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += other;
    }
    upto += before;
    const uint32_t past = __ballot_sync(0xffffffffu, upto > index);
    if (past != 0) {
      const int owner = __ffs(past) - 1;
      u->r.start = __shfl_sync(0xffffffffu, r.start, owner);
      u->r.n = __shfl_sync(0xffffffffu, r.n, owner);
      u->r.context = __shfl_sync(0xffffffffu, r.context, owner);
      u->seq = base + owner;
      const int units = __shfl_sync(0xffffffffu, count, owner);
      unit = units - 1 - (index - __shfl_sync(0xffffffffu, upto - count, owner));  // the longest first
      found = true;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  if (!found) return false;
  u->head = head;
  u->i0 = unit * kUnit;
  u->rows = min(kUnit, u->r.n * a.group - u->i0);
  const bool two = u->rows > kTile;
  const int j0 = u->i0 / a.group, j1 = (u->i0 + u->rows - 1) / a.group;
  TileKeys t = causal_keys(a, u->r, j0, j1);
  if (a.depth != nullptr) {
    t.end = int(u->r.context) + u->r.n;
    t.lo = t.full_end = kUnreachable;
    t.full_lo = 0;
    for (int j = j0 + lane; j <= j1; j += 32) widen(t, row_mask(a, u->r, j));
    t.lo = min(t.end, int(__reduce_min_sync(0xffffffffu, t.lo)));
    t.full_lo = __reduce_max_sync(0xffffffffu, t.full_lo);
    t.full_end = __reduce_min_sync(0xffffffffu, t.full_end);
    t.sinks = min(a.sinks, t.lo);
  }
  t.count<kTile>();
  u->keys = u->stream_keys[0] = u->stream_keys[1] = t;
  Turns& turns = u->turns;
  turns.two = two ? 1 : 0;
  turns.t_begin = int(int64_t(split) * t.chunks / a.splits);
  turns.t_end = int(int64_t(split + 1) * t.chunks / a.splits);
  turns.sinks0 = turns.begin0 = turns.sinks1 = turns.begin1 = 0;
  turns.end0 = turns.end1 = t.chunks;
  if (two && a.depth == nullptr) {
    const int mid = u->i0 + kTile;
    const int main = t.sink_chunks - t.lo / kTile;  // from a key's tile to its number
    auto limit = [&](const TileKeys& k, int& sinks, int& begin, int& end) {
      sinks = min(t.sink_chunks, (k.sinks + kTile - 1) / kTile);
      begin = k.sinks > t.lo / kTile * kTile ? t.sink_chunks : main + k.lo / kTile;
      end = main + (k.end + kTile - 1) / kTile;
    };
    u->stream_keys[0] = causal_keys(a, u->r, j0, (mid - 1) / a.group);
    u->stream_keys[1] = causal_keys(a, u->r, mid / a.group, j1);
    limit(u->stream_keys[0], turns.sinks0, turns.begin0, turns.end0);
    limit(u->stream_keys[1], turns.sinks1, turns.begin1, turns.end1);
  }
  return true;
}

// Places of keys in the pages.
constexpr uint32_t kNoRow = 0xffffffffu;
struct PageRows {
  const int32_t* table;
  int page_shift, page_mask, num_pages, kv_heads, head;
  int* err;
  // Key kv's row within a plane, in rows of d elements (a plane on the device has fewer than 2^32), or kNoRow where
  // there is none to fetch.
  __device__ __forceinline__ uint32_t row(const TileKeys& t, int kv) const {
    if (!t.needed(kv)) return kNoRow;
    const int page = table[kv >> page_shift];
    if (unsigned(page) >= unsigned(num_pages)) {
      record_error(err, kErrBadIndex);
      return kNoRow;
    }
    return (uint32_t(page) * uint32_t(kv_heads) + uint32_t(head)) * uint32_t(page_mask + 1) + uint32_t(kv & page_mask);
  }
};

template <typename T, bool E4M3>
__device__ __forceinline__ bool any_non_finite(const uint4& x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int at = 0; at < (E4M3 ? 4 : 2); ++at) any |= non_finite<T, E4M3>(w[i], at);
  return any;
}
template <typename T, bool E4M3>
__device__ __forceinline__ void drop_non_finite(uint4& x) {
  uint32_t* w = &x.x;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int at = 0; at < (E4M3 ? 4 : 2); ++at)
      if (non_finite<T, E4M3>(w[i], at)) w[i] &= ~((E4M3 ? 0xffu : 0xffffu) << ((E4M3 ? 8 : 16) * at));
}

// What softmax needs to know of a tile of e4m3 keys. Normally the scales of a tile are powers of two within 2^15 of
// each other, and the codes are brought to the largest one's on the way into shared memory, exactly: then the tile has
// one scale. Otherwise they stay as they are, and softmax applies the scales key by key. A weight that goes by the tile's
// scale of values may lie above its key's own term by what the scales lie apart, 2^spread. Softmax keeps m so far below the
// largest weight, so that f16, whose smallest step is 2^-24, holds every term to 2^-25 of the largest term of the sum; the
// lazy maximum has that much less room (2048 rows over 8048 keys, scales within 1, 2^6 and 2^14: 234, 236 and 238 us; one
// fixed reserve of 2^5, and key by key beyond it: 231, 255 and 361).
struct TileScales {
  float k[kTile], log_v[kTile], inv_v[kTile];  // by key; where `one`, the first of each is the tile's
};

// What the fetching threads share of a tile.
struct FetchRows {
  uint32_t row[2][kTile];                            // of a tile's keys, in turns of two
  float k_relative[2][kTile], v_relative[2][kTile];  // e4m3: the share of the tile's largest scale that a key's is, or 1
  float low[2][4], high[2][4];                       // K's and V's, by warp
  int odd[2][4];
  int abort;                                         // a wait ran out: the four warps stop together
};
static_assert(sizeof(TileScales) == 3 * kTile * 4 && sizeof(FetchRows) <= kFetchBytes, "shared memory");

// Of the scales of a tile's keys, a key each thread (`live` false: none), what one warp sees of them.
__device__ __forceinline__ void note_scales(FetchRows* rows, int which, bool live, float scale) {
  const int tid = threadIdx.x & (kRoleThreads - 1);
  const float low = -warp_max(live ? -scale : -INFINITY), high = warp_max(live ? scale : 0.f);
  const bool odd = __any_sync(0xffffffffu, live && ((__float_as_uint(scale) & 0x7fffffu) != 0 ||
                                                    !(scale > 0.f && scale < INFINITY)));
  if ((tid & 31) == 0) {
    rows->low[which][tid >> 5] = low;
    rows->high[which][tid >> 5] = high;
    rows->odd[which][tid >> 5] = odd ? 1 : 0;
  }
}
// Whether the tile has one scale, after a barrier; *top is the largest, 2^*spread of the smallest, *relative the share of it
// that `scale` is.
__device__ __forceinline__ bool one_scale(const FetchRows* rows, int which, bool live, float scale, float* relative,
                                          float* top, int* spread) {
  const float* low = rows->low[which];
  const float* high = rows->high[which];
  const int* odd = rows->odd[which];
  *top = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
  const float least = fminf(fminf(low[0], low[1]), fminf(low[2], low[3]));
  const bool one = (odd[0] | odd[1] | odd[2] | odd[3]) == 0 && *top > 0.f && least * 32768.f >= *top;
  // quotients of powers of two
  *spread = int(__float_as_uint(*top) - __float_as_uint(least)) >> 23;
  *relative = one && live ? __uint_as_float(__float_as_uint(scale) - __float_as_uint(*top) + 0x3f800000u) : 1.f;
  return one;
}

// Fetches all key and value tiles of the CTA into their rings of two: 128 threads.
template <int HD, typename T, bool E4M3>
__device__ __forceinline__ void fetch_tiles(const CacheAttnArgs& a, const Unit& u, uint8_t* smem, PrefillBarriers* bars) {
  using S = PrefillSmem<HD>;
  constexpr int NAMED = 2;
  const int tid = threadIdx.x & (kRoleThreads - 1), lane = tid & 31;
  FetchRows* share = reinterpret_cast<FetchRows*>(smem + S::FETCH);
  constexpr int ES = E4M3 ? 1 : 2;
  constexpr int VECS = HD * ES / 16;            // 16-byte vectors of a row in the page
  constexpr int PER_PASS = kRoleThreads / VECS; // rows that the threads fetch together
  constexpr int PASSES = kTile / PER_PASS;
  const int vec = tid % VECS, first = tid / VECS;
  const uint8_t* const k_plane = static_cast<const uint8_t*>(a.c.k) + vec * 16;
  const uint8_t* const v_plane = static_cast<const uint8_t*>(a.c.v) + vec * 16;
  const PageRows rows = {a.s.tables + u.seq * a.s.table_stride, a.c.page_shift, a.c.page_size - 1,
                         a.c.num_pages, a.c.kv_heads, u.head, a.err};
  const TileKeys keys = u.keys;
  const int t_begin = u.turns.t_begin, tiles = u.turns.t_end - t_begin;
  auto arrive = [&](uint64_t* bar) {
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  // A tile's place in a ring, free: false (for all four warps) once a wait has run out.
  auto place = [&](uint64_t* empty, int n) {
    if (n < 2) return true;
    if (!warp_wait(empty + (n & 1), ((n >> 1) - 1) & 1, a.err, kErrTimeoutEmpty)) share->abort = 1;
    named_barrier_sync(NAMED, kRoleThreads);
    return share->abort == 0;
  };
  auto row_of = [&](int n) { return n < tiles ? rows.row(keys, keys.key<kTile>(t_begin + n) + tid) : kNoRow; };
  auto masked = [&](int n) { return !keys.all_seen(keys.key<kTile>(t_begin + n), kTile); };  // not every row sees every key
  if constexpr (!E4M3) {
    // In turns the copies of K(n) and V(n - 1), and of V(n) and K(n), are on their way together. What a place waits for
    // needs no tile that has not been announced: K(n)'s place the products Q K(n - 2), V(n)'s the products P V(n - 2).
    uint32_t next = row_of(0);
    auto copy = [&](uint8_t* dst, const uint8_t* plane, int n) {
      const uint32_t* const row = share->row[n & 1];
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const uint32_t from = row[first + p * PER_PASS];
        cp_async_16(dst + (n & 1) * S::TILE + tile_at(first + p * PER_PASS, vec),
                    plane + (from == kNoRow ? 0 : size_t(from) * (HD * ES)), from != kNoRow);
      }
      cp_async_commit();
    };
    auto values_landed = [&](int n) {
      if (masked(n)) {
#pragma unroll 1
        for (int p = 0; p < PASSES; ++p) {
          uint4* x = reinterpret_cast<uint4*>(smem + S::V + (n & 1) * S::TILE + tile_at(first + p * PER_PASS, vec));
          if (any_non_finite<T, false>(*x)) {
            drop_non_finite<T, false>(*x);
            bars->odd = 1;
          }
        }
      }
      arrive(bars->v_full + (n & 1));
    };
    int n = 0;
    for (; n < tiles; ++n) {
      share->row[n & 1][tid] = next;
      next = row_of(n + 1);
      named_barrier_sync(NAMED, kRoleThreads);
      if (!place(bars->k_empty, n)) break;
      copy(smem + S::K, k_plane, n);
      if (n > 0) {
        cp_async_wait<1>();
        values_landed(n - 1);
      }
      if (!place(bars->v_empty, n)) break;
      copy(smem + S::V, v_plane, n);
      cp_async_wait<1>();
      arrive(bars->k_full + (n & 1));
    }
    cp_async_wait<0>();
    if (n == tiles && tiles > 0) values_landed(tiles - 1);
  } else {
    // A tile's codes are on their way to registers while the tile before is stored.
    auto load = [&](uint4(&codes)[PASSES], const uint8_t* plane, int n) {
      const uint32_t* const row = share->row[n & 1];
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const uint32_t from = row[first + p * PER_PASS];
        codes[p] = make_uint4(0, 0, 0, 0);
        if (from != kNoRow) codes[p] = *reinterpret_cast<const uint4*>(plane + size_t(from) * HD);
      }
    };
    // 16 codes of a row to f16 times the row's share of the tile's scale, exactly.
    auto store = [&](uint8_t* dst, const uint4(&codes)[PASSES], const float* relative) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int at = first + p * PER_PASS;
        const __half2 by = __float2half2_rn(relative[at]);
        const uint32_t w[4] = {codes[p].x, codes[p].y, codes[p].z, codes[p].w};
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = e4m3x2_to_f16x2(uint16_t(w[i / 2] >> (16 * (i & 1))));
          const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x), by);
          h[i] = *reinterpret_cast<const uint32_t*>(&y);
        }
        // the upper half of a row's threads the other way round: all eight groups of banks in each store
        const uint4 x = make_uint4(h[0], h[1], h[2], h[3]), y = make_uint4(h[4], h[5], h[6], h[7]);
        const bool swap = HD == 128 && vec >= 4;
        *reinterpret_cast<uint4*>(dst + tile_at(at, 2 * vec + (swap ? 1 : 0))) = swap ? y : x;
        *reinterpret_cast<uint4*>(dst + tile_at(at, 2 * vec + (swap ? 0 : 1))) = swap ? x : y;
      }
    };
    auto block_of = [&](uint32_t row) { return row == kNoRow ? 0 : row >> a.c.block_shift; };  // blocks divide pages
    uint4 k_codes[PASSES], v_codes[PASSES];
    uint32_t mine = row_of(0), next = row_of(1);
    float ks = a.c.k_scale[block_of(mine)], vs = a.c.v_scale[block_of(mine)];
    share->row[0][tid] = mine;
    named_barrier_sync(NAMED, kRoleThreads);
    if (tiles > 0) {
      load(k_codes, k_plane, 0);
      load(v_codes, v_plane, 0);
    }
    for (int n = 0; n < tiles; ++n) {
      const bool live = mine != kNoRow;
      if (!live) ks = vs = 1.f;
      vs = fmaxf(vs, kLeastScale);
      share->row[(n + 1) & 1][tid] = next;
      note_scales(share, 0, live, ks);
      note_scales(share, 1, live, vs);
      named_barrier_sync(NAMED, kRoleThreads);
      float k_relative, v_relative, k_top, v_top;
      int k_spread, v_spread;
      const bool k_one = one_scale(share, 0, live, ks, &k_relative, &k_top, &k_spread);
      const bool v_one = one_scale(share, 1, live, vs, &v_relative, &v_top, &v_spread);
      share->k_relative[n & 1][tid] = k_relative;
      share->v_relative[n & 1][tid] = v_relative;
      mine = next;
      const float ks_next = a.c.k_scale[block_of(mine)], vs_next = a.c.v_scale[block_of(mine)];
      next = row_of(n + 2);
      if (!place(bars->k_empty, n)) break;
      {
        // The scales' slot: its last readers, the softmax of tile n - 4, are done. The products Q K of tiles n - 3 and
        // n - 2 have run, and a stream's products start only when its softmax of the tile before is over.
        const int slot = n % kScaleSlots;
        TileScales& scales = reinterpret_cast<TileScales*>(smem + S::SCALES)[slot];
        const float v = v_one ? v_top : vs;
        scales.k[tid] = k_one ? k_top : ks;
        scales.log_v[tid] = lg2(v);
        scales.inv_v[tid] = rcp(v);
        if (tid == 0) bars->one[slot] = k_one && v_one ? 1 + v_spread : 0;
        named_barrier_sync(NAMED, kRoleThreads);  // and every key's share of the scale is there
        if (lane == 0) mbar_arrive(bars->scales_full + slot);
      }
      ks = ks_next;
      vs = vs_next;
      store(smem + S::K + (n & 1) * S::TILE, k_codes, share->k_relative[n & 1]);
      arrive(bars->k_full + (n & 1));
      load(k_codes, k_plane, n + 1);
      if (masked(n)) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          if (any_non_finite<T, true>(v_codes[p])) {
            drop_non_finite<T, true>(v_codes[p]);
            bars->odd = 1;
          }
        }
      }
      if (!place(bars->v_empty, n)) break;
      store(smem + S::V + (n & 1) * S::TILE, v_codes, share->v_relative[n & 1]);
      arrive(bars->v_full + (n & 1));
      load(v_codes, v_plane, n + 1);
    }
  }
}

// A stream's products: one thread each, with as little to do as can be (alone, a thread takes five or more clocks for an
// instruction, and every one stands in the stream's chain Q K, softmax, P V).
template <int HD, bool BF16>
__device__ __forceinline__ void issue_products(const CacheAttnArgs& a, const Turns& turns, const int stream, uint8_t* smem,
                                               PrefillBarriers* bars) {
  using S = PrefillSmem<HD>;
  constexpr uint32_t QK = umma_idesc_f16(kTile, kTile, BF16);
  constexpr uint32_t PV = umma_idesc_f16(kTile, HD, BF16) | (1u << 16);  // B transposed
  constexpr int PANEL = kTile * 128;
  constexpr int STEP = S::TILE >> 4;  // a tile, in a descriptor's units
  const bool two = turns.two != 0;
  const uint32_t t_s = bars->tmem + stream * kTile, t_o = t_s + 2 * kTile;
  const uint64_t q = umma_desc_sw128(smem_u32(smem + S::Q + (two ? stream : 0) * S::TILE));
  const uint64_t k_desc = umma_desc_sw128(smem_u32(smem + S::K));
  const uint64_t v_desc = umma_desc_transposed(smem_u32(smem + S::V), PANEL);
  // Tile numbers within the CTA: this stream's sinks and range, and the other one's.
  const int t0 = turns.t_begin, tiles = turns.t_end - t0;
  const int sinks = (stream ? turns.sinks1 : turns.sinks0) - t0, begin = (stream ? turns.begin1 : turns.begin0) - t0,
            end = min(tiles, (stream ? turns.end1 : turns.end0) - t0);
  const int o_sinks = (stream ? turns.sinks0 : turns.sinks1) - t0, o_begin = (stream ? turns.begin0 : turns.begin1) - t0,
            o_end = (stream ? turns.end0 : turns.end1) - t0;
  auto next = [&](int n) {
    if (!two) return n + ((n ^ stream) & 1);
    if (n >= sinks) n = max(n, begin);
    return n < end || n < sinks ? n : tiles;
  };
  auto release = [&](uint64_t* empty, int n) {  // both streams' arrivals, where the other one has no use for the tile
    umma_commit(empty + (n & 1));
    if (!two || !(n < o_sinks || (n >= o_begin && n < o_end))) umma_commit(empty + (n & 1));
  };
  if (!mbar_wait(&bars->q_ready, 0, a.err, kErrTimeoutPeer)) return;
  int n = next(0);
  // Products are issued one stream at a time, and P V together with the next Q K: were two streams' products to mix, both
  // would end late, both softmaxes would run at the same time, and the tensor core would idle under them. The lock is never
  // held over a wait.
  auto lock = [&]() {
    for (uint32_t looks = 1; atomicExch(&bars->issuing, 1) != 0; ++looks)
      if (looks == (1u << 24)) {
        record_error(a.err, kErrTimeoutPeer);
        return false;
      }
    return true;
  };
  auto unlock = [&]() { atomicExch(&bars->issuing, 0); };
  auto scores = [&](int n) {
    const uint64_t k = k_desc + (n & 1) * STEP;
#pragma unroll
    for (int x = 0; x < HD / 16; ++x) {
      const int off = ((x >> 2) * PANEL + (x & 3) * 32) >> 4;
      umma_f16(t_s, q + off, k + off, QK, x > 0 ? 1u : 0u);
    }
  };
  if (n >= tiles) return;
  if (!mbar_wait(bars->k_full + (n & 1), (n >> 1) & 1, a.err, kErrTimeoutFull) || !lock()) return;
  tc_fence_after();
  scores(n);
  unlock();
  umma_commit(bars->s_full + stream);
  release(bars->k_empty, n);
  for (int count = 0;; ++count) {
    const int after = next(n + 1), at = n & 1;
    if (!mbar_wait(bars->v_full + at, (n >> 1) & 1, a.err, kErrTimeoutFull) ||
        !mbar_wait(bars->p_ready + stream, count & 1, a.err, kErrTimeoutPeer) || !lock())
      return;
    tc_fence_after();
    const uint64_t v = v_desc + at * STEP;
    const uint32_t first = count > 0 ? 1u : 0u;
#pragma unroll
    for (int x = 0; x < kTile / 16; ++x)
      umma_f16_ts(t_o, t_s + x * 8, v + ((x * 2048) >> 4), PV, x > 0 ? 1u : first);
    // Commits take their time; but without its keys the next product may be waiting for this tile's place.
    const bool ready = after < tiles && mbar_try_wait(bars->k_full + (after & 1), (after >> 1) & 1);
    if (ready) {
      tc_fence_after();
      scores(after);
      unlock();
      umma_commit(bars->s_full + stream);
      umma_commit(bars->pv_done + stream);
      release(bars->v_empty, n);
      release(bars->k_empty, after);
    } else {
      unlock();
      umma_commit(bars->pv_done + stream);
      release(bars->v_empty, n);
      if (after >= tiles) return;
      if (!mbar_wait(bars->k_full + (after & 1), (after >> 1) & 1, a.err, kErrTimeoutFull) || !lock()) return;
      tc_fence_after();
      scores(after);
      unlock();
      umma_commit(bars->s_full + stream);
      release(bars->k_empty, after);
    }
    n = after;
  }
}

// A thread's packed rows when the threads of a stream go through its tile together, every N-th: as row of the sequence
// and head of the group.
template <int N>
struct RowWalk {
  static constexpr int STEP = N;
  int packed, j, g, dj, dg;
  __device__ __forceinline__ void advance(int group) {
    packed += N;
    j += dj;
    g += dg;
    if (g >= group) {
      g -= group;
      ++j;
    }
  }
};

template <int HD, typename T, bool E4M3>
__global__ void __launch_bounds__(kPrefillThreads, 1) prefill_attention_kernel(const CacheAttnArgs a) {
  using M = typename std::conditional<E4M3, __half, T>::type;  // type of the products
  using S = PrefillSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PrefillBarriers* bars = reinterpret_cast<PrefillBarriers*>(smem + S::BARRIERS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dependency_wait();
  allow_dependents();
  const int split = blockIdx.x % a.splits, index = blockIdx.x / a.splits;
  const Unit& u = *reinterpret_cast<const Unit*>(smem + S::UNIT);
  if (warp == 1) {
    Unit found;
    found.rows = 0;
    find_unit(a, index / a.c.kv_heads, index % a.c.kv_heads, split, &found);
    if (lane == 0) *reinterpret_cast<Unit*>(smem + S::UNIT) = found;
  }
  if (tid == 0) {
    mbar_init(&bars->q_ready, 8);
    bars->issuing = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars->k_full + i, 4);
      mbar_init(bars->k_empty + i, 2);
      mbar_init(bars->v_full + i, 4);
      mbar_init(bars->v_empty + i, 2);
      mbar_init(bars->s_full + i, 1);
      mbar_init(bars->p_ready + i, 4);
      mbar_init(bars->pv_done + i, 1);
    }
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(bars->scales_full + i, 4);
    bars->odd = 0;
    reinterpret_cast<FetchRows*>(smem + S::FETCH)->abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  if (u.rows == 0) {  // past the last unit
    if (a.splits > 1 && split == 0 && tid == 0) static_cast<SplitUnit*>(a.workspace)[index].rows = 0;
    return;
  }
  if (warp == 0) tmem_alloc(&bars->tmem, kTmemColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  const int role = tid / kRoleThreads;
  if (role == 2) {
    fetch_tiles<HD, T, E4M3>(a, u, smem, bars);
  } else if (role == 3) {
    if (lane == 0) {
      const Turns turns = u.turns;
      issue_products<HD, std::is_same<M, __nv_bfloat16>::value>(a, turns, warp & 1, smem, bars);
    }
  } else {
    const int stream = role;
    float m = -INFINITY, l = 0.f;
    int done = 0;  // key tiles this stream has worked on
    bool ok = true;
    const uint32_t t_lane = tmem + (uint32_t((warp & 3) * 32) << 16);
    const int row = tid & (kRoleThreads - 1);                       // of the stream's tile
    const int i = u.i0 + (u.turns.two && stream == 1 ? kTile : 0) + row;  // packed row
    const bool live = i < u.i0 + u.rows;
    // ---- the stream's queries into shared memory (with one row tile both streams' are the same, and stream 0 brings
    // them): 16-byte vectors along the rows, then each row to f16 by its own thread where that has to be
    constexpr bool RESCALE = E4M3 && std::is_same<T, __nv_bfloat16>::value;
    constexpr int QV = HD / 8;  // vectors of a row
    using Walk = RowWalk<kRoleThreads / QV>;
    const int walk_first = i - row + row / QV;
    const Walk walk = {walk_first, walk_first / a.group, walk_first % a.group, Walk::STEP / a.group, Walk::STEP % a.group};
    uint8_t* const q_tile = smem + S::Q + (u.turns.two ? stream : 0) * S::TILE;
    const int unit_rows = u.i0 + u.rows;
    if (u.turns.two || stream == 0) {
      Walk at = walk;
#pragma unroll
      for (int p = 0; p < QV; ++p, at.advance(a.group)) {
        const bool there = at.packed < unit_rows;
        const T* from = static_cast<const T*>(a.q) + (u.r.start + at.j) * a.q_stride + (u.head * a.group + at.g) * HD;
        cp_async_16(q_tile + tile_at(row / QV + p * Walk::STEP, row % QV),
                    there ? from + row % QV * 8 : static_cast<const T*>(a.q), there);
      }
      cp_async_commit();
      cp_async_wait<0>();
    }
    float q_scale = a.scale_log2;
    if constexpr (RESCALE) {
      named_barrier_sync(1, 2 * kRoleThreads);  // both streams read the rows, one may write them
      uint32_t top = 0;
#pragma unroll
      for (int vec = 0; vec < QV; ++vec) {
        const uint4 x = *reinterpret_cast<const uint4*>(q_tile + tile_at(row, vec));
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
      }
      const int e = query_exponent(top);
      const float up = power_of_two_f32(-e);
      q_scale *= power_of_two_f32(e);
      named_barrier_sync(1, 2 * kRoleThreads);
      if (u.turns.two || stream == 0) {
#pragma unroll
        for (int vec = 0; vec < QV; ++vec) {
          uint4* at = reinterpret_cast<uint4*>(q_tile + tile_at(row, vec));
          const uint4 x = *at;
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          uint32_t h[4];
#pragma unroll
          for (int y = 0; y < 4; ++y)
            h[y] = pack2<__half>(__uint_as_float(w[y] << 16) * up, __uint_as_float(w[y] & 0xffff0000u) * up);
          *at = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
    }
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->q_ready);
    auto row_sees = [&]() { return live ? row_mask(a, u.r, i / a.group) : no_row(); };
    const Turns turns = u.turns;
    const int full_lo = u.stream_keys[stream].full_lo, full_end = u.stream_keys[stream].full_end,
              full_sinks = u.stream_keys[stream].sinks;
    const uint32_t t_s = t_lane + stream * kTile, t_o = t_lane + 2 * kTile + stream * kTile;

    for (int n = turns.next(stream, turns.t_begin) - turns.t_begin; n < turns.t_end - turns.t_begin;
         n = turns.next(stream, turns.t_begin + n + 1) - turns.t_begin) {
      const int kv0 = u.keys.key<kTile>(turns.t_begin + n);
      const bool full = kv0 + kTile <= full_end && (kv0 >= full_lo || kv0 + kTile <= full_sinks);
      const int slot = n % kScaleSlots;
      ok = (!E4M3 || warp_wait(bars->scales_full + slot, (n / kScaleSlots) & 1, a.err, kErrTimeoutFull)) &&
           warp_wait(bars->s_full + stream, done & 1, a.err, kErrTimeoutDone);
      if (!ok) break;
      tc_fence_after();
      // A score x counts as x by + add, in units of log2 and with its value's scale in it; a weight w as w inv_v in l.
      const TileScales& scales = reinterpret_cast<const TileScales*>(smem + S::SCALES)[slot];
      float by = q_scale, add = 0.f, inv_v = 1.f;  // by is above 0, so that -inf by stays -inf
      const bool one = !E4M3 || bars->one[slot] != 0;
      if (E4M3 && one) {
        by *= scales.k[0];
        add = scales.log_v[0];
        inv_v = scales.inv_v[0];
      }
      by = fmaxf(by, 1.17549435e-38f);
      // Bit e: whether the row sees key c + e of the tile, 32 of them.
      auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };  // bits [0, n)
      RowMask mask = no_row();
      if (!full) mask = row_sees();
      auto seen = [&](int c) {
        const int at = kv0 + c;
        uint32_t bits = below(mask.last + 1 - at) & (~below(mask.first - at) | below(a.sinks - at));
        if (a.depth != nullptr) bits |= below(mask.own_last + 1 - at) & ~below(mask.own_first - at);
        return bits;
      };
      auto hide = [&](int c, float* x) {
        const uint32_t bits = seen(c);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(bits & (1u << e))) x[e] = -INFINITY;
      };
      // A row's maximum to `top` (in units of log2), O and l with it.
      auto raise = [&](float top) {
        top = fmaxf(top, m);
        const Keep keep(m - (top == -INFINITY ? 0.f : top));
        m = top;
        l = keep.l(l);
        if (done == 0) return;
        ok = warp_wait(bars->pv_done + stream, (done - 1) & 1, a.err, kErrTimeoutDone);
        if (!ok) return;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          float y[16];
          tmem_ld_16(t_o + c, y);
          tmem_wait_ld();
          uint32_t z[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) z[e] = __float_as_uint(y[e] * keep.o());
          tmem_st_16cols(t_o + c, z);
        }
      };
      if constexpr (!E4M3) {
        // One pass with the maximum as it is, a guess for a row that has seen no key yet; should it prove too small, or the
        // guess too large, it is put right and the pass repeated. So a row's largest weight is never below 1, and f16,
        // whose smallest step is 2^-24, holds the others to 2^-25 of it.
        uint32_t p[kTile / 2];
        while (true) {
          const bool fresh = m == -INFINITY;
          const float from = add - (fresh ? kGuess : m);
          const f32x2 scale2 = pair(by, by), from2 = pair(from, from);
          f32x2 sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
          float top = -INFINITY;
          float x[2][32];
          tmem_ld_32(t_s, x[0]);
#pragma unroll
          for (int c = 0; c < kTile; c += 32) {
            float(&y)[32] = x[(c / 32) & 1];
            tmem_wait_ld();
            if (c + 32 < kTile) tmem_ld_32(t_s + c + 32, x[(c / 32 + 1) & 1]);
            if (!full) hide(c, y);
            float tops[2] = {top, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              tops[0] = fmaxf(fmaxf(tops[0], y[e]), y[e + 1]);
              tops[1] = fmaxf(fmaxf(tops[1], y[e + 2]), y[e + 3]);
            }
            top = fmaxf(tops[0], tops[1]);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float lo, hi;
              unpair(fma2(pair(y[e], y[e + 1]), scale2, from2), lo, hi);
              lo = ex2(lo);
              hi = ex2(hi);
              sums[(e >> 1) & 1] = add2(pair(lo, hi), sums[(e >> 1) & 1]);
              p[(c + e) / 2] = pack2<M>(lo, hi);
            }
          }
          top = top == -INFINITY ? top : fmaf(top, by, add);
          const bool again = top > (fresh ? kGuess : m) + kLazy || (fresh && top < kGuess && top > -INFINITY);
          if (!__any_sync(0xffffffffu, again)) {
            float lo, hi;
            unpair(add2(sums[0], sums[1]), lo, hi);
            l = fmaf(lo + hi, inv_v, l);
            if (fresh && top > -INFINITY) m = kGuess;
            break;
          }
          raise(top);
          if (!ok) break;
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st_16cols(t_s + c * 16, p + c * 16);  // over scores that have been read
      } else {
        // Short loops, the tile's maximum first: beside the fetching warps' code the pass above, straight-line for all of
        // the tile, is fetched anew by every warp (2048 rows over 8048 keys: 274 us instead of 244; for 16-bit pages the
        // pass above is the faster one, 8191 windowed rows in 144 us instead of 156). The next 32 scores are on their
        // way while 32 are in work.
        float x0[32], x1[32];
        auto each = [&](auto&& work) {
          tmem_ld_32(t_s, x0);
#pragma unroll 1
          for (int c = 0; c < kTile; c += 64) {
            tmem_wait_ld();
            tmem_ld_32(t_s + c + 32, x1);
            if (!full) hide(c, x0);
            work(c, x0);
            tmem_wait_ld();
            if (c + 64 < kTile) tmem_ld_32(t_s + c + 64, x0);
            if (!full) hide(c + 32, x1);
            work(c + 32, x1);
          }
        };
        float top = -INFINITY, low = INFINITY;
        if (one) {
          each([&](int, const float(&x)[32]) {
            float tops[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y) tops[y] = fmaxf(fmaxf(tops[y], x[e + 2 * y]), x[e + 2 * y + 1]);
            top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          });
          if (top > -INFINITY) top = fmaf(top, by, add);
        } else {
          each([&](int c, const float(&x)[32]) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float y = fmaf(x[e] * by, scales.k[c + e], scales.log_v[c + e]);
              top = fmaxf(top, y);
              low = fminf(low, y == -INFINITY ? low : y);  // of the keys that the row sees
            }
          });
        }
        if (__any_sync(0xffffffffu, top > m + kLazy)) raise(one ? top - float(bars->one[slot] - 1) : top);
        if (!ok) break;
        const float from = m == -INFINITY ? 0.f : m;
        // With one scale it is the scores near the tile's largest that count, and their weights are floats unless that one
        // itself stays this far below the row's maximum.
        const bool apart = __any_sync(0xffffffffu, top > -INFINITY && top < m - 90.f);
        if (one && !apart) {
          const f32x2 scale2 = pair(by, by), from2 = pair(add - from, add - from);
          f32x2 sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
          each([&](int c, const float(&x)[32]) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float lo, hi;
              unpair(fma2(pair(x[e], x[e + 1]), scale2, from2), lo, hi);
              lo = ex2(lo);
              hi = ex2(hi);
              sums[(e >> 1) & 1] = add2(pair(lo, hi), sums[(e >> 1) & 1]);
              p[e / 2] = pack2<M>(lo, hi);
            }
            tmem_st_16cols(t_s + c / 2, p);  // over scores that have been read
          });
          float lo, hi;
          unpair(add2(sums[0], sums[1]), lo, hi);
          l = fmaf(lo + hi, inv_v, l);
        } else {
          const float by = fmaxf(q_scale, 1.17549435e-38f);  // the keys' scales come one by one
          if (__any_sync(0xffffffffu, one || low < m - 125.f)) {
#pragma unroll 1
            for (int c = 0; c < kTile; c += 8) {  // little code: it is seldom run
              float x[8];
              tmem_ld_8(t_s + c, x);
              tmem_wait_ld();
              const uint32_t bits = full ? 0xffu : seen(c);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float y = fmaf(x[e] * by, scales.k[c + e], scales.log_v[c + e]) - from;
                if ((bits & (1u << e)) && ex2(y) == 0.f) l += small_share(y, scales.log_v[c + e]);
              }
            }
          }
          each([&](int c, const float(&x)[32]) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float lo = ex2(fmaf(x[e] * by, scales.k[c + e], scales.log_v[c + e]) - from);
              const float hi = ex2(fmaf(x[e + 1] * by, scales.k[c + e + 1], scales.log_v[c + e + 1]) - from);
              l = fmaf(lo, scales.inv_v[c + e], l);
              l = fmaf(hi, scales.inv_v[c + e + 1], l);
              p[e / 2] = pack2<M>(lo, hi);
            }
            tmem_st_16cols(t_s + c / 2, p);
          });
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars->p_ready + stream);
      ++done;
    }
    if (ok && done > 0) warp_wait(bars->pv_done + stream, (done - 1) & 1, a.err, kErrTimeoutDone);
    tc_fence_after();
    named_barrier_sync(1, 2 * kRoleThreads);  // every product has run (or a wait has run out)

    // ---- results: with one row tile stream 1's part passes through shared memory
    constexpr int LD = HD + 4;  // floats between rows: rows meet different banks
    float* part1 = reinterpret_cast<float*>(smem);  // [128][LD], then (m, l), over queries and keys
    float* ml1 = part1 + kTile * LD;
    if (!u.turns.two && stream == 1) {
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float x[32];
        tmem_ld_32cols(t_o + c, x);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4*>(part1 + row * LD + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
      }
      ml1[2 * row] = m;
      ml1[2 * row + 1] = l;
    }
    named_barrier_sync(1, 2 * kRoleThreads);
    if (u.turns.two || stream == 0) {
      float keep0 = 1.f, keep1 = 0.f;
      if (!u.turns.two) {
        const float m1 = ml1[2 * row], top = fmaxf(m, m1), from = top == -INFINITY ? 0.f : top;
        const Keep mine(m - from), other(m1 - from);
        keep0 = mine.o();
        keep1 = other.o();
        m = top;
        l = mine.l(l) + other.l(ml1[2 * row + 1]);
      }
      const bool theirs = keep1 > 0.f;  // stream 1 may not have had a tile: then its memory means nothing
      const float inverse = l == 0.f ? 0.f : 1.f / l;
      // The stream's queries, whose place the output takes on its way, have been used. (Stream 1's part ends in front of
      // the values' ring, where a unit with one row tile goes.)
      uint8_t* const out_tile = u.turns.two ? q_tile : smem + S::V;
      float* part = nullptr;
      if (a.splits > 1) {
        float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + split_unit_bytes(gridDim.x / a.splits));
        part = parts + size_t(blockIdx.x) * part_floats<HD>();
        if (live) *reinterpret_cast<float2*>(part + kUnit * HD + 2 * (i - u.i0)) = make_float2(m, l);
        if (split == 0 && row == 0 && stream == 0)
          static_cast<SplitUnit*>(a.workspace)[index] = {u.r.start, u.i0, u.rows, u.head};
      }
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float x[32];
        tmem_ld_32cols(t_o + c, x);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = done > 0 ? x[e] * keep0 : 0.f;
        if (theirs) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = fmaf(part1[row * LD + c + e], keep1, x[e]);
        }
        if (live && bars->odd) {
          // non-finite values of the masked tiles, added to the rows that see them
          const RowMask mask = row_sees();
          const PageRows rows = {a.s.tables + u.seq * a.s.table_stride, a.c.page_shift, a.c.page_size - 1,
                                 a.c.num_pages, a.c.kv_heads, u.head, nullptr};
#pragma unroll 1
          for (int t = turns.t_begin; t < turns.t_end; ++t) {
            const int kv0 = u.keys.key<kTile>(t);
            if (u.keys.all_seen(kv0, kTile)) continue;
#pragma unroll 1
            for (int kv = kv0; kv < kv0 + kTile; ++kv) {
              const uint32_t at = mask.sees(kv, a.sinks) ? rows.row(u.keys, kv) : kNoRow;
              if (at == kNoRow) continue;
              const uint32_t* w = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.c.v) +
                                                                    (size_t(at) * HD + c) * (E4M3 ? 1 : 2));
              constexpr int PER = E4M3 ? 4 : 2;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (non_finite<T, E4M3>(w[e / PER], e % PER)) x[e] += element_f32<T, E4M3>(w[e / PER], e % PER);
            }
          }
        }
        if (live && a.splits > 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(part + size_t(i - u.i0) * HD + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        } else if (a.splits == 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4*>(out_tile + tile_at(row, (c + e) / 8)) =
                make_uint4(pack2<T>(x[e] * inverse, x[e + 1] * inverse), pack2<T>(x[e + 2] * inverse, x[e + 3] * inverse),
                           pack2<T>(x[e + 4] * inverse, x[e + 5] * inverse), pack2<T>(x[e + 6] * inverse, x[e + 7] * inverse));
        }
        __syncwarp();
      }
      if (a.splits == 1) {
        if (stream == 0) named_barrier_sync(3, kRoleThreads);
        else named_barrier_sync(4, kRoleThreads);
        Walk at = walk;
#pragma unroll 4
        for (int p = 0; p < QV; ++p, at.advance(a.group)) {
          if (at.packed < unit_rows)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (u.r.start + at.j) * a.out_stride +
                                      (u.head * a.group + at.g) * HD + row % QV * 8) =
                *reinterpret_cast<const uint4*>(out_tile + tile_at(row / QV + p * Walk::STEP, row % QV));
        }
      }
    }
    tc_fence_before();
    named_barrier_sync(1, 2 * kRoleThreads);
    if (warp == 0) {
      tc_fence_after();
      tmem_dealloc(tmem, kTmemColumns);
    }
  }
}

// Adds up the parts of a unit: blockIdx.x the unit, blockIdx.y 8 of its rows, a warp to a row.
template <int HD, typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const CacheAttnArgs a) {
  grid_dependency_wait();
  allow_dependents();
  const SplitUnit u = static_cast<const SplitUnit*>(a.workspace)[blockIdx.x];
  const int row = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (row >= u.rows) return;
  const float* parts =
      reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + split_unit_bytes(gridDim.x)) +
      size_t(blockIdx.x) * a.splits * part_floats<HD>();
  join_row<HD, T>(a, a.splits, [&](int i) { return parts + size_t(i) * part_floats<HD>(); }, row * HD, kUnit * HD + 2 * row,
                  u.row0, u.i0 + row, u.head);
}

// Units of a call, at most: a sequence has one more than its full ones.
int64_t prefill_units(const CacheAttnArgs& a) {
  const int64_t per_seq = (int64_t(a.s.max_rows) * a.group + kUnit - 1) / kUnit;
  return std::min<int64_t>(int64_t(a.s.rows) * a.group / kUnit + a.s.n_seqs, per_seq * a.s.n_seqs) * a.c.kv_heads;
}

// CTAs that share a unit's keys: as many as there are SMs for, with at least two key tiles each. It is one number for the
// call: beside a prompt of many units a single token's keys are one CTA's for each kv head, however many they are (2048 rows
// of 32 heads over 8, and one token at 32768 keys: e4m3 pages 84 us, 25 us, in one call 902; 16-bit 59, 32, 1470).
int prefill_splits(const CacheAttnArgs& a, int64_t max_keys, int num_sms) {
  const int64_t keys = a.window > 0 ? std::min<int64_t>(max_keys, int64_t(a.window) + a.sinks + kUnit) : max_keys;
  const int64_t tiles = (keys + kTile - 1) / kTile;
  return int(std::max<int64_t>(1, std::min<int64_t>(num_sms / prefill_units(a), tiles / 2)));
}

template <int HD, typename T, bool E4M3>
int launch_prefill(CacheAttnArgs a, int64_t max_keys, int num_sms, cudaStream_t stream) {
  auto kernel = prefill_attention_kernel<HD, T, E4M3>;
  constexpr int SMEM = PrefillSmem<HD>::BYTES;
  int st = raise_smem_limit(reinterpret_cast<const void*>(kernel), SMEM, "prefill_attention_kernel: shared memory");
  if (st != PLM_OK) return st;
  const int64_t units = prefill_units(a);
  a.splits = prefill_splits(a, max_keys, num_sms);
  if (units * a.splits >= (int64_t(1) << 31))
    return fail(PLM_ERR_UNSUPPORTED, "plm_cache_attention: %lld units of rows in one call", (long long)units);
  st = check_cuda(launch(kernel, dim3(unsigned(units * a.splits)), dim3(kPrefillThreads), SMEM, stream, true, a),
                  "prefill_attention_kernel");
  if (st != PLM_OK || a.splits == 1) return st;
  const int rows = int(std::min<int64_t>(kUnit, (int64_t(a.s.max_rows) * a.group + 7) / 8 * 8));
  return check_cuda(launch(join_parts_kernel<HD, T>, dim3(unsigned(units), rows / 8), dim3(256), 0, stream, true, a),
                    "join_parts_kernel");
}

}  // namespace

size_t prefill_workspace(const CacheAttnArgs& a, int head_dim, int64_t max_keys, int num_sms) {
  const int splits = prefill_splits(a, max_keys, num_sms);
  if (splits == 1) return 0;
  const int64_t units = prefill_units(a);
  return split_unit_bytes(units) + size_t(units) * splits * kUnit * (head_dim + 2) * sizeof(float);
}

int prefill_attention(const CacheAttnArgs& a, int kind, int dtype, int head_dim, int64_t max_keys, int num_sms,
                      cudaStream_t stream) {
  const bool e4m3 = kind == PLM_CACHE_E4M3;
  if (dtype == PLM_F16) {
    if (head_dim == 128)
      return e4m3 ? launch_prefill<128, __half, true>(a, max_keys, num_sms, stream)
                  : launch_prefill<128, __half, false>(a, max_keys, num_sms, stream);
    return e4m3 ? launch_prefill<64, __half, true>(a, max_keys, num_sms, stream)
                : launch_prefill<64, __half, false>(a, max_keys, num_sms, stream);
  }
  if (head_dim == 128)
    return e4m3 ? launch_prefill<128, __nv_bfloat16, true>(a, max_keys, num_sms, stream)
                : launch_prefill<128, __nv_bfloat16, false>(a, max_keys, num_sms, stream);
  return e4m3 ? launch_prefill<64, __nv_bfloat16, true>(a, max_keys, num_sms, stream)
              : launch_prefill<64, __nv_bfloat16, false>(a, max_keys, num_sms, stream);
}

}  // namespace plm
