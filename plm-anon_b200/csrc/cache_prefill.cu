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
// The issuing order P0 V, Q0 K', P1 V, Q1 K' lets one stream's two products (4 x 128 x 128 x d flops) run under the other
// one's softmax. Products of one thread execute in order, so S may be overwritten as soon as the product that reads P
// has been issued.
//
// Roles: warps 0-3 and 4-7 softmax of stream 0 and 1, warps 8-11 fetch keys, warps 12-15 values (16-bit pages by
// 16-byte asynchronous copies, e4m3 codes through registers, exactly to f16), warp 16 issues the products. Operands lie
// in 128-byte rows with the 128-byte swizzle, d = 128 in two panels. Every wait is bounded.
//
// Softmax: base 2, lazy maximum (O is rescaled only when a score passes m by more than 2^8), scales of e4m3 pages kept
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
constexpr int kPrefillThreads = 5 * kRoleThreads;
constexpr int kFactorSlots = 4;
constexpr uint32_t kTmemColumns = 512;

template <int HD>
struct PrefillSmem {
  static constexpr int TILE = kTile * HD * 2;  // a tile of 128 rows, keys or values
  static constexpr int Q = 0;
  static constexpr int K = 2 * TILE;
  static constexpr int V = 4 * TILE;
  static constexpr int FACTORS = 6 * TILE;     // [slot][k scale, log2 v scale, 1 / v scale][128]
  static constexpr int BARRIERS = FACTORS + kFactorSlots * 3 * kTile * 4;
  static constexpr int BYTES = BARRIERS + 256 + 1024;  // and the alignment's slack
};

struct PrefillBarriers {
  uint64_t q_ready, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], pv_done[2],
      factors_full[kFactorSlots];
  uint32_t tmem;
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
__device__ __forceinline__ void tmem_st_16cols(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32cols(uint32_t taddr, const float (&v)[32]) {
  uint32_t r[16];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[h * 16 + i]);
    tmem_st_16cols(taddr + h * 16, r);
  }
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void registers_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Byte offset of 16-byte vector `vec` of row `row` in a tile of 128 rows of d 16-bit elements.
__device__ __forceinline__ int tile_at(int row, int vec) {
  return (vec >> 3) * (kTile * 128) + row * 128 + (((vec & 7) ^ (row & 7)) << 4);
}

// What a CTA works on.
struct Unit {
  SeqRange r;
  int seq, head, i0, rows;    // packed rows [i0, i0 + rows)
  bool two;                   // row tiles
  TileKeys keys;              // of all its rows, in tiles of 128 keys
  TileKeys stream_keys[2];    // of a stream's rows
  int t_begin, t_end;         // this CTA's key tiles
  // Whether stream s works on key tile t: with two row tiles, unless none of its rows sees a key there.
  __device__ __forceinline__ bool active(int s, int t) const {
    if (!two) return ((t - t_begin) & 1) == s;
    const int kv = keys.key<kTile>(t);
    return kv < stream_keys[s].end && (kv + kTile > stream_keys[s].lo || kv < stream_keys[s].sinks);
  }
};

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
  u->two = u->rows > kTile;
  const int j0 = u->i0 / a.group, j1 = (u->i0 + u->rows - 1) / a.group;
  TileKeys t = causal_keys(a, u->r, j0, j1);
  if (a.depth != nullptr) {
    t.end = int(u->r.context) + u->r.n;
    t.lo = t.full_end = kUnreachable;
    t.full_lo = 0;
    for (int j = j0 + lane; j <= j1; j += 32) widen(t, row_mask(a, u->r, j));
    t.lo = __reduce_min_sync(0xffffffffu, t.lo);
    t.full_lo = __reduce_max_sync(0xffffffffu, t.full_lo);
    t.full_end = __reduce_min_sync(0xffffffffu, t.full_end);
    t.sinks = min(a.sinks, t.lo);
  }
  t.count<kTile>();
  u->keys = u->stream_keys[0] = u->stream_keys[1] = t;
  if (u->two && a.depth == nullptr) {
    u->stream_keys[0] = causal_keys(a, u->r, j0, (u->i0 + kTile - 1) / a.group);
    u->stream_keys[1] = causal_keys(a, u->r, (u->i0 + kTile) / a.group, j1);
  }
  u->t_begin = int(int64_t(split) * t.chunks / a.splits);
  u->t_end = int(int64_t(split + 1) * t.chunks / a.splits);
  return true;
}

// Places of keys in the pages.
struct PageRows {
  const int32_t* table;
  int page_shift, page_mask, num_pages, kv_heads, head, page_size;
  int* err;
  // Key kv's row within a plane, in rows of d elements, or -1 where there is none to fetch.
  __device__ __forceinline__ int64_t row(const TileKeys& t, int kv) const {
    if (!t.needed(kv)) return -1;
    const int page = table[kv >> page_shift];
    if (unsigned(page) >= unsigned(num_pages)) {
      record_error(err, kErrBadIndex);
      return -1;
    }
    return (int64_t(page) * kv_heads + head) * page_size + (kv & page_mask);
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

// Fetches all key tiles (VALUES false) or value tiles of the CTA into its ring of two: 128 threads.
template <int HD, typename T, bool E4M3, bool VALUES>
__device__ __forceinline__ void fetch_tiles(const CacheAttnArgs& a, const Unit& u, uint8_t* smem, PrefillBarriers* bars) {
  using S = PrefillSmem<HD>;
  const int tid = threadIdx.x & (kRoleThreads - 1), lane = tid & 31;
  uint64_t* full = VALUES ? bars->v_full : bars->k_full;
  uint64_t* empty = VALUES ? bars->v_empty : bars->k_empty;
  uint8_t* ring = smem + (VALUES ? S::V : S::K);
  const uint8_t* plane = static_cast<const uint8_t*>(VALUES ? a.c.v : a.c.k);
  constexpr int ES = E4M3 ? 1 : 2;
  constexpr int VECS = HD * ES / 16;            // 16-byte vectors of a row in the page
  constexpr int PER_PASS = kRoleThreads / VECS; // rows that the threads fetch together
  constexpr int PASSES = kTile / PER_PASS;
  const int vec = tid % VECS, first = tid / VECS;
  const PageRows rows = {a.s.tables + u.seq * a.s.table_stride, a.c.page_shift, a.c.page_size - 1,
                                   a.c.num_pages, a.c.kv_heads, u.head, a.c.page_size, a.err};
  float* factors = reinterpret_cast<float*>(smem + S::FACTORS);
  auto arrive = [&](uint64_t* bar) {
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  // Values of a masked tile that are no numbers: 16-bit ones are looked for where they have landed.
  auto landed = [&](int n) {
    const int t = u.t_begin + n;
    if constexpr (VALUES && !E4M3) {
      if (!u.keys.all_seen(u.keys.key<kTile>(t), kTile)) {
#pragma unroll 1
        for (int p = 0; p < PASSES; ++p) {
          uint4* x = reinterpret_cast<uint4*>(ring + (n & 1) * S::TILE + tile_at(first + p * PER_PASS, vec));
          if (any_non_finite<T, false>(*x)) {
            drop_non_finite<T, false>(*x);
            bars->odd = 1;
          }
        }
      }
    }
    arrive(full + (n & 1));
  };
  const int tiles = u.t_end - u.t_begin;
  for (int n = 0; n < tiles; ++n) {
    const int kv0 = u.keys.key<kTile>(u.t_begin + n);
    if constexpr (!E4M3) {
      if (n >= 2 && !warp_wait(empty + (n & 1), ((n >> 1) - 1) & 1, a.err, kErrTimeoutEmpty)) break;
      uint8_t* dst = ring + (n & 1) * S::TILE;
#pragma unroll 4
      for (int p = 0; p < PASSES; ++p) {
        const int row = first + p * PER_PASS;
        const int64_t at = rows.row(u.keys, kv0 + row);
        cp_async_16(dst + tile_at(row, vec), plane + (at < 0 ? 0 : size_t(at) * (HD * ES) + vec * 16), at >= 0);
      }
      cp_async_commit();
      if (n > 0) {
        cp_async_wait<1>();
        landed(n - 1);
      }
    } else {
      uint4 codes[PASSES];
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int64_t at = rows.row(u.keys, kv0 + first + p * PER_PASS);
        codes[p] = make_uint4(0, 0, 0, 0);
        if (at >= 0) codes[p] = *reinterpret_cast<const uint4*>(plane + size_t(at) * HD + vec * 16);
      }
      float ks = 0.f, vs = 1.f;  // the scales of key tid
      if constexpr (!VALUES) {
        const int64_t at = rows.row(u.keys, kv0 + tid);
        if (at >= 0) {
          const int64_t block = (at >> a.c.page_shift) * (a.c.page_size >> a.c.block_shift) +
                                ((at & (a.c.page_size - 1)) >> a.c.block_shift);
          ks = a.c.k_scale[block];
          vs = fmaxf(a.c.v_scale[block], kLeastScale);
        }
      }
      if (n >= 2 && !warp_wait(empty + (n & 1), ((n >> 1) - 1) & 1, a.err, kErrTimeoutEmpty)) break;
      if constexpr (!VALUES) {
        // Their slot's last readers, the softmax of tile n - 4, are done: the products Q K of tiles n - 3 and n - 2 have
        // run, and a stream's products start only when its softmax of the tile before is over.
        float* f = factors + (n % kFactorSlots) * 3 * kTile;
        f[tid] = ks;
        f[kTile + tid] = lg2(vs);
        f[2 * kTile + tid] = rcp(vs);
        __syncwarp();
        if (lane == 0) mbar_arrive(bars->factors_full + n % kFactorSlots);
      }
      uint8_t* dst = ring + (n & 1) * S::TILE;
      const bool look = VALUES && !u.keys.all_seen(kv0, kTile);
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        if (look && any_non_finite<T, true>(codes[p])) {
          drop_non_finite<T, true>(codes[p]);
          bars->odd = 1;
        }
        const uint32_t w[4] = {codes[p].x, codes[p].y, codes[p].z, codes[p].w};
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[2 * i] = e4m3x2_to_f16x2(uint16_t(w[i]));
          h[2 * i + 1] = e4m3x2_to_f16x2(uint16_t(w[i] >> 16));
        }
        const int row = first + p * PER_PASS;
        *reinterpret_cast<uint4*>(dst + tile_at(row, 2 * vec)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + tile_at(row, 2 * vec + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      arrive(full + (n & 1));
    }
  }
  if constexpr (!E4M3) {
    cp_async_wait<0>();
    if (tiles > 0) landed(tiles - 1);
  }
}

// Issues all products: one warp, its first lane.
template <int HD, bool BF16>
__device__ __forceinline__ void issue_products(const CacheAttnArgs& a, const Unit& u, uint8_t* smem, PrefillBarriers* bars) {
  using S = PrefillSmem<HD>;
  constexpr uint32_t QK = umma_idesc_f16(kTile, kTile, BF16);
  constexpr uint32_t PV = umma_idesc_f16(kTile, HD, BF16) | (1u << 16);  // B transposed
  constexpr int PANEL = kTile * 128;
  const int lane = threadIdx.x & 31;
  const uint32_t tmem = bars->tmem;
  const uint32_t q_addr = smem_u32(smem + S::Q), k_addr = smem_u32(smem + S::K), v_addr = smem_u32(smem + S::V);
  const int tiles = u.t_end - u.t_begin;
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (!ok) return;
    int got = 1;
    if (lane == 0) got = mbar_wait(bar, parity, a.err, code) ? 1 : 0;
    ok = __shfl_sync(0xffffffffu, got, 0) != 0;
  };
  auto users = [&](int n) { return (u.active(0, u.t_begin + n) ? 1 : 0) + (u.active(1, u.t_begin + n) ? 1 : 0); };
  auto after = [&](int s, int n) {  // the stream's next tile from n on
    while (n < tiles && !u.active(s, u.t_begin + n)) ++n;
    return n;
  };
  auto scores = [&](int s, int n) {
    wait(bars->k_full + (n & 1), (n >> 1) & 1, kErrTimeoutFull);
    if (!ok) return;
    tc_fence_after();
    if (lane == 0) {
      const uint32_t q = q_addr + (u.two ? s : 0) * S::TILE, k = k_addr + (n & 1) * S::TILE;
#pragma unroll
      for (int x = 0; x < HD / 16; ++x) {
        const uint32_t at = (x >> 2) * PANEL + (x & 3) * 32;
        umma_f16(tmem + s * kTile, umma_desc_sw128(q + at), umma_desc_sw128(k + at), QK, x > 0 ? 1u : 0u);
      }
      umma_commit(bars->s_full + s);
      umma_commit(bars->k_empty + (n & 1));
      if (users(n) == 1) umma_commit(bars->k_empty + (n & 1));  // the other stream has no use for it
    }
    __syncwarp();
  };
  auto values = [&](int s, int n, int count) {
    wait(bars->v_full + (n & 1), (n >> 1) & 1, kErrTimeoutFull);
    wait(bars->p_ready + s, count & 1, kErrTimeoutPeer);
    if (!ok) return;
    tc_fence_after();
    if (lane == 0) {
      const uint32_t v = v_addr + (n & 1) * S::TILE;
#pragma unroll
      for (int x = 0; x < kTile / 16; ++x)
        umma_f16_ts(tmem + 2 * kTile + s * kTile, tmem + s * kTile + x * 8, umma_desc_transposed(v + x * 2048, PANEL), PV,
                    count > 0 || x > 0 ? 1u : 0u);
      umma_commit(bars->pv_done + s);
      umma_commit(bars->v_empty + (n & 1));
      if (users(n) == 1) umma_commit(bars->v_empty + (n & 1));
    }
    __syncwarp();
  };
  wait(&bars->q_ready, 0, kErrTimeoutPeer);
  int at[2] = {after(0, 0), after(1, 0)}, count = 0;
#pragma unroll
  for (int s = 0; s < 2; ++s)
    if (at[s] < tiles) scores(s, at[s]);
  while (ok && (at[0] < tiles || at[1] < tiles)) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (at[s] >= tiles) continue;
      const int next = after(s, at[s] + 1);
      values(s, at[s], count);
      if (next < tiles) scores(s, next);
      at[s] = next;
    }
    ++count;
  }
}

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
  Unit u;
  if (!find_unit(a, index / a.c.kv_heads, index % a.c.kv_heads, split, &u)) {
    if (a.splits > 1 && split == 0 && tid == 0) static_cast<SplitUnit*>(a.workspace)[index].rows = 0;
    return;
  }
  if (tid == 0) {
    mbar_init(&bars->q_ready, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars->k_full + i, 4);
      mbar_init(bars->k_empty + i, 2);
      mbar_init(bars->v_full + i, 4);
      mbar_init(bars->v_empty + i, 2);
      mbar_init(bars->s_full + i, 1);
      mbar_init(bars->p_ready + i, 4);
      mbar_init(bars->pv_done + i, 1);
    }
    for (int i = 0; i < kFactorSlots; ++i) mbar_init(bars->factors_full + i, 4);
    bars->odd = 0;
    fence_barrier_init();
  }
  if (warp == 0) tmem_alloc(&bars->tmem, kTmemColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  // Registers: 96 a thread at launch, 5 x 96 = 480 for the five groups of four warps: 2 x 160 + 2 x 56 + 48 = 480.
  const int role = tid / kRoleThreads;
  if (role == 2) {
    registers_dec<56>();
    fetch_tiles<HD, T, E4M3, false>(a, u, smem, bars);
  } else if (role == 3) {
    registers_dec<56>();
    fetch_tiles<HD, T, E4M3, true>(a, u, smem, bars);
  } else if (role == 4) {
    registers_dec<48>();
    if (warp == 16) issue_products<HD, std::is_same<M, __nv_bfloat16>::value>(a, u, smem, bars);
  } else {
    registers_inc<160>();
    const int stream = role;
    float m = -INFINITY, l = 0.f;
    int done = 0;  // key tiles this stream has worked on
    bool ok = true;
    const uint32_t t_lane = tmem + (uint32_t((warp & 3) * 32) << 16);
    const int row = tid & (kRoleThreads - 1);                       // of the stream's tile
    const int i = u.i0 + (u.two && stream == 1 ? kTile : 0) + row;  // packed row
    const bool live = i < u.i0 + u.rows;
    // ---- the row's query into shared memory (with one row tile, stream 0's threads bring it)
    float q_scale = a.scale_log2;
    const T* src = static_cast<const T*>(a.q) + (u.r.start + (live ? i : u.i0) / a.group) * a.q_stride +
                   (u.head * a.group + (live ? i : u.i0) % a.group) * HD;
    float up = 1.f;
    if constexpr (E4M3 && std::is_same<T, __nv_bfloat16>::value) {
      uint32_t top = 0;
#pragma unroll 4
      for (int vec = 0; vec < HD / 8; ++vec) {
        const uint4 x = live ? reinterpret_cast<const uint4*>(src)[vec] : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
      }
      const int e = query_exponent(top);
      up = power_of_two_f32(-e);
      q_scale *= power_of_two_f32(e);
    }
    if (u.two || stream == 0) {
      uint8_t* dst = smem + S::Q + stream * S::TILE;
#pragma unroll 4
      for (int vec = 0; vec < HD / 8; ++vec) {
        uint4 x = live ? reinterpret_cast<const uint4*>(src)[vec] : make_uint4(0, 0, 0, 0);
        if constexpr (E4M3 && std::is_same<T, __nv_bfloat16>::value) {
          uint32_t* w = &x.x;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pack2<__half>(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
        }
        *reinterpret_cast<uint4*>(dst + tile_at(row, vec)) = x;
      }
    }
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->q_ready);
    const RowMask mask = live ? row_mask(a, u.r, i / a.group) : no_row();
    const TileKeys& keys = u.stream_keys[stream];
    const float* factors = reinterpret_cast<const float*>(smem + S::FACTORS);
    const uint32_t t_s = t_lane + stream * kTile, t_o = t_lane + 2 * kTile + stream * kTile;

    for (int n = 0; n < u.t_end - u.t_begin; ++n) {
      if (!u.active(stream, u.t_begin + n)) continue;
      const int kv0 = u.keys.key<kTile>(u.t_begin + n);
      const bool full = keys.all_seen(kv0, kTile);
      const float* f = factors + (n % kFactorSlots) * 3 * kTile;
      ok = (!E4M3 || warp_wait(bars->factors_full + n % kFactorSlots, (n / kFactorSlots) & 1, a.err, kErrTimeoutFull)) &&
           warp_wait(bars->s_full + stream, done & 1, a.err, kErrTimeoutDone);
      if (!ok) break;
      tc_fence_after();
      // Scores of 32 keys in units of log2.
      auto load_scores = [&](int c, float(&x)[32]) {
        tmem_ld_32cols(t_s + c, x);
        if constexpr (E4M3) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 ks = *reinterpret_cast<const float4*>(f + c + e);
            const float4 lv = *reinterpret_cast<const float4*>(f + kTile + c + e);
            x[e] = fmaf(x[e] * q_scale, ks.x, lv.x);
            x[e + 1] = fmaf(x[e + 1] * q_scale, ks.y, lv.y);
            x[e + 2] = fmaf(x[e + 2] * q_scale, ks.z, lv.z);
            x[e + 3] = fmaf(x[e + 3] * q_scale, ks.w, lv.w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] *= q_scale;
        }
        if (!full) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!mask.sees(kv0 + c + e, a.sinks)) x[e] = -INFINITY;
        }
      };
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
        float x[32];
        load_scores(c, x);
#pragma unroll
        for (int e = 0; e < 32; ++e) top = fmaxf(top, x[e]);
      }
      if (__any_sync(0xffffffffu, top > m + kLazy)) {
        top = fmaxf(top, m);
        const float keep = ex2(m - (top == -INFINITY ? 0.f : top));
        m = top;
        l *= keep;
        if (done > 0) {
          ok = warp_wait(bars->pv_done + stream, (done - 1) & 1, a.err, kErrTimeoutDone);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            float x[32];
            tmem_ld_32cols(t_o + c, x);
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] *= keep;
            tmem_st_32cols(t_o + c, x);
          }
        }
      }
      const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
        float x[32];
        load_scores(c, x);
        uint32_t p[16];
        if constexpr (E4M3) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 iv = *reinterpret_cast<const float4*>(f + 2 * kTile + c + e);
            x[e] = ex2(x[e] - from);
            x[e + 1] = ex2(x[e + 1] - from);
            x[e + 2] = ex2(x[e + 2] - from);
            x[e + 3] = ex2(x[e + 3] - from);
            l = fmaf(x[e], iv.x, l);
            l = fmaf(x[e + 1], iv.y, l);
            l = fmaf(x[e + 2], iv.z, l);
            l = fmaf(x[e + 3], iv.w, l);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            x[e] = ex2(x[e] - from);
            l += x[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = pack2<M>(x[2 * e], x[2 * e + 1]);
        tmem_st_16cols(t_s + c / 2, p);  // over scores that have been read
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
    if (!u.two && stream == 1) {
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
    if (u.two || stream == 0) {
      float keep0 = 1.f, keep1 = 0.f;
      if (!u.two) {
        const float m1 = ml1[2 * row], top = fmaxf(m, m1), from = top == -INFINITY ? 0.f : top;
        keep0 = ex2(m - from);
        keep1 = ex2(m1 - from);
        m = top;
        l = l * keep0 + ml1[2 * row + 1] * keep1;
      }
      const bool theirs = keep1 > 0.f;  // stream 1 may not have had a tile: then its memory means nothing
      const float inverse = l == 0.f ? 0.f : 1.f / l;
      T* dst = static_cast<T*>(a.out) + (u.r.start + (live ? i : u.i0) / a.group) * a.out_stride +
               (u.head * a.group + (live ? i : u.i0) % a.group) * HD;
      float* part = nullptr;
      if (a.splits > 1) {
        float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + split_unit_bytes(gridDim.x / a.splits));
        part = parts + size_t(blockIdx.x) * part_floats<HD>();
        if (live) *reinterpret_cast<float2*>(part + kUnit * HD + 2 * (i - u.i0)) = make_float2(m, l);
        if (split == 0 && tid == 0)
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
          const PageRows rows = {a.s.tables + u.seq * a.s.table_stride, a.c.page_shift, a.c.page_size - 1,
                                 a.c.num_pages, a.c.kv_heads, u.head, a.c.page_size, nullptr};
#pragma unroll 1
          for (int t = u.t_begin; t < u.t_end; ++t) {
            const int kv0 = u.keys.key<kTile>(t);
            if (u.keys.all_seen(kv0, kTile)) continue;
#pragma unroll 1
            for (int kv = kv0; kv < kv0 + kTile; ++kv) {
              const int64_t at = mask.sees(kv, a.sinks) ? rows.row(u.keys, kv) : -1;
              if (at < 0) continue;
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
        } else if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4*>(dst + c + e) =
                make_uint4(pack2<T>(x[e] * inverse, x[e + 1] * inverse), pack2<T>(x[e + 2] * inverse, x[e + 3] * inverse),
                           pack2<T>(x[e + 4] * inverse, x[e + 5] * inverse), pack2<T>(x[e + 6] * inverse, x[e + 7] * inverse));
        }
        __syncwarp();
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

// Adds up the parts of a unit in order: blockIdx.x the unit, blockIdx.y 32 of its rows.
template <int HD, typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const CacheAttnArgs a) {
  grid_dependency_wait();
  allow_dependents();
  const SplitUnit u = static_cast<const SplitUnit*>(a.workspace)[blockIdx.x];
  const float* parts =
      reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + split_unit_bytes(gridDim.x)) +
      size_t(blockIdx.x) * a.splits * part_floats<HD>();
  constexpr int Q4 = HD / 4;
  const int row_end = min(u.rows, int(blockIdx.y + 1) * 32);
  for (int item = blockIdx.y * 32 * Q4 + threadIdx.x; item < row_end * Q4; item += 256) {
    const int row = item / Q4, d = (item % Q4) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, total = 0.f;
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) {
      const float* part = parts + size_t(i) * part_floats<HD>();
      const float2 ml = *reinterpret_cast<const float2*>(part + kUnit * HD + 2 * row);
      const float4 x = *reinterpret_cast<const float4*>(part + size_t(row) * HD + d);
      const float now = fmaxf(top, ml.x), from = now == -INFINITY ? 0.f : now;
      const float keep = ex2(top - from), f = ex2(ml.x - from);
      top = now;
      sum.x = sum.x * keep + f * x.x;
      sum.y = sum.y * keep + f * x.y;
      sum.z = sum.z * keep + f * x.z;
      sum.w = sum.w * keep + f * x.w;
      total = total * keep + f * ml.y;
    }
    store_row4<T>(a, u.row0, u.i0 + row, u.head, HD, d, sum, total);
  }
}

// Units of a call, at most: a sequence has one more than its full ones.
int64_t prefill_units(const CacheAttnArgs& a) {
  const int64_t per_seq = (int64_t(a.s.max_rows) * a.group + kUnit - 1) / kUnit;
  return std::min<int64_t>(int64_t(a.s.rows) * a.group / kUnit + a.s.n_seqs, per_seq * a.s.n_seqs) * a.c.kv_heads;
}

// CTAs that share a unit's keys: as many as there are SMs for, with at least two key tiles each.
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
  return check_cuda(launch(join_parts_kernel<HD, T>, dim3(unsigned(units), kUnit / 32), dim3(256), 0, stream, true, a),
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
