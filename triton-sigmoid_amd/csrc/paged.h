// Paged key/value cache: parameters, work units and tile copies of the kernels
// that read it.
#pragma once

#include "common.h"

namespace sigattn {

// Attention over a paged cache.  The base's q, out, k, v, score_mod, cu_q,
// rows_q, sq_*, sk_t, sk_h, B, H, Tq (longest query sequence), Tk (tokens a
// block-table row can hold) and dmem mean what they do there; H counts query
// heads, and `out` is contiguous [rows_q, H, dmem].
//
// A kernel's work unit is (sequence, block of query columns, K / V head, chunk
// of the keys); the columns of a sequence are its tokens times the G query
// heads of a K / V head, column c = token c / G of head c % G.  A kernel takes
// the sequences of more than cols_lo and at most cols_hi columns.  split_units
// > 0: sequences are cut into chunks of at least min_chunk keys, total_units
// (split_units more than the uncut batch can have) at most; a unit of a cut sequence leaves its fp32 sums in
// `ws`, and cut[b] where they begin, for the reduction.
struct PagedParams : KParams {
  static constexpr bool kPaged = true;
  const int32_t *table;  // [B, max_pages], row stride table_stride
  const int32_t *lens;   // [B] keys
  int64_t table_stride, mod_stride, sk_p;
  int Hkv, G;            // K / V heads, query heads of each
  int lp, num_pages;     // log2 of the page size
  float fscale, fbias;
  int own_bias;          // 0: the bias is -log(keys)
  int cols_lo, cols_hi;
  int split_units, total_units, min_chunk;
  int max_units;         // units that `ws` has room for
  int2 *cut;             // [B] (first unit / Hkv, chunks)

  __device__ __forceinline__ int keys(int b) const { return clamp_len(lens, b, Tk); }
  __device__ __forceinline__ float bias_of(int Lk) const { return own_bias ? fbias : -logf((float)Lk); }
  // Blocks of `block` columns that this kernel runs of a sequence of n tokens.
  __device__ __forceinline__ int blocks_of(int n, int block) const {
    const int cols = n * G;
    return cols > cols_lo && cols <= cols_hi ? (cols + block - 1) / block : 0;
  }
};

// Most chunks of a sequence: the reduction reads them all.  320 / 384 / 448, whole
// call, us, bf16 B=1 H=16 Hkv=2 D=128: 32000 keys 18.9 / 16.8 / 16.8, 65535 21.9 /
// 21.3 / 21.9 (512: 22.1), 131072 31.7 / 31.0 / 31.1.
constexpr int kMostChunks = 384;

// The chunk length that gives every unit `keys` keys, `least` at least: one more,
// and 2^30 + 1 at most.  A sequence has fewer than 2^30 keys, so a chunk of that
// many never cuts it, and a length and a chunk together fit 31 bits.
constexpr int kNoCut = 1 << 30;
__host__ __device__ inline int chunk_for(float keys, int least) {
  const int n = (int)(keys < (float)kNoCut ? keys : (float)kNoCut) + 1;
  return n > least ? n : least;
}

// Columns of a decoding unit: sequences of up to this many (new tokens times the
// query heads of a K / V head) are the decoding kernels', longer ones the blocks'.
// The matrix instructions' 32 columns; no block of columns is as small.
constexpr int kDecodeCols = 32;

struct PagedUnit {
  int b = 0, hk = 0, qb = 0;  // sequence, K / V head, column block
  int Lq = 0, Lk = 0;         // its tokens and keys
  int k0 = 0, k1 = 0;         // keys of the chunk
  int nck = 0;                // chunks of the sequence (0: no such unit)
};

// Inclusive sums over the lanes of the wave, by data-parallel-primitive adds (a
// few cycles each, where a shuffle through LDS takes about a hundred): within
// rows of 16 lanes, then rows 1 and 3 take row 0's and 2's total, then the upper
// half the lower's.  Lane 63 has the sum.
template <typename N> __device__ __forceinline__ N wave_scan(N x) {
  const auto step = [&](auto ctrl, auto rows) SIGATTN_INLINE {
    const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                  decltype(rows)::value, 0xf, false);
    x += __builtin_bit_cast(N, moved);
  };
  step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_scan(x)), 63));
}

// Unit u of the kernel with column blocks of `block`, from the lengths on the
// device (no host synchronisation): sequences in order, their blocks last
// (under the causal mask longest) first, chunks, K / V heads fastest.  Every wave computes it
// alike, 64 sequences at a time.  Chunks: with work W = sum of blocks times
// keys, C = W Hkv / split_units keys (min_chunk at least), ceil(keys / C) chunks at
// most, of equal length: no more than split_units + the units of an uncut batch.  Batches
// of up to 64 sequences take a shorter C where that many units allow it.
__device__ __forceinline__ PagedUnit paged_unit(const PagedParams &p, int u, int block) {
  const int lane = __lane_id();
  if (block == kDecodeCols && p.split_units == 0) {
    // Decoding, nothing cut: a unit is a sequence's K / V head.
    PagedUnit un;
    un.b = u / p.Hkv, un.hk = u - un.b * p.Hkv;
    if (un.b >= p.B) return un;
    un.Lq = p.len_q(un.b), un.Lk = un.k1 = p.keys(un.b);
    un.nck = p.blocks_of(un.Lq, block);
    for (int *x : {&un.b, &un.hk, &un.Lq, &un.Lk, &un.k1, &un.nck}) *x = __builtin_amdgcn_readfirstlane(*x);
    return un;
  }
  // The first 64 * kKeep sequences' lengths stay in registers, their loads in
  // flight together.
  constexpr int kKeep = 4;
  int tokens[kKeep], keys[kKeep];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int b = lane + 64 * i;
    tokens[i] = b < p.B ? p.len_q(b) : 0, keys[i] = b < p.B ? p.keys(b) : 0;
  }
  int C = kNoCut;
  if (p.split_units > 0) {
    const int nqb0 = p.blocks_of(tokens[0], block), Lk0 = keys[0];
    float work = 0.0f;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) work += (float)p.blocks_of(tokens[i], block) * (float)keys[i];
    for (int b = lane + 64 * kKeep; b < p.B; b += 64)
      work += (float)p.blocks_of(p.len_q(b), block) * (float)p.keys(b);
    work = wave_sum(work) * (float)p.Hkv;
    const float c = work / (float)p.split_units;
    C = chunk_for(c, p.min_chunk);
    if (p.B <= 64 && p.Tk < 1 << 23) {  // (where the quotients below are exact enough)
      // The smallest of 64 lengths, one a lane, that gives no more units than
      // fit: from the work's share of all of them up to C, which does.
      const float least = work / (float)p.total_units;
      const int mine = lane == 63 ? C : chunk_for(least + (c - least) * lane / 63.0f, p.min_chunk);
      int rows = 0;
      for (int b = 0; b < p.B; ++b) {
        const int n = __builtin_amdgcn_readlane(nqb0, b), L = __builtin_amdgcn_readlane(Lk0, b);
        rows += n * max((int)ceilf((float)L / (float)mine), 1);
      }
      const uint64_t fits = __ballot(rows * (int64_t)p.Hkv <= p.total_units) | (1ull << 63);
      C = __builtin_amdgcn_readlane(mine, __builtin_ctzll(fits));
    }
    C = __builtin_amdgcn_readfirstlane(C);
  }
  PagedUnit un;
  const int row = u / p.Hkv;
  un.hk = u - row * p.Hkv;
  int base = 0;
  // Whether the unit is one of the 64 sequences' from b0 on (then `un` has it).
  const auto among = [&](int b0, int Lq, int Lk) SIGATTN_INLINE {
    const int nqb = p.blocks_of(Lq, block), most = min(max((Lk + C - 1) / C, 1), kMostChunks);
    // Equal chunks of a multiple of `round` keys, as few as that takes.  Quotients
    // in floats, corrected, where lengths are exact in them (0.5 to 1 us a call
    // faster than by integer division).
    const int round = block == kDecodeCols ? 32 : 64;
    int len, nck;
    if (p.Tk < 1 << 23) {
      len = round * max((int)((float)Lk * __builtin_amdgcn_rcpf((float)(most * round))), 1);
      if (len * most < Lk) len += round;
      if (len * most < Lk) len += round;
      nck = max((int)((float)Lk * __builtin_amdgcn_rcpf((float)len)), 1);
      if (nck * len < Lk) ++nck;
    } else {
      len = max(((Lk + most - 1) / most + round - 1) & -round, round);
      nck = max((Lk + len - 1) / len, 1);
    }
    const int sum = wave_scan(nqb * nck), first = base + sum - nqb * nck;
    const uint64_t m = __ballot(row >= first && row < base + sum);
    base += __builtin_amdgcn_readlane(sum, 63);
    if (m == 0) return false;
    const int at = __builtin_ctzll(m);
    un.b = b0 + at;
    un.Lq = __builtin_amdgcn_readlane(Lq, at), un.Lk = __builtin_amdgcn_readlane(Lk, at);
    un.nck = __builtin_amdgcn_readlane(nck, at);
    const int r = row - __builtin_amdgcn_readlane(first, at), q = r / un.nck, chunk = r - q * un.nck;
    un.qb = __builtin_amdgcn_readlane(nqb, at) - 1 - q;
    const int size = __builtin_amdgcn_readlane(len, at);
    un.k0 = chunk * size, un.k1 = min(un.k0 + size, un.Lk);
    if (p.split_units > 0 && r == 0 && un.hk == 0 && lane == at) p.cut[un.b] = make_int2(first, nck);
    return true;
  };
  bool found = false;
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (!found && 64 * i < p.B) found = among(64 * i, tokens[i], keys[i]);
  for (int b0 = 64 * kKeep; !found && b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    found = among(b0, b < p.B ? p.len_q(b) : 0, b < p.B ? p.keys(b) : 0);
  }
  // Wave-uniform as they are; the compiler is told so (scalar addresses).
  for (int *x : {&un.b, &un.hk, &un.qb, &un.Lq, &un.Lk, &un.k0, &un.k1, &un.nck})
    *x = __builtin_amdgcn_readfirstlane(*x);
  return un;
}

// fp32 sums of unit u: [block columns][D] at u * block * D floats of ws.
// (a: column block's 16-row accumulators; col: this lane's column of the
// sequence, cc: of the unit; further column blocks 32 columns on.)
template <typename T, int D, int NCB, class Acc>
__device__ __forceinline__ void paged_store(const PagedParams &p, const PagedUnit &un, const Acc &acc, int col, int cc,
                                            int block, int unit, int hi, bool half) {
  constexpr int NDB = D / 32;
  const int d = half ? 16 : D;
  const int64_t row0 = packed_first(p.cu_q, p.rows_q, un.b);
#pragma unroll
  for (int c = 0; c < NCB; ++c) {
    const int q = col + 32 * c;
    if (q >= un.Lq * p.G) continue;
    const int tok = q / p.G;
    uint16_t *orow = (uint16_t *)p.out + ((row0 + tok) * p.H + un.hk * p.G + q - tok * p.G) * d;
    float *part = p.ws + ((int64_t)unit * block + cc + 32 * c) * D;
    const auto store = [&](auto &&put) SIGATTN_INLINE {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (half && g >= 2) break;  // columns 16..31: not in the tensor
          const f32x16 &a = acc[c][db];
          put(db * 32 + 8 * g + 4 * hi, (f32x4){a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]});
        }
    };
    if (un.nck == 1)
      store([&](int d0, f32x4 v) SIGATTN_INLINE {
        *(u32x2 *)(orow + d0) = (u32x2){Elem<T>::pack(v.x, v.y), Elem<T>::pack(v.z, v.w)};
      });
    else
      store([&](int d0, f32x4 v) SIGATTN_INLINE { *(f32x4 *)(part + d0) = v; });
  }
}

// A 16-byte source of zeros.
static __device__ const uint32_t kZeroPiece[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

// DmaPlan for tiles of a paged cache: ROWS keys from a key that is a multiple
// of 16, copied by NWAVES waves, each a run of rows that begins at a multiple of
// its length.  Pages hold a power of two of rows, 16 at least, so 16 rows of a
// tile lie on one page: their table entry is a scalar load (made one tile
// ahead of its use) and the page's address scalar arithmetic in 64 bits; the
// lanes keep 32-bit offsets within 16 rows.  Rows past the chunk and rows on a
// page outside the cache come from kZeroPiece: every instruction still issues,
// so counted waits hold.  NT: non-temporal loads, for rows that are read once.
// fp32 rows of D / 2 elements (ESIZE = 4) are the same bytes.
template <int ROWS, int D, int NWAVES, bool NT = false, int ESIZE = 2> struct PagedDma {
  static constexpr int CPR = D / 8, RPI = 64 / CPR;
  static constexpr int RPW = ROWS / NWAVES, NI = RPW / RPI;  // rows, instructions per wave
  static constexpr int NE = RPW > 16 ? RPW / 16 : 1;         // table entries per wave and tile
  static_assert(NI >= 1 && RPW % RPI == 0 && (RPW <= 16 ? 16 % RPW == 0 : RPW % 16 == 0), "tile shape");
  typedef const __attribute__((address_space(4))) int32_t *ScalarInts;

  uint32_t voff[NI];  // byte offset of this lane's piece from the wave's first row of 16
  uint32_t cbyte[NI];
  ScalarInts row;     // the sequence's table row
  int ent[NE];        // pages of the next tile
  int key0, keys, r0, lrow, lp, pages;  // chunk's first key and length; the wave's first row; the lane's row of an instruction
  int64_t page_bytes;
  uint32_t row_bytes;

  __device__ __forceinline__ void init(const PagedParams &p, int b, int first, int n, int wave, int lane, bool half) {
    const int cmask = half ? CPR / 2 - 1 : CPR - 1;
    key0 = first, keys = n, lp = p.lp, pages = p.num_pages;
    r0 = wave * RPW;
    lrow = lane / CPR;
    // (Uniform to the compiler, so that the entries are scalar loads: a vector
    // load would count among the tile copies that the kernels wait for.)
    const uint64_t at = (uint64_t)(uintptr_t)(p.table + (int64_t)b * p.table_stride);
    row = (ScalarInts)(((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32) |
                       (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at));
    page_bytes = p.sk_p * ESIZE, row_bytes = (uint32_t)(p.sk_t * ESIZE);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int in_tile = r0 + i * RPI + lrow;
      cbyte[i] = 16 * (((lane % CPR) ^ swz<D>(in_tile)) & cmask);
      voff[i] = (uint32_t)((i * RPI) % 16 + lrow) * row_bytes + cbyte[i];
    }
  }
  // Entries of the tile whose first key is `tile` of the chunk (of its last
  // key's page beyond; keys > 0).
  __device__ __forceinline__ void entries(int tile, int (&to)[NE]) const {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int key = key0 + min(tile + r0 + 16 * e, keys - 1);
      to[e] = row[__builtin_amdgcn_readfirstlane(key >> lp)];
    }
  }
  __device__ __forceinline__ void load(int tile) { entries(tile, ent); }
  static __device__ __forceinline__ void copy(uint16_t *lds, const char *base, uint32_t off) {
    const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    if constexpr (NT)
      asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" : : "v"(off), "s"(base), "{m0}"(dst) : "memory");
    else
      asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(dst) : "memory");
  }
  static __device__ __forceinline__ void copy_at(uint16_t *lds, const char *at) {
    const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(at), "{m0}"(dst) : "memory");
  }
  // Copies one tensor's tile with the entries `at` (head: the head's element 0
  // of page 0).
  __device__ __forceinline__ void issue_one(uint16_t *lds, const uint16_t *head, int tile) const {
    issue_at(lds, head, tile, ent);
  }
  __device__ __forceinline__ void issue_at(uint16_t *lds, const uint16_t *head, int tile, const int (&at)[NE]) const {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int first = tile + r0 + 16 * e;  // of the chunk
      const int id = at[e], n = keys - first;
      const bool there = id >= 0 && id < pages;
      const int in_page = (key0 + first) & ((1 << lp) - 1);
      const char *base = (const char *)head + (there ? id : 0) * page_bytes + (int64_t)in_page * row_bytes;
      constexpr int PER = NI / NE;
      if (there && n >= (RPW < 16 ? RPW : 16)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) copy(lds + (r0 + (e * PER + i) * RPI) * D, base, voff[e * PER + i]);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const bool in = there && i * RPI + lrow < n;
          copy_at(lds + (r0 + (e * PER + i) * RPI) * D, in ? base + voff[e * PER + i] : (const char *)kZeroPiece);
        }
      }
    }
  }
  // The same, for a tile that is followed by the one from key `next` on.
  __device__ __forceinline__ void issue_last(uint16_t *lds, const uint16_t *head, int tile, int next) {
    issue_one(lds, head, tile);
    if (next < keys) load(next);
  }
};

// Attention of every sequence: any dtype, alignment and strides.
void launch_paged_generic(const PagedParams &p, int dtype, int D, bool causal, hipStream_t st);
// MFMA kernels, dtype in {kF16, kBF16}, D in {32, 64, 128} (16 as 32 with
// dmem = 16), 16-byte aligned rows: blocks of paged_block(D) columns; a wave
// per chunk for sequences of up to kDecodeCols columns; and the sums of cut
// sequences.  ngap leading workgroups (pf's) zero the rows outside every sequence.
int paged_block(int D);
void launch_paged_fwd(const PagedParams &p, int units, int dtype, int D, bool causal, hipStream_t st);
void launch_paged_decode(const PagedParams &p, int units, int dtype, int D, bool causal, hipStream_t st);
// Both in one launch (nf and nd units).
void launch_paged_mixed(const PagedParams &pf, int nf, const PagedParams &pd, int nd, int dtype, int D, bool causal,
                        hipStream_t st);
// fp32, D in {32, 64, 128} (16 as above): blocks of kPagedBlockF32 columns, and a
// wave per chunk where every sequence has up to kDecodeCols.
constexpr int kPagedBlockF32 = 128;
void launch_paged_decode_f32(const PagedParams &p, int units, int D, bool causal, hipStream_t st);
void launch_paged_f32(const PagedParams &p, int units, int D, bool causal, hipStream_t st);
void launch_paged_reduce(const PagedParams &fwd, const PagedParams &decode, int dtype, int D, hipStream_t st);

}  // namespace sigattn
