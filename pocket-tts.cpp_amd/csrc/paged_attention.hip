// Attention of every request's new rows over its pages (pocket_tts_amd.h, ptts_paged_attention).
//
// The G query heads of a key head share its keys, so the rows of one request and one key head are packed: packed row m is new
// row m / G under head m % G.  Two forms work on tiles of packed rows:
//
//   chunk   128 packed rows, four waves of 32; key blocks of 64 go through LDS and are read by all four waves
//   few     16 packed rows; four waves walk different keys straight from memory and join at the end (float rows, and the
//           smallest calls, where its steps of 128 keys make the shorter chain)
//   merge   joins the results of rows whose keys were cut into splits
//
// The work is 4 head_dim operations a visible (query, key) pair and head against 4 head_dim bytes (16 bit) a key and key head, so a chunk
// is bound by the matrix pipes and the exponentials, single rows by the one read of the keys and values, short calls by the chain
// of dependent reads (lengths, page ids, rows).  Measured: 2048 rows on 16384 keys, 32 / 8 heads of 128, bf16: 509 us, 1.01 PFLOP/s (a
// library product of 8192^3 reaches 1.21); 16 rows on up to 16384 keys each, same heads, f16: 682 MB in 138 us, 4.9 TB/s (the
// same reads alone 6.0, a large copy 5.1); 64 rows on about 594 keys, 16 heads of 64: 102 MB in 26 us; one float row on 218 keys 8 us.
//
// All products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane keeps one query for the whole kernel (its
// running maximum and sum are scalars of the lane) and the weights leave the first product in the layout the second one takes
// them in.  Softmax statistics and both sums are float32; the weights are rounded once, to the rows' type, because the matrix
// instructions take both operands in one type (at most half a step of the type on each weight; float rows keep float weights).
//
// The running maximum is a reference that lags: sums are rescaled only when a score passes it by 2^8, which saves most rescales.
// Float16 weights are kept 2^7 times larger (at most 2^15, inside the type), so that a weight has to lie 2^-21 below the largest
// before it loses bits and 2^-32 below before it is lost; bf16 has float32's range and needs none of this.
#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "paged.h"

namespace ptts {

namespace {

constexpr int kChunkRows = 128, kChunkKeys = 64;   // chunk kernel: packed rows of a workgroup, keys of a block
constexpr int kFewRows = 16;                       // few kernel: packed rows of a workgroup
constexpr float kLn2 = 0.69314718055994531f, kLag = 8.0f;
template <typename T> constexpr float kLift = std::is_same<T, _Float16>::value ? 7.0f : 0.0f;

// How a call is cut: which form runs, over how many tiles, into how many splits of the keys.
struct Cut {
    bool chunk;
    long long tiles;
    int splits, least;          // least: fewest key blocks (chunk) or steps (few) of a split
    long long parts, bytes;     // rows of one split's results in the workspace; its size
};

struct AttnArgs {
    PttsPagedAttention p;
    FastDiv page, group;
    float scale2;               // scale * log2(e)
    long long tile0, tile1;     // tiles of this launch: tile0 .. tile1 - 1
    int splits, least;
    // results of splits: [split][row][head][dim] values, normalised by the split's own sum, and [split][row][head] of log2 sum exp2
    float *part, *lse;
    long long parts;
};

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
template <typename T> using x8 = T __attribute__((ext_vector_type(8)));
template <typename T> using x4 = T __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mma32(x8<__bf16> a, x8<__bf16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(x8<_Float16> a, x8<_Float16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(x8<__bf16> a, x8<__bf16> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(x8<_Float16> a, x8<_Float16> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Both halves of the wave (all four rows of 16 lanes) combined, result in every lane.
__device__ __forceinline__ float max_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_rows(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_half(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_rows(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return sum_half(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A tile of packed rows: the request that owns it and what its rows see.
struct Tile {
    int i, row0, n, len, pos0;      // request, its first row, row count, length, position of its first row
    int m0, m1;                     // packed rows m0 .. m1 - 1 of the request
    int p0, p1;                     // positions of the first and the last row of the tile
    int low;                        // first key of the window of row m0 (the lowest of the tile)
    int bad;
};

// Tile numbers of request i begin at cu_rows[i] * G / BM + i: its ceil(n G / BM) tiles end before those of the next request
// begin, so a tile finds its request without prefix sums, 64 requests at a time, and a few numbers stay unused.
__device__ __forceinline__ bool find_tile(const AttnArgs& a, long long tile, int rows_per_tile, Tile& t) {
    const PttsPagedAttention& p = a.p;
    const int lane = threadIdx.x & 63, G = a.group.d;
    int sub, end;
    auto first_of = [&](int i, int cu) { return (long long)cu * G / rows_per_tile + i; };
    int lo = 0, span = p.requests;
    while (span > 64) {
        const int step = (span + 63) >> 6, i = lo + lane * step;
        const bool hit = lane * step < span && first_of(i, p.cu_rows[i]) <= tile;
        const int hits = __popcll(__ballot(hit));
        if (hits == 0) return false;
        const int left = span - (hits - 1) * step;
        lo += (hits - 1) * step;
        span = left < step ? left : step;
    }
    // the last round reads all that the tile needs of its request at once
    int cu = 0, next = 0, len = 0;
    bool hit = false;
    if (lane < span) {
        cu = p.cu_rows[lo + lane];
        next = p.cu_rows[lo + lane + 1];
        len = p.kv_len[lo + lane];
        hit = first_of(lo + lane, cu) <= tile;
    }
    const int hits = __popcll(__ballot(hit));
    if (hits == 0) return false;
    t.i = lo + hits - 1;
    t.row0 = __builtin_amdgcn_readlane(cu, hits - 1);
    end = __builtin_amdgcn_readlane(next, hits - 1);
    t.len = __builtin_amdgcn_readlane(len, hits - 1);
    const long long first = first_of(t.i, t.row0);
    if (tile < first || tile - first > 0x7fffffff) return false;
    sub = (int)(tile - first);
    t.bad = 0;
    t.n = end - t.row0;
    if (t.row0 < 0 || end > p.rows || end < t.row0) {
        if (p.status && threadIdx.x == 0) atomicOr(p.status, kStatusRows);
        return false;
    }
    const int cap = p.table_width * p.pages.page_size;
    if (t.len < 0) { t.len = 0; t.bad = kStatusLength; }
    if (t.len > cap) { t.len = cap; t.bad = kStatusLength; }
    const long long packed = (long long)t.n * G, from = (long long)sub * rows_per_tile;
    if (from >= packed) return false;
    t.m0 = (int)from;
    t.m1 = (int)(packed - from < rows_per_tile ? packed : from + rows_per_tile);
    t.pos0 = t.len - t.n;
    t.p0 = t.pos0 + (int)a.group.div(t.m0);
    t.p1 = t.pos0 + (int)a.group.div(t.m1 - 1);
    t.low = p.window > 0 && t.p0 - p.window + 1 > 0 ? t.p0 - p.window + 1 : 0;
    return true;
}

// The key blocks that a tile has to look at: those of the sinks, then those from the window's first key to the last row's own.
struct Blocks {
    int sink, start, count;
    __device__ __forceinline__ Blocks(const Tile& t, int sinks, int keys) {
        sink = 0;
        start = t.low / keys;
        if (t.low > 0 && sinks > 0) sink = ((sinks < t.low ? sinks : t.low) + keys - 1) / keys;
        if (start < sink) start = sink;
        count = t.p1 < 0 ? 0 : sink + (t.p1 / keys - start + 1 > 0 ? t.p1 / keys - start + 1 : 0);
    }
    __device__ __forceinline__ int block(int u) const { return u < sink ? u : start + u - sink; }
};

__device__ __forceinline__ bool seen(const PttsPagedAttention& p, int key, int pos) {
    return key <= pos && (p.window <= 0 || key > pos - p.window || key < p.sinks);
}
// whether rows at positions p0 .. p1 all see the keys k0 .. k1 / whether none of them sees any
__device__ __forceinline__ bool all_seen(const PttsPagedAttention& p, int k0, int k1, int p0, int p1) {
    return k1 <= p0 && (p.window <= 0 || k0 > p1 - p.window || k1 < p.sinks);
}
__device__ __forceinline__ bool none_seen(const PttsPagedAttention& p, int k0, int k1, int p0, int p1) {
    return k0 > p1 || (p.window > 0 && k1 <= p0 - p.window && k0 >= p.sinks);
}

// The page id of a key, kUnseen where no row of the tile sees it.  The id is not looked at here, so that the load stays in flight.
constexpr int kUnseen = -0x7fffffff;
__device__ __forceinline__ int page_of(const AttnArgs& a, const Tile& t, const int* table, int key) {
    int id = kUnseen;
    if (key <= t.p1 && (key >= t.low || key < a.p.sinks)) id = table[a.page.div(key)];
    return id;
}
// Element offset of a key's row under one key head.  Rows that are not read (no row of the tile sees the key, or its page id is
// not one) have offset 0, inside the pool, and ok false: what is loaded there is replaced by zeros.
__device__ __forceinline__ long long row_at(const AttnArgs& a, int id, int key, int kvh, int& bad, bool& ok) {
    const PttsPages& g = a.p.pages;
    ok = id >= 0 && id < g.pages;
    if (!ok && id != kUnseen) bad |= kStatusPage;
    const long long at = (long long)id * g.page_stride + (long long)(key - (int)a.page.div(key) * g.page_size) * g.row_stride + (long long)kvh * g.head_stride;
    return ok ? at : 0;
}

// Values that are NaN or infinite and stand at keys which only some rows of a tile see must not meet the other rows' zero weights.
// In blocks at the border of what is seen they are replaced by zeros on their way to the products, and a workgroup that met one
// goes over its border blocks once more at the end and adds them, one by one, to the sums of the rows that see them (a weight is
// positive, so a NaN or an infinity reaches the sum as it is).
template <typename T> __device__ __forceinline__ unsigned finite_mask(unsigned w) {     // ones where a value of the word is finite
    if constexpr (std::is_same<T, float>::value) return (w & 0x7f800000u) == 0x7f800000u ? 0u : ~0u;
    constexpr unsigned e = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
    return ((w & e) == e ? 0u : 0xffffu) | (((w >> 16) & e) == e ? 0u : 0xffff0000u);
}
// N words cleaned; `kept` loses the bits of what was replaced
template <typename T, int N> __device__ __forceinline__ void clean(unsigned (&w)[N], unsigned& kept) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const unsigned m = finite_mask<T>(w[i]);
        w[i] &= m;
        kept &= m;
    }
}
__device__ __forceinline__ float add_not_finite(float sum, float v) { return fabsf(v) < INFINITY ? sum : sum + v; }

// exp2 of what is at most kLag + kLift; denormals flush to zero
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// ------------------------------------------------------------------ chunk

// LDS holds a block's 64 rows of DH values without padding.  16-byte unit c of row r lies at unit c ^ swizzle(r), which spreads the
// reads of one instruction over all banks: rows 0 .. 15 at one unit for the keys (16 bytes a lane), eight rows of four units each
// for the transposed reads of the values (8 bytes a lane).
template <int DH> __device__ __forceinline__ int key_swizzle(int row) { return DH >= 128 ? row & 15 : (row >> 1) & 7; }
template <int DH> __device__ __forceinline__ int value_swizzle(int row) { return DH >= 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

template <typename T, int DH> struct ChunkLds {
    T k[2][kChunkKeys * DH], v[2][kChunkKeys * DH];      // one block is read while the next arrives
};

// 16 bytes a lane from memory to LDS: lane l's land at `to` + 16 l
__device__ __forceinline__ void copy16(const void* from, void* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)from, (__attribute__((address_space(3))) unsigned*)to, 16, 0, 0);
}

// 128 rows a workgroup: each block of keys is read from LDS by four waves, and two (heads of 128) to four workgroups share a unit, so that
// one's exponentials run beside another's products.  The next block comes by asynchronous copies into the other LDS buffer; passing it through
// registers took 638 us in place of 588 (2048 rows on 16384 keys, at that stage), three buffers 780, the next block's scores beside
// this one's weights 650.
template <typename T, int DH> __global__ __launch_bounds__(256, DH == 256 ? 1 : DH == 128 ? 2 : 3) void attention_chunk_kernel(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) ChunkLds<T, DH> lds;
    const unsigned block = blockIdx.x;
    constexpr int kUnits = DH / 8, kPassRows = 256 / kUnits, kPasses = kChunkKeys / kPassRows, KS = DH / 16, NT = DH / 32;
    const PttsPagedAttention& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // matrix instructions ignore the lane mask: every branch around one is scalar
    // key heads first (neighbouring workgroups go to different dies, so a die's cache sees few heads), and the tiles that see
    // most keys first
    const int kvh = block % p.pages.kv_heads;
    const unsigned rest = block / p.pages.kv_heads;
    const int splits = a.splits, split = rest % splits;
    Tile t;
    if (!find_tile(a, a.tile1 - 1 - rest / splits, kChunkRows, t)) return;
    const int G = a.group.d, dim = p.pages.head_dim;
    const Blocks list(t, p.sinks, kChunkKeys);
    const int per = max(a.least, (list.count + splits - 1) / splits);
    const int u0 = split * per, u1 = min(list.count, u0 + per);

    // this lane's query, and the positions of this wave's rows
    const int mw = t.m0 + wave * 32, m = min(mw + col, t.m1 - 1), tok = a.group.div(m), head = kvh * G + m - tok * G;
    const bool live = mw + col < t.m1;
    const int pos = t.pos0 + tok, row = t.row0 + tok;
    const int pw0 = t.pos0 + (int)a.group.div(min(mw, t.m1 - 1)), pw1 = t.pos0 + (int)a.group.div(min(mw + 31, t.m1 - 1));
    const bool idle = mw >= t.m1;
    x8<T> qf[KS];
    {
        const T* q = (const T*)p.q + (long long)row * p.q_row_stride + (long long)head * p.q_head_stride + 8 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const x8<T> zero = {};
            qf[ks] = 16 * ks + 8 * h < dim ? *(const x8<T>*)(q + 16 * ks) : zero;
        }
    }

    const int* table = p.block_table + (long long)t.i * p.table_stride;
    const int unit = tid % kUnits, sr = tid / kUnits;
    const int place = (wave * (kPassRows / 4)) * DH;       // of the wave's rows in a pass
    int bad = t.bad, id = kUnseen;
    unsigned long long holes = 0;           // keys of the block on its way that are not read
    if (dim < DH) {                         // units behind the head's values stay zero
        for (int i = tid; i < (int)(sizeof(lds) / 16); i += 256) reinterpret_cast<uint4*>(&lds)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    // Lane l of every wave looks up key l of a block, one block before its rows are read; the threads that copy the row take its
    // place from there.
    auto look_up = [&](int u) { id = page_of(a, t, table, list.block(u) * kChunkKeys + lane); };
    auto load = [&](int u, int into) {
        bool ok;
        const long long mine = row_at(a, id, list.block(u) * kChunkKeys + lane, kvh, bad, ok);
        holes = __ballot(!ok);
        long long at[kPasses];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) at[i] = __shfl(mine, sr + kPassRows * i, 64);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int c = (unit ^ key_swizzle<DH>(sr + kPassRows * i)) * 8;      // the unit that lies at this lane's place
            if (DH == dim || c < dim) copy16((const T*)p.pages.k + at[i] + c, lds.k[into] + place + i * kPassRows * DH);
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int c = (unit ^ value_swizzle<DH>(sr + kPassRows * i)) * 8;
            if (DH == dim || c < dim) copy16((const T*)p.pages.v + at[i] + c, lds.v[into] + place + i * kPassRows * DH);
        }
    };

    f32x16 o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.f;
    float top = -INFINITY, sum = 0.f;      // reference of the exponents in log2 units, this lane's part of the sum

    const int vrow = 4 * h + ((lane & 15) >> 2);
    const int vunit = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vx = value_swizzle<DH>(vrow);
    int kbase = col * DH * 2 + ((key_swizzle<DH>(col) ^ h) << 4), vbase = vrow * DH * 2 + 8 * (lane & 1);    // bytes
    int now = 0;
    auto key_frag = [&](int b, int ks) {    // rows 32 b + col, head values 16 ks + 8 h ..: the swizzle is a part of kbase
        return *(const x8<T>*)((const char*)lds.k[now] + (kbase ^ (ks << 5)) + b * 32 * DH * 2);
    };
    auto value = [&](int n, int s) {        // V^T of 32 head values from 32 n and keys 16 s ..: keys 4 h + 0..3 and 8 + 4 h + 0..3
        const char* at = (const char*)lds.v[now] + vbase + (((4 * n + vunit) ^ vx) << 4) + 16 * s * DH * 2;
        union { s16x4 w[2]; x8<T> v; } u;
        u.w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        u.w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 8 * DH * 2));
        return u.v;
    };

    unsigned kept = ~0u;
    if (u0 < u1) {
        look_up(u0);
        load(u0, 0);
        if (u0 + 1 < u1) look_up(u0 + 1);
    }
    for (int u = u0; u < u1; ++u) {
        const int k0 = list.block(u) * kChunkKeys, k1 = k0 + kChunkKeys - 1;
        const bool border = !all_seen(p, k0, k1, t.p0, t.p1);       // some row of the tile does not see the block whole
        now = (u - u0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // what this wave copied has landed
        if (holes || border) {
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                uint4* kp = reinterpret_cast<uint4*>(lds.k[now] + place + i * kPassRows * DH) + lane;
                uint4* vp = reinterpret_cast<uint4*>(lds.v[now] + place + i * kPassRows * DH) + lane;
                if ((holes >> (sr + kPassRows * i)) & 1) { *kp = make_uint4(0, 0, 0, 0); *vp = make_uint4(0, 0, 0, 0); }
                else if (border) {
                    uint4 x = *vp;
                    clean<T>(reinterpret_cast<unsigned(&)[4]>(x), kept);
                    *vp = x;
                }
            }
        }
        __syncthreads();                    // the block is whole, and the one before is consumed
        if (u + 1 < u1) {
            load(u + 1, now ^ 1);
            if (u + 2 < u1) look_up(u + 2);
        }
        if (idle || (border && none_seen(p, k0, k1, pw0, pw1))) continue;
        asm volatile("" : "+v"(kbase));     // its variants are formed anew: kept, they would be spilled

        f32x16 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < 2; ++b) s[b] = mma32(key_frag(b, ks), qf[ks], s[b]);
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int i = 0; i < KS - 3; ++i) { __builtin_amdgcn_sched_group_barrier(0x8, 2, 0); __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); }
        __builtin_amdgcn_sched_group_barrier(0x8, 6, 0);
        // From here to the end of the block this wave goes first: two waves of a unit that run in step would otherwise form scores together
        // and weights together, each waiting for the same pipe (2048 rows on 16384 keys: 598 us without, 530 with it).
        __builtin_amdgcn_s_setprio(1);
        // lane: query col; s[b][r] belongs to key k0 + 32 b + 8 (r / 4) + 4 h + r % 4
        if (border) {
            const int mine = k0 + 4 * h, up = pos - mine, from = p.window > 0 ? up - p.window : -1, sink = p.sinks - mine;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int c = 32 * b + 8 * (r >> 2) + (r & 3);           // seen(p, mine + c, pos)
                    s[b][r] = c <= up && (c > from || c < sink) ? s[b][r] : -INFINITY;
                }
        }
        float best = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) best = fmaxf(best, s[b][r]);
        best = max_half(best) * a.scale2;
        if (__any(best > top + (kLag + kLift<T>))) {
            const float next = fmaxf(top, best - kLift<T>), fade = top == -INFINITY ? 0.f : exp2_of(top - next);
            top = next;
            sum *= fade;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[n][r] *= fade;
        }
        const float base = top == -INFINITY ? 0.f : top;
        x8<T> w[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = exp2_of(__builtin_fmaf(s[b][r], a.scale2, -base));
                sum += e;
                w[2 * b + (r >> 3)][r & 7] = (T)e;
            }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n] = mma32(value(n, k), w[k], o[n]);
        __builtin_amdgcn_s_setprio(0);
    }
    if (__syncthreads_or(kept != ~0u)) {
        for (int u = u0; u < u1; ++u) {
            const int k0 = list.block(u) * kChunkKeys;
            if (all_seen(p, k0, k0 + kChunkKeys - 1, t.p0, t.p1)) continue;
            look_up(u);
            bool ok;
            const long long mine = row_at(a, id, k0 + lane, kvh, bad, ok);
            const unsigned long long there = __ballot(ok);
#pragma unroll 1
            for (int j = 0; j < kChunkKeys; ++j) {
                const long long at = __shfl(mine, j, 64);
                if (!((there >> j) & 1) || !seen(p, k0 + j, pos)) continue;
                const T* v = (const T*)p.pages.v + at + 4 * h;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (32 * n + 8 * q < dim) {
                            const x4<T> x = *(const x4<T>*)(v + 32 * n + 8 * q);
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[n][4 * q + r] = add_not_finite(o[n][4 * q + r], (float)x[r]);
                        }
            }
        }
    }

    if (bad && p.status) atomicOr(p.status, bad);
    sum = sum_half(sum);
    if (!live) return;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum, lse2 = sum == 0.f ? -INFINITY : top + __log2f(sum);
    if (splits == 1) {
        T* out = (T*)p.out + (long long)row * p.out_row_stride + (long long)head * p.out_head_stride + 4 * h;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (32 * n + 8 * q < dim) {
                    x4<T> v;
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = (T)(sum == 0.f ? 0.f : o[n][4 * q + r] * inv);
                    *(x4<T>*)(out + 32 * n + 8 * q) = v;
                }
        if (p.lse && h == 0) p.lse[(long long)row * p.lse_row_stride + head] = lse2 * kLn2;
    } else {
        const long long at = split * a.parts + (long long)row * p.q_heads + head;
        float* part = a.part + at * dim + 4 * h;
        if (sum != 0.f)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (32 * n + 8 * q < dim)
                        *(f32x4*)(part + 32 * n + 8 * q) = f32x4{o[n][4 * q] * inv, o[n][4 * q + 1] * inv, o[n][4 * q + 2] * inv, o[n][4 * q + 3] * inv};
        if (h == 0) a.lse[at] = lse2;
    }
}

// ------------------------------------------------------------------ few

// Bound by the chain of reads: rows are asked for one step ahead and page ids three, which took 16 rows on 16384 keys from 169 to 150 us
// against reads at their use.
//
// Fragments of one step of a wave, straight from memory: NA blocks of 16 keys.  Keys: lane (row lane % 16, quarter g = lane / 16) reads
// the units g of its row.  Values: the lane reads head values CPL m .. CPL m + CPL - 1 (m = lane % 16) of the rows 4 g + r, so that
// column t of every lane forms the operand of output tile t; the output's order is then CPL * (its row) + t.
template <typename T, typename C, int DH> struct Step {
    static constexpr bool kFloat = std::is_same<T, float>::value;
    static constexpr int NA = kFloat ? 1 : 2, CPL = DH / 16, KS = kFloat ? DH / 16 : DH / 32, KW = kFloat ? 4 : 8;
    static constexpr int VW = CPL < 8 ? CPL : 8, VN = CPL / VW;     // values of one access, accesses of a row
    typedef C kvec __attribute__((ext_vector_type(KW)));
    typedef C vvec __attribute__((ext_vector_type(VW)));
    kvec k[NA][KS];
    vvec v[4 * NA][VN];
};

template <int DH> struct FewLds {
    union {
        long long places[4][32];                   // where the keys of a step lie: the step at work, the next and the one after
        float joined[kFewRows][DH + 4];            // +4: the waves' columns of one row do not meet in one bank
    } of[4];                                       // one for each wave
    float tops[4][kFewRows], sums[4][kFewRows];
};

// kFull: the head fills DH, so that no lane's values lie behind it.
template <typename T, typename C, int DH, bool kFull>
__global__ __launch_bounds__(256, DH == 256 ? 1 : DH == 128 ? 2 : 3) void attention_few_kernel(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) FewLds<DH> lds;
    const unsigned block = blockIdx.x;
    using S = Step<T, C, DH>;
    constexpr int NA = S::NA, CPL = S::CPL, KS = S::KS, KW = S::KW, VW = S::VW, VN = S::VN, kWaveKeys = 16 * NA, kKeys = 4 * kWaveKeys;
    constexpr bool kFloat = S::kFloat;
    auto &tops = lds.tops, &sums = lds.sums;
    const PttsPagedAttention& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // matrix instructions ignore the lane mask: every branch around one is scalar
    const int kvh = block % p.pages.kv_heads;
    const unsigned rest = block / p.pages.kv_heads;
    const int splits = a.splits, split = rest % splits;
    Tile t;
    if (!find_tile(a, a.tile0 + rest / splits, kFewRows, t)) return;
    const int G = a.group.d, dim = p.pages.head_dim;
    const Blocks list(t, p.sinks, kKeys);
    const int per = max(a.least, (list.count + splits - 1) / splits);
    const int u0 = split * per, u1 = min(list.count, u0 + per);

    const int m = min(t.m0 + li, t.m1 - 1), tok = a.group.div(m), head = kvh * G + m - tok * G, row = t.row0 + tok, pos = t.pos0 + tok;
    T qf[KS][KW];
    {
        const T* q = (const T*)p.q + (long long)row * p.q_row_stride + (long long)head * p.q_head_stride + KW * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < KW; ++j) qf[ks][j] = 4 * KW * ks + KW * g < dim ? q[4 * KW * ks + j] : (T)0.f;
    }

    const int* table = p.block_table + (long long)t.i * p.table_stride;
    int bad = t.bad;
    // Every step issues the same reads in the same order (page ids three steps ahead, rows one step ahead), whatever it will see of
    // them: waits count reads, and a branch around one would make the compiler wait for all.  Keys that are not read after
    // all are taken from the pool's first row and replaced by zeros when their step is at work.
    auto& mine = lds.of[wave];
    const int kk = lane % kWaveKeys;
    auto key_of = [&](int u, int k) { return list.block(u) * kKeys + wave * kWaveKeys + k; };
    auto fetch = [&](int u) { return table[a.page.div(min(key_of(min(u, u1 - 1), kk), t.p1))]; };
    auto settle = [&](int u, int id) {      // returns the keys of the step that are read, a bit each
        u = min(u, u1 - 1);
        const int key = key_of(u, kk);
        bool ok;
        const long long at = row_at(a, key <= t.p1 && (key >= t.low || key < p.sinks) ? id : kUnseen, min(key, t.p1), kvh, bad, ok);
        mine.places[u & 3][kk] = at;
        __builtin_amdgcn_wave_barrier();
        return (unsigned)__ballot(ok) | (kWaveKeys < 32 ? ~0u << (kWaveKeys & 31) : 0u);
    };
    auto load = [&](int u, S& x) {
        const long long* at = mine.places[min(u, u1 - 1) & 3];
#pragma unroll
        for (int b = 0; b < NA; ++b) {
            const C* k = (const C*)p.pages.k + at[16 * b + li];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = 4 * KW * ks + KW * g;
                x.k[b][ks] = *(const typename S::kvec*)(k + (kFull || d < dim ? d : 0));
            }
        }
#pragma unroll
        for (int r = 0; r < 4 * NA; ++r) {
            const C* v = (const C*)p.pages.v + at[16 * (r >> 2) + 4 * g + (r & 3)];
#pragma unroll
            for (int n = 0; n < VN; ++n) {
                const int d = CPL * li + VW * n;
                x.v[r][n] = *(const typename S::vvec*)(v + (kFull || d < dim ? d : 0));      // what lies behind the head is not stored
            }
        }
    };

    f32x4 o[CPL];
#pragma unroll
    for (int n = 0; n < CPL; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;

    unsigned kept = ~0u;
    auto work = [&](int u, S& x, unsigned there) {
        const int k0 = list.block(u) * kKeys + wave * kWaveKeys, k1 = k0 + kWaveKeys - 1;
        if (none_seen(p, k0, k1, t.p0, t.p1)) return;
        if constexpr (!kFull) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                if (4 * KW * ks + KW * g >= dim)
#pragma unroll
                    for (int b = 0; b < NA; ++b) x.k[b][ks] = typename S::kvec{};
        }
        if (there != ~0u) {
#pragma unroll
            for (int b = 0; b < NA; ++b)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    if (!((there >> (16 * b + li)) & 1)) x.k[b][ks] = typename S::kvec{};
#pragma unroll
            for (int r = 0; r < 4 * NA; ++r)
#pragma unroll
                for (int n = 0; n < VN; ++n)
                    if (!((there >> (16 * (r >> 2) + 4 * g + (r & 3))) & 1)) x.v[r][n] = typename S::vvec{};
        }
        f32x4 s[NA];
#pragma unroll
        for (int b = 0; b < NA; ++b) {
            s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (kFloat) {
#pragma unroll
                    for (int j = 0; j < KW; ++j) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)x.k[b][ks][j], qf[ks][j], s[b], 0, 0, 0);
                } else {
                    x8<T> q;
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[j] = qf[ks][j];
                    s[b] = mma16(x.k[b][ks], q, s[b]);
                }
            }
        }
        // lane: query li; s[b][r] belongs to key k0 + 16 b + 4 g + r
        if (!all_seen(p, k0, k1, t.p0, t.p1)) {
#pragma unroll
            for (int b = 0; b < NA; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[b][r] = seen(p, k0 + 16 * b + 4 * g + r, pos) ? s[b][r] : -INFINITY;
            if (t.p0 != t.p1) {            // rows of one position see the same keys, and what they do not see was not read
#pragma unroll
                for (int r = 0; r < 4 * NA; ++r)
#pragma unroll
                    for (int n = 0; n < VN; ++n) clean<C>(reinterpret_cast<unsigned(&)[sizeof(C) * VW / 4]>(x.v[r][n]), kept);
            }
        }
        float best = s[0][0];
#pragma unroll
        for (int b = 0; b < NA; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) best = fmaxf(best, s[b][r]);
        best = max_rows(best) * a.scale2;
        if (__any(best > top + (kLag + kLift<T>))) {
            const float next = fmaxf(top, best - kLift<T>), fade = top == -INFINITY ? 0.f : exp2_of(top - next);
            top = next;
            sum *= fade;
#pragma unroll
            for (int n = 0; n < CPL; ++n) o[n] *= fade;
        }
        const float base = top == -INFINITY ? 0.f : top;
        float e[4 * NA];
#pragma unroll
        for (int b = 0; b < NA; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                e[4 * b + r] = exp2_of(__builtin_fmaf(s[b][r], a.scale2, -base));
                sum += e[4 * b + r];
            }
        if constexpr (kFloat) {
#pragma unroll
            for (int n = 0; n < CPL; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[n] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)x.v[r][n / VW][n % VW], e[r], o[n], 0, 0, 0);
        } else {
            x8<T> w;
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = (T)e[j];
#pragma unroll
            for (int n = 0; n < CPL; ++n) {
                // column n of the eight rows: halves of their registers put together in pairs
                union { unsigned d[4]; x8<T> v; } u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    union { typename S::vvec v; unsigned d[VW / 2]; } lo, hi;
                    lo.v = x.v[2 * j][n / VW];
                    hi.v = x.v[2 * j + 1][n / VW];
                    u.d[j] = __builtin_amdgcn_perm(hi.d[n % VW / 2], lo.d[n % VW / 2], n & 1 ? 0x07060302u : 0x05040100u);
                }
                o[n] = mma16(u.v, w, o[n]);
            }
        }
    };

    if (u0 < u1) {
        S one, two;
        const int first = fetch(u0), second = fetch(u0 + 1);
        int id = fetch(u0 + 2);
        unsigned now = settle(u0, first), next = settle(u0 + 1, second);
        load(u0, one);
        for (int u = u0; u < u1; u += 2) {
            int after = fetch(u + 3);
            load(u + 1, two);
            unsigned then = settle(u + 2, id);
            work(u, one, now);
            id = fetch(u + 4);
            load(u + 2, one);
            now = then;
            then = settle(u + 3, after);
            if (u + 1 < u1) work(u + 1, two, next);
            next = then;
        }
    }
    if (__any(kept != ~0u)) {
        for (int u = u0; u < u1; ++u) {
            const int k0 = list.block(u) * kKeys + wave * kWaveKeys;
            if (all_seen(p, k0, k0 + kWaveKeys - 1, t.p0, t.p1) || none_seen(p, k0, k0 + kWaveKeys - 1, t.p0, t.p1)) continue;
#pragma unroll
            for (int b = 0; b < NA; ++b) {
                bool ok;
                const long long mine = row_at(a, page_of(a, t, table, k0 + 16 * b + li), k0 + 16 * b + li, kvh, bad, ok);
                const unsigned there = (unsigned)__ballot(ok);
#pragma unroll 1
                for (int j = 0; j < 16; ++j) {
                    const long long at = __shfl(mine, j, 64);
                    if (!((there >> j) & 1) || !seen(p, k0 + 16 * b + j, pos)) continue;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int n = 0; n < VN; ++n) {
                            const int d = CPL * (4 * g + r) + VW * n;
                            if (d >= dim) continue;
                            const typename S::vvec v = *(const typename S::vvec*)((const C*)p.pages.v + at + d);
#pragma unroll
                            for (int c = 0; c < VW; ++c) o[VW * n + c][r] = add_not_finite(o[VW * n + c][r], (float)v[c]);
                        }
                }
            }
        }
    }
    if (bad && p.status) atomicOr(p.status, bad);

    // join the four waves: lane holds query li, head values CPL (4 g + r) + n
    sum = sum_rows(sum);
    if (g == 0) { tops[wave][li] = top; sums[wave][li] = sum; }
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) all = fmaxf(all, tops[w][li]);
    const float weight = top == -INFINITY ? 0.f : exp2_of(top - all);
    const int n_live = t.m1 - t.m0;
    if (li < n_live) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < CPL; n += 4)
                *(f32x4*)&mine.joined[li][CPL * (4 * g + r) + n] = f32x4{o[n][r], o[n + 1][r], o[n + 2][r], o[n + 3][r]} * weight;
    }
    __syncthreads();
    const int quads = dim / 4;
    for (int x = tid; x < n_live * quads; x += 256) {
        const int q = x / quads, d = 4 * (x - q * quads);
        float big = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) big = fmaxf(big, tops[w][q]);
#pragma unroll
        for (int w = 0; w < 4; ++w) total += tops[w][q] == -INFINITY ? sums[w][q] : sums[w][q] * exp2_of(tops[w][q] - big);     // 0 or NaN
        f32x4 v = *(f32x4*)&lds.of[0].joined[q][d];
#pragma unroll
        for (int w = 1; w < 4; ++w) v += *(f32x4*)&lds.of[w].joined[q][d];
        const float inv = total == 0.f ? 0.f : 1.0f / total, lse2 = total == 0.f ? -INFINITY : big + __log2f(total);
        const int mq = t.m0 + q, tq = a.group.div(mq), hq = kvh * G + mq - tq * G;
        const long long rq = t.row0 + tq;
        if (splits == 1) {
            x4<T> w;
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = (T)(total == 0.f ? 0.f : v[r] * inv);
            *(x4<T>*)((T*)p.out + rq * p.out_row_stride + (long long)hq * p.out_head_stride + d) = w;
            if (p.lse && d == 0) p.lse[rq * p.lse_row_stride + hq] = lse2 * kLn2;
        } else {
            const long long at = split * a.parts + rq * p.q_heads + hq;
            if (total != 0.f) *(f32x4*)(a.part + at * dim + d) = v * inv;
            if (d == 0) a.lse[at] = lse2;
        }
    }
}

// ------------------------------------------------------------------ merge

// `Many` splits taken in: top, total and v are the state so far.  Their reads are on their way together; a split that saw nothing wrote no
// values.
template <int Many>
__device__ __forceinline__ void merge_some(const float* part, const float* lse, long long stride, int s, int splits, long long at, int dim, int d, float& top,
                                           float& total, f32x4& v) {
    float l[Many], next = top;
    f32x4 x[Many];
#pragma unroll
    for (int j = 0; j < Many; ++j) {
        const long long from = min(s + j, splits - 1) * stride + at;
        l[j] = s + j < splits ? lse[from] : -INFINITY;
        x[j] = *(const f32x4*)(part + from * dim + d);
    }
#pragma unroll
    for (int j = 0; j < Many; ++j) next = fmaxf(next, l[j]);
    const float fade = top == -INFINITY ? 1.0f : exp2_of(top - next), base = next == -INFINITY ? 0.f : next;
    top = next;
    total *= fade;
    v *= fade;
#pragma unroll
    for (int j = 0; j < Many; ++j)
        if (l[j] != -INFINITY) {
            const float w = exp2_of(l[j] - base);        // NaN if the split's is
            total += w;
            v += x[j] * w;
        }
}

// out = sum over splits of exp2(lse_s - lse) part_s, four values a thread.  A chain of reads: 16 splits at a time, with four, a call of one row on
// 32768 keys in 64 splits took 27.2 us in place of 22.
template <typename T>
__device__ __forceinline__ void merge_one(const AttnArgs& a, long long row, int head, int d) {
    const PttsPagedAttention& p = a.p;
    const int splits = a.splits;
    const long long at = row * p.q_heads + head;
    float top = -INFINITY, total = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    int s = 0;
    for (; s + 4 < splits; s += 16) merge_some<16>(a.part, a.lse, a.parts, s, splits, at, p.pages.head_dim, d, top, total, v);
    if (s < splits) merge_some<4>(a.part, a.lse, a.parts, s, splits, at, p.pages.head_dim, d, top, total, v);
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    x4<T> y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = (T)(v[r] * inv);
    *(x4<T>*)((T*)p.out + row * p.out_row_stride + (long long)head * p.out_head_stride + d) = y;
    if (p.lse && d == 0) p.lse[row * p.lse_row_stride + head] = total == 0.f ? -INFINITY : (top + __log2f(total)) * kLn2;
}

// A row for each workgroup in x; workgroups along y share its heads.
template <typename T> __global__ __launch_bounds__(256) void attention_merge_kernel(AttnArgs a) {
    const PttsPagedAttention& p = a.p;
    const int quads = p.pages.head_dim / 4;
    const int lane = threadIdx.x & 63, row = blockIdx.x;
    // the request that owns the row: the last i with cu_rows[i] <= row
    int i = 0, span = p.requests;
    while (span > 1) {
        const int step = (span + 63) >> 6, at = i + lane * step;
        const int hits = __popcll(__ballot(lane * step < span && p.cu_rows[at] <= row));
        if (hits == 0) return;
        const int left = span - (hits - 1) * step;
        i += (hits - 1) * step;
        span = left < step ? left : step;
    }
    const int r0 = p.cu_rows[i], r1 = p.cu_rows[i + 1];
    if (r0 < 0 || r0 > row || row >= r1 || r1 > p.rows) return;
    const int x = blockIdx.y * 256 + threadIdx.x;
    if (x < p.q_heads * quads) {
        const int head = x / quads;
        merge_one<T>(a, row, head, 4 * (x - head * quads));
    }
}

// ------------------------------------------------------------------ host

constexpr int kMostSplits = 64;

Cut cut_of(const PttsPagedAttention& p, int cus) {
    Cut c;
    const int kvh = p.pages.kv_heads;
    const long long G = p.q_heads / kvh, packed = p.rows * G;
    const bool is_float = p.q_type == PTTS_TYPE_F32;
    const long long most_rows = p.max_rows > 0 ? std::min(p.max_rows, p.rows) : p.rows;
    long long keys = std::max(1ll, static_cast<long long>(p.table_width) * p.pages.page_size);
    if (p.max_kv > 0) keys = std::min<long long>(keys, p.max_kv);
    if (p.window > 0) keys = std::min<long long>(keys, static_cast<long long>(p.window) + p.sinks + most_rows);  // what a tile sees
    // Float rows have the few form alone.  Others take it where one workgroup a unit and a few of its longer steps do the whole call, that is where
    // latency is all: one row of 16 heads of 64 on 200 keys takes 6.2 us and 9.2 in the chunk form, one of 16 / 2 heads of 128 on 600 keys
    // 12.4 and 13.8; on 2048 keys the first takes 13.2 and 12.1, 64 such rows on 1024 keys 65 and 61, 16 rows of 16 / 2 heads of 128 on
    // 4096 keys 30 and 23, 16 of 32 / 8 heads on 16384 keys 144 and 138, four rows a request 33 and 25.
    c.chunk = !is_float && (most_rows * G > kFewRows || keys > 1024 || static_cast<long long>(p.requests) * kvh > cus);
    const int rows = c.chunk ? kChunkRows : kFewRows;
    c.tiles = packed / rows + p.requests;
    // Splits cost a second launch and a round trip of the rows.  They are made up to what the compute units hold at once (24
    // requests of one row, 16 heads of 64, about 1000 keys in a window: two a unit 30.2 us, three 26.1; heads of 128: 256 rows on 16384 keys without
    // splits 351 us, one a unit 62, two 53, three 65), and none is shorter than what pays for the rest: 256 keys in the chunk form (16 requests of 4 rows on 4096
    // keys: 128 keys 35 us, 256 28, 512 29, 1024 39), 256 KB of keys and values in the few form.
    const long long want = (p.pages.head_dim <= 64 ? 3 : p.pages.head_dim <= 128 ? 2 : 1) * static_cast<long long>(cus);
    const long long groups = std::max<long long>(p.requests, packed / rows) * kvh;
    const long long least_keys = c.chunk ? 256 : (256 << 10) / (2 * p.pages.head_dim * type_size(p.pages.type));
    c.splits = static_cast<int>(std::max(1ll, std::min({want / groups, keys / least_keys, static_cast<long long>(kMostSplits)})));
    const int step = c.chunk ? kChunkKeys : is_float ? 64 : 128;          // keys of a block, of one step of a workgroup
    c.least = static_cast<int>(std::max(1ll, (keys / step + c.splits - 1) / c.splits));
    c.parts = static_cast<long long>(p.rows) * p.q_heads;
    c.bytes = c.splits > 1 ? c.splits * c.parts * (p.pages.head_dim + 1ll) * 4 : 0;
    return c;
}

template <typename T, typename C, int DH> void launch_few_of(const AttnArgs& a, unsigned grid, hipStream_t s) {
    if (a.p.pages.head_dim == DH) launch_paged(attention_few_kernel<T, C, DH, true>, dim3(grid), s, a);
    else launch_paged(attention_few_kernel<T, C, DH, false>, dim3(grid), s, a);
}
template <typename T, typename C> void launch_few(const AttnArgs& a, unsigned grid, hipStream_t s) {
    const int d = a.p.pages.head_dim;
    if (d <= 64) launch_few_of<T, C, 64>(a, grid, s);
    else if (d <= 128) launch_few_of<T, C, 128>(a, grid, s);
    else launch_few_of<T, C, 256>(a, grid, s);
}
template <typename T> void launch_chunk(const AttnArgs& a, unsigned grid, hipStream_t s) {
    const int d = a.p.pages.head_dim;
    if (d <= 64) launch_paged(attention_chunk_kernel<T, 64>, dim3(grid), s, a);
    else if (d <= 128) launch_paged(attention_chunk_kernel<T, 128>, dim3(grid), s, a);
    else launch_paged(attention_chunk_kernel<T, 256>, dim3(grid), s, a);
}

// A launch holds fewer than 2^32 threads.
constexpr long long kMostGroups = (1 << 24) - 1;

}  // namespace

void check_paged_attention(const PttsPagedAttention& p) {
    const std::string w = "paged_attention: ";
    if (p.rows < 0 || p.rows >= 1 << 30) throw std::runtime_error(w + "rows must be 0 to 2^30 - 1");
    if (p.requests < 0 || p.requests > 65536) throw std::runtime_error(w + "requests must be 0 to 65536");
    check_pages(p.pages, "paged_attention");
    if (p.q_heads > 0 && static_cast<long long>(p.rows) * (p.q_heads / p.pages.kv_heads) >= 1ll << 30)
        throw std::runtime_error(w + "rows * q_heads / kv_heads must be below 2^30");
    if (p.q_type != PTTS_TYPE_F32 && p.q_type != PTTS_TYPE_BF16 && p.q_type != PTTS_TYPE_F16) throw std::runtime_error(w + "unknown type");
    if (p.pages.type != p.q_type && !(p.q_type == PTTS_TYPE_F32 && p.pages.type == PTTS_TYPE_BF16))
        throw std::runtime_error(w + "pages must have the rows' type, or bf16 under f32 rows");
    if (p.q_heads < 1 || p.q_heads > 65535 || p.q_heads % p.pages.kv_heads) throw std::runtime_error(w + "q_heads must be a multiple of kv_heads, at most 65535");
    if (!(p.scale > 0.f) || !std::isfinite(p.scale)) throw std::runtime_error(w + "scale must be positive and finite");
    if (p.sinks < 0) throw std::runtime_error(w + "sinks must not be negative");
    if (p.max_rows < 0 || p.max_kv < 0) throw std::runtime_error(w + "max_rows and max_kv must not be negative");
    if (p.table_width < 0 || static_cast<long long>(p.table_width) * p.pages.page_size >= 1ll << 30)
        throw std::runtime_error(w + "table_width * page_size must be below 2^30");
    if (p.requests > 1 && p.table_stride < p.table_width) throw std::runtime_error(w + "table_stride is smaller than table_width");
    if (p.rows == 0 || p.requests == 0) return;
    if (!p.q || !p.out || !p.cu_rows || !p.kv_len || (p.table_width > 0 && !p.block_table))
        throw std::runtime_error(w + "q, out, cu_rows, kv_len and block_table are required");
    if (!aligned({p.block_table, p.cu_rows, p.kv_len, p.lse, p.status}, 4))
        throw std::runtime_error(w + "block_table, cu_rows, kv_len, lse and status must be aligned to 4 bytes");
    if (p.q == p.out) throw std::runtime_error(w + "out must not be q");
    const int e = 16 / type_size(p.q_type);
    if (reinterpret_cast<uintptr_t>(p.q) % 16 || p.q_row_stride % e || p.q_head_stride % e || reinterpret_cast<uintptr_t>(p.out) % 16 ||
        p.out_row_stride % e || p.out_head_stride % e)
        throw std::runtime_error(w + "q and out must be aligned to 16 bytes, strides too");
}

long long paged_attention_workspace(const PttsPagedAttention& p, int cus) { return p.rows == 0 || p.requests == 0 ? 0 : cut_of(p, cus).bytes; }

void launch_paged_attention(const PttsPagedAttention& p, int cus, hipStream_t s) {
    if (p.rows == 0 || p.requests == 0) return;
    const Cut c = cut_of(p, cus);
    if (c.bytes > 0) {
        if (!p.workspace || p.workspace_bytes < c.bytes)
            throw std::runtime_error("paged_attention: a workspace of " + std::to_string(c.bytes) + " bytes is required");
        if (reinterpret_cast<uintptr_t>(p.workspace) % 16) throw std::runtime_error("paged_attention: the workspace must be aligned to 16 bytes");
    }
    AttnArgs a;
    a.p = p;
    if (p.window > 1 << 30) a.p.window = 0;          // no context is that long
    a.page = FastDiv::of(static_cast<unsigned>(p.pages.page_size));
    a.group = FastDiv::of(static_cast<unsigned>(p.q_heads / p.pages.kv_heads));
    a.scale2 = p.scale * 1.4426950408889634f;
    a.splits = c.splits;
    a.least = c.least;
    a.part = static_cast<float*>(p.workspace);
    a.lse = a.part + c.splits * c.parts * p.pages.head_dim;
    a.parts = c.parts;
    // all tiles in one launch, as far as one holds them
    const long long groups = static_cast<long long>(c.splits) * p.pages.kv_heads, most = kMostGroups / groups;
    for (a.tile0 = 0; a.tile0 < c.tiles; a.tile0 = a.tile1) {
        a.tile1 = std::min(a.tile0 + most, c.tiles);
        const unsigned grid = static_cast<unsigned>((a.tile1 - a.tile0) * groups);
        if (c.chunk) {
            if (p.q_type == PTTS_TYPE_BF16) launch_chunk<__bf16>(a, grid, s);
            else launch_chunk<_Float16>(a, grid, s);
        } else if (p.q_type == PTTS_TYPE_F32 && p.pages.type == PTTS_TYPE_BF16) {
            launch_few<float, __bf16>(a, grid, s);
        } else if (p.q_type == PTTS_TYPE_F32) {
            launch_few<float, float>(a, grid, s);
        } else if (p.q_type == PTTS_TYPE_BF16) {
            launch_few<__bf16, __bf16>(a, grid, s);
        } else {
            launch_few<_Float16, _Float16>(a, grid, s);
        }
    }
    if (c.bytes > 0) {
        const long long items = static_cast<long long>(p.q_heads) * (p.pages.head_dim / 4);
        const dim3 merge(p.rows, static_cast<unsigned>((items + 255) / 256));
        if (p.q_type == PTTS_TYPE_F32) launch_paged(attention_merge_kernel<float>, merge, s, a);
        else if (p.q_type == PTTS_TYPE_BF16) launch_paged(attention_merge_kernel<__bf16>, merge, s, a);
        else launch_paged(attention_merge_kernel<_Float16>, merge, s, a);
    }
}

}  // namespace ptts
