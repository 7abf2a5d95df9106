// Dense products of batches with several models and of 8-bit matrices (include/dgcn.h: dgcn_transform_grouped_batch,
// dgcn_transform_int8_batch, dgcn_transform_grouped_int8_batch).
//
//   Y[r][n] = act( epilogue( sum_k H[r][k] * W[e(r)][n][k] ) + bias[e(r)][n] )
//
// Every type runs the same tile loop in BYTES: 64 bytes of a row of H and of W feed one step of a 16 x 16 output tile, 16 bytes per
// lane (lane & 15 = the row, lane >> 4 = which 16 of the 64 bytes): one MFMA of int8 (k = 64), bf16 / fp16 (k = 32), four of float32
// (k = 4 each).  W is the MFMA's A operand and H its B operand, so a lane ends with four output columns n of ONE row r.
#include <atomic>
#include <type_traits>

#include "common.h"

namespace dgcn {

using i32x4 = __attribute__((ext_vector_type(4))) int;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f64x4 = __attribute__((ext_vector_type(4))) double;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

enum Kind { K_I8 = 0, K_BF16 = 1, K_F16 = 2, K_F32 = 3, K_F32P = 4 };  // (F32P: the chain in double)

struct ProductArgs {
    const char* H;       // [rows][ldh] (NULL: float32 only, every entry is h_const)
    const char* W;       // [num_models][ctot][cin]
    void* Y;             // [rows][ldy]
    const float* bias;   // [num_models][ctot] or NULL
    const float* hs;     // [rows] (int8)
    const float* ws;     // [num_models][ctot] (int8)
    const int32_t* gptr; // [num_groups + 1] or NULL: one group of all rows
    const int32_t* mog;  // [num_groups] or NULL: model g
    int32_t* status;
    int64_t ldh, ldy;    // elements
    float h_const;
    int rows, cin, ctot, num_groups, num_models, act, out_dtype;
    bool dwords_h, dwords_w;  // rows of H, of W start at multiples of 4 bytes
    bool stream;              // Y is stored past the caches (see streams_out)
    bool counted;             // tiles are numbered by find_tile_counted
};

template <int KIND> struct Elem;
template <> struct Elem<K_I8> { static constexpr int size = 1; using Acc = i32x4; };
template <> struct Elem<K_BF16> { static constexpr int size = 2; using Acc = f32x4; };
template <> struct Elem<K_F16> { static constexpr int size = 2; using Acc = f32x4; };
template <> struct Elem<K_F32> { static constexpr int size = 4; using Acc = f32x4; };
template <> struct Elem<K_F32P> { static constexpr int size = 4; using Acc = f64x4; };

struct Tile { int row0, row1, model, col; };  // rows [row0, row1), columns from col on; row0 >= row1: nothing to do

// Workgroups go to the XCDs round robin; tile numbers are dealt so that an XCD's workgroups take neighbouring tiles (shared rows of
// H and W meet in its L2).  (A launch has fewer than 2^24 workgroups: tile numbers and their divisions are 32 bits wide.)
__device__ __forceinline__ int xcd_order(int b, int total) {
    const int q = total >> 3, r = total & 7, x = b & 7;
    return x * q + min(x, r) + (b >> 3);
}

// Tile number `tile` of slots x col_tiles -> slot; `col` <- column tile.  Four slots side by side, column by column: a square-ish patch is
// in flight at a time.
__device__ __forceinline__ int patch_order(int tile, int slots, int col_tiles, int& col) {
    if (col_tiles == 1) { col = 0; return tile; }
    const int first = (int)((unsigned)tile / (4u * (unsigned)col_tiles)) * 4;
    const unsigned h = (unsigned)min(4, slots - first), in = (unsigned)(tile - first * col_tiles);
    col = (int)(in / h);
    return first + (int)(in % h);
}

__device__ __forceinline__ bool bad_group(const ProductArgs& a, int p0, int p1, int e) {
    return p0 < 0 || p1 < p0 || p1 > a.rows || e < 0 || e >= a.num_models;
}

// Up to 256 groups and rows of more than 256 bytes (see product_dispatch): every wave reads the whole table, four groups per lane, and counts their row tiles, so that every workgroup up to
// the number of tiles has one (at most min(rows, floor(rows / BM) + num_groups) x column tiles) and the XCDs' shares are equal.  A
// group's tiles are neighbours, column by column: its weights are read into an XCD's L2 once (64 groups of 256 rows on average, int8
// 2 000 x 2 050: with the groups' last, shorter tiles numbered behind all others 654 MB passed the L2 instead of 448).  Workgroup 0
// reports bad entries.  Pointers are clamped to [0, rows] before use: a bad table cannot lead out of the matrix.
constexpr int kCountedGroups = 256;
template <int BM> __device__ __forceinline__ Tile find_tile_counted(const ProductArgs& a, int b, int col_tiles) {
    constexpr int N = kCountedGroups / 64;
    const int lane = threadIdx.x & 63;
    const int per = (a.num_groups + 63) >> 6;
    int p[N], len[N], e[N], sum = 0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int g = lane * per + i;
        p[i] = len[i] = 0;
        e[i] = -1;
        if (i < per && g < a.num_groups) {
            const int v0 = a.gptr[g], v1 = a.gptr[g + 1];
            e[i] = a.mog ? a.mog[g] : g;
            bad |= bad_group(a, v0, v1, e[i]);
            p[i] = min(max(v0, 0), a.rows);
            len[i] = max(min(max(v1, 0), a.rows) - p[i], 0);
        }
        sum += (int)((unsigned)(len[i] + BM - 1) / BM);
    }
    if (b == 0 && bad) atomicOr(a.status, (int)DGCN_FAULT_BAD_GROUP);
    int upto = sum;  // row tiles of this lane's groups and of all before
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int w = __shfl_up(upto, d);
        if (lane >= d) upto += w;
    }
    Tile t{0, 0, 0, 0};
    const int slots = __builtin_amdgcn_readlane(upto, 63);
    if (b >= (int64_t)slots * col_tiles) return t;  // (a table that goes back and forth counts rows twice: the product may be large)
    const int tile = xcd_order(b, slots * col_tiles);
    const int slot = (int)((unsigned)tile / (unsigned)col_tiles);  // (in the order of groups: says which group, not yet which of its tiles)
    const unsigned long long m = __ballot(upto > slot);
    if (m == 0) return t;
    const int owner = __builtin_ctzll(m);
    int base = upto - sum, q0 = 0, qn = 0, qe = -1, qb = 0;  // the owner's group with that slot: first row, rows, model, first slot
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int n = (int)((unsigned)(len[i] + BM - 1) / BM);
        if (slot >= base && slot < base + n) { q0 = p[i]; qn = len[i]; qe = e[i]; qb = base; }
        base += n;
    }
    q0 = __builtin_amdgcn_readlane(q0, owner); qn = __builtin_amdgcn_readlane(qn, owner);
    qe = __builtin_amdgcn_readlane(qe, owner); qb = __builtin_amdgcn_readlane(qb, owner);
    if (qe < 0 || qe >= a.num_models) return t;
    const int tiles = (int)((unsigned)(qn + BM - 1) / BM), at = patch_order(tile - qb * col_tiles, tiles, col_tiles, t.col);
    if ((unsigned)at >= (unsigned)tiles || (unsigned)t.col >= (unsigned)col_tiles) return t;  // (such a table only)
    t.row0 = q0 + at * BM;
    t.row1 = min(t.row0 + BM, q0 + qn);
    t.model = qe;
    return t;
}

// Otherwise no count at all.  Group g's row tiles start at slot floor(p_g / BM) + g, which is increasing in g, and
// ceil((p_{g+1} - p_g) / BM) never exceeds the distance to the next group's start.  So floor(rows / BM) + num_groups slots cover every
// tile (some slots are empty), and a slot finds its group by search: 64-ary, a lane per probe.  Slot g < num_groups checks entry g.
template <int BM> __device__ __forceinline__ Tile find_tile(const ProductArgs& a, int b, int slots, int col_tiles) {
    if (a.counted) return find_tile_counted<BM>(a, b, col_tiles);
    Tile t{0, 0, 0, 0};
    const int slot = patch_order(xcd_order(b, slots * col_tiles), slots, col_tiles, t.col);
    if (!a.gptr) {
        t.row0 = slot * BM;
        t.row1 = min(t.row0 + BM, a.rows);
        return t;
    }
    if (t.col == 0 && slot < a.num_groups && threadIdx.x == 0) {
        if (bad_group(a, a.gptr[slot], a.gptr[slot + 1], a.mog ? a.mog[slot] : slot)) atomicOr(a.status, (int)DGCN_FAULT_BAD_GROUP);
    }
    const int lane = threadIdx.x & 63;
    auto start = [&](int g, int p) { return (int)((unsigned)p / BM) + g; };  // (below 2^24 for every group of a launch)
    auto clamp = [&](int p) { return min(max(p, 0), a.rows); };
    int lo = 0, n = a.num_groups;  // the group is in [lo, lo + n)
    while (n > 64) {
        const int step = (n + 63) >> 6;
        const int i = min(lane * step, n - 1);
        const unsigned long long m = __ballot(lane * step < n && start(lo + i, clamp(a.gptr[lo + i])) <= slot);
        const int k = m == ~0ull ? 64 : __builtin_ctzll(~m);
        if (k == 0) return t;  // in front of the first group
        const int at = (k - 1) * step;
        lo += at;
        n = min(step, n - at);
    }
    // at most 64 candidates: a lane each, its pointers and model number with it
    const int g = lo + min(lane, n - 1);
    const int p0 = clamp(a.gptr[g]), p1 = clamp(a.gptr[g + 1]), e = a.mog ? a.mog[g] : g;
    const unsigned long long m = __ballot(lane < n && start(g, p0) <= slot);
    const int k = m == ~0ull ? 64 : __builtin_ctzll(~m);
    if (k == 0) return t;
    const int at = __builtin_amdgcn_readfirstlane(k - 1);
    const int q0 = __builtin_amdgcn_readlane(p0, at), q1 = __builtin_amdgcn_readlane(p1, at), qe = __builtin_amdgcn_readlane(e, at);
    const int64_t r = q0 + (int64_t)(slot - start(lo + at, q0)) * BM;
    if (r < q0 || r >= q1 || qe < 0 || qe >= a.num_models) return t;
    t.row0 = (int)r;
    t.row1 = (int)min(r + BM, (int64_t)q1);
    t.model = qe;
    return t;
}

template <int KIND>
__device__ __forceinline__ typename Elem<KIND>::Acc mfma_step(i32x4 w, i32x4 h, typename Elem<KIND>::Acc c) {
    if constexpr (KIND == K_I8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, h, c, 0, 0, 0);
    if constexpr (KIND == K_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, h), c, 0, 0, 0);
    if constexpr (KIND == K_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, h), c, 0, 0, 0);
    if constexpr (KIND == K_F32 || KIND == K_F32P) {
        const f32x4 wf = __builtin_bit_cast(f32x4, w), hf = __builtin_bit_cast(f32x4, h);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if constexpr (KIND == K_F32) c = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[s], hf[s], c, 0, 0, 0);
            else c = __builtin_amdgcn_mfma_f64_16x16x4f64((double)wf[s], (double)hf[s], c, 0, 0, 0);
        }
        return c;
    }
}

// A lane's 16 bytes of a 64-byte step.  float32 takes element 4 s + (lane >> 4) for MFMA s (the chain is then ascending in k);
// the other types take chunk lane >> 4 as it lies.  `row` is the LDS row, `key` its chunk permutation, `step` the 64-byte step.
template <int KIND, int ROW_BYTES>
__device__ __forceinline__ i32x4 lds_frag(const char* base, int row, int key, int step) {
    const int q = (threadIdx.x & 63) >> 4;
    if constexpr (KIND == K_F32 || KIND == K_F32P) {
        i32x4 v;
#pragma unroll
        for (int s = 0; s < 4; ++s) v[s] = *reinterpret_cast<const int*>(base + row * ROW_BYTES + (((step * 4 + s) ^ key) << 4) + (q << 2));
        return v;
    } else {
        return *reinterpret_cast<const i32x4*>(base + row * ROW_BYTES + (((step * 4 + q) ^ key) << 4));
    }
}

// CH output columns n .. n + CH - 1 of row r: scales, bias, activation, one rounding.  `ws`, `bias`: those columns' values.
template <int KIND, class O, int CH>
__device__ __forceinline__ void finish(const ProductArgs& a, int64_t r, int n, const float (&v)[CH], float hs, const float (&ws)[CH],
                                       const float (&bias)[CH]) {
    using V = __attribute__((ext_vector_type(CH))) O;
    V o;
    float x[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) x[i] = KIND == K_I8 ? (v[i] * hs) * ws[i] : v[i];
    if (a.bias || a.act != DGCN_ACT_LINEAR) {
        const bool relu = a.act == DGCN_ACT_RELU;
        const float slope = a.act == DGCN_ACT_LEAKY_RELU ? kLeakyAlpha : 1.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            x[i] += bias[i];
            x[i] = x[i] <= 0.f ? (relu ? 0.f : x[i] * slope) : x[i];  // (NaN stays NaN)
        }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) o[i] = (O)x[i];
    O* y = reinterpret_cast<O*>(a.Y) + r * a.ldy + n;
    if (n + CH <= a.ctot) {
        if (sizeof(o) % 16 == 0 && a.stream) {
            i32x4 piece[sizeof(o) / 16 + (sizeof(o) < 16)];
            __builtin_memcpy(piece, &o, sizeof(o));
#pragma unroll
            for (int i = 0; i < (int)(sizeof(o) / 16); ++i) __builtin_nontemporal_store(piece[i], reinterpret_cast<i32x4*>(y) + i);
        } else {
            __builtin_memcpy(y, &o, sizeof(o));
        }
    } else {
#pragma unroll
        for (int i = 0; i < CH - 1; ++i)
            if (n + i < a.ctot) y[i] = o[i];
    }
}

__device__ const float g_minus_zero = -0.f;

// Scales and biases of the columns n .. n + CH - 1 of a model (the last column's again behind the end).  Without a bias -0 is added:
// it changes no value, +0 would turn -0 into +0.
template <int KIND, int CH>
__device__ __forceinline__ void column_values(const ProductArgs& a, int model, int n, float (&ws)[CH], float (&bias)[CH]) {
    const int64_t base = (int64_t)model * a.ctot;
    const float* b = a.bias ? a.bias + base : &g_minus_zero;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = min(n + i, a.ctot - 1);
        ws[i] = KIND == K_I8 ? a.ws[base + c] : 0.f;
        bias[i] = b[a.bias ? c : 0];
    }
}

// 16-bit results come in pairs of tiles where TN is even: a lane's columns of two tiles are neighbours and leave in one 16-byte store.
template <int TN, class O> constexpr bool kPairs = sizeof(O) == 2 && TN % 2 == 0;
template <int KIND, int TN> __device__ __forceinline__ bool in_pairs(const ProductArgs& a) {
    if constexpr (TN % 2 != 0 || KIND == K_F32 || KIND == K_F32P) return false;
    else if constexpr (KIND == K_I8) return a.out_dtype != DGCN_F32;
    else return true;
}
// The output column (within a wave's columns) that MFMA row i of tile j computes.  An MFMA leaves rows 4 q .. 4 q + 3 in lane group q
// (double: rows q, q + 4, ..): columns are dealt so that a lane group's 4 - in pairs of tiles 8 - are neighbours.
template <int KIND> __device__ __forceinline__ int w_row(int i, int j, bool pairs) {
    if constexpr (KIND == K_F32P) return j * 16 + 4 * (i & 3) + (i >> 2);
    else return pairs ? (j >> 1) * 32 + (i >> 2) * 8 + (j & 1) * 4 + (i & 3) : j * 16 + i;
}
// The chunk permutation of an LDS row: 16-byte reads - eight lanes in a row read eight different bank groups; dword reads - sixteen rows'
// dwords lie in sixty-four different banks.
template <int KIND> __device__ __forceinline__ int h_key(int row) { return KIND == K_F32 || KIND == K_F32P ? (row >> 1) & 7 : row & 7; }
template <int KIND> __device__ __forceinline__ int w_key(int row, bool pairs) { return pairs ? (row & 3) | ((row >> 1) & 4) : h_key<KIND>(row); }

// One wave's TM x TN tiles.
template <int KIND, class O, int TM, int TN>
__device__ __forceinline__ void write_tiles(const ProductArgs& a, const Tile& t, int row, int col, const typename Elem<KIND>::Acc (&acc)[TM][TN]) {
    constexpr int PW = kPairs<TN, O> ? 2 : 1, CH = 4 * PW;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    float hs[TM];
    if constexpr (KIND == K_I8) {
#pragma unroll
        for (int i = 0; i < TM; ++i) hs[i] = a.hs[t.row0 + (int64_t)min(row + i * 16 + (lane & 15), t.row1 - 1 - t.row0)];
    }
    float ws[TN / PW][CH], bias[TN / PW][CH];
#pragma unroll
    for (int p = 0; p < TN / PW; ++p) column_values<KIND, CH>(a, t.model, min(col + p * 16 * PW + q * CH, a.ctot - 1), ws[p], bias[p]);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t r = (int64_t)t.row0 + row + i * 16 + (lane & 15);
        if (r >= t.row1) continue;
#pragma unroll
        for (int p = 0; p < TN / PW; ++p) {  // (a row's columns one behind the other: its lines leave the caches whole)
            const int n = col + p * 16 * PW + q * CH;
            if (n >= a.ctot) continue;
            float v[CH];
#pragma unroll
            for (int x = 0; x < CH; ++x) v[x] = (float)acc[i][p * PW + (x >> 2)][x & 3];
            finish<KIND, O, CH>(a, r, n, v, KIND == K_I8 ? hs[i] : 0.f, ws[p], bias[p]);
        }
    }
}

// 16 bytes at byte offset `off` of a row of `row_bytes` bytes, any alignment; bytes behind the row's end are zero: a chunk that crosses
// the end is the row's last 16 bytes, shifted down.
__device__ __forceinline__ i32x4 load_chunk(const char* row, int64_t off, int64_t row_bytes) {
    unsigned long long u0 = 0, u1 = 0;
    int64_t over = off;  // how far the chunk lies behind what has been loaded
    if (row_bytes >= 16) {
        over = max(off - (row_bytes - 16), (int64_t)0);
        __builtin_memcpy(&u0, row + (off - over), 8);
        __builtin_memcpy(&u1, row + (off - over) + 8, 8);
    } else {
        for (int i = 0; i < (int)row_bytes; ++i) {
            const unsigned long long byte = (unsigned char)row[i];
            if (i < 8) u0 |= byte << (i * 8);
            else u1 |= byte << (i * 8 - 64);
        }
    }
    const int sh = (int)min(over, (int64_t)16) * 8;  // 0 .. 128
    const unsigned long long lo = sh >= 128 ? 0 : sh >= 64 ? u1 >> (sh - 64) : (u0 >> sh) | ((u1 << 1) << (63 - sh));
    const unsigned long long hi = sh >= 64 ? 0 : u1 >> sh;
    return i32x4{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}

// A row's last 16 bytes -> the chunk that starts `by` bytes behind their start (by <= 0: it is whole already): zeros move in.
__device__ __forceinline__ i32x4 shift_chunk(i32x4 v, int by) {
    by = min(max(by, 0), 16);
    const bool two = by & 8, one = by & 4;
    int a = two ? v[2] : v[0], b = two ? v[3] : v[1], c = two ? 0 : v[2], d = two ? 0 : v[3];
    a = one ? b : a; b = one ? c : b; c = one ? d : c; d = one ? 0 : d;
    if (by == 16) a = b = c = d = 0;
    return i32x4{(int)__builtin_amdgcn_alignbyte(b, a, by & 3), (int)__builtin_amdgcn_alignbyte(c, b, by & 3), (int)__builtin_amdgcn_alignbyte(d, c, by & 3),
                 (int)__builtin_amdgcn_alignbyte(0, d, by & 3)};
}

// load_chunk for a chunk that lies at least 16 bytes behind its row's start and ends at least 4 bytes in front of its end, in rows that
// start at any byte: five aligned dwords, shifted by the address' low bits.  (A 16-byte load from an address that is no multiple of 4
// takes several times as long.)
struct Dwords { i32x4 v; int v4; };
__device__ __forceinline__ Dwords load_dwords(const char* p) {
    const char* d = reinterpret_cast<const char*>(__builtin_assume_aligned(p - ((uintptr_t)p & 3), 4));
    Dwords r;
    __builtin_memcpy(&r.v, d, 16);
    __builtin_memcpy(&r.v4, d + 16, 4);
    return r;
}
__device__ __forceinline__ i32x4 shift_dwords(const Dwords& r, int by) {
    return i32x4{(int)__builtin_amdgcn_alignbyte(r.v[1], r.v[0], by), (int)__builtin_amdgcn_alignbyte(r.v[2], r.v[1], by),
                 (int)__builtin_amdgcn_alignbyte(r.v[3], r.v[2], by), (int)__builtin_amdgcn_alignbyte(r.v4, r.v[3], by)};
}

__device__ __attribute__((aligned(16))) const int g_zeros[4] = {0, 0, 0, 0};

// Every wave of the workgroup is here, with its LDS accesses (DIRECT: and all but the last LATER of its loads to LDS) done.
template <bool DIRECT, int LATER> __device__ __forceinline__ void arrive_all() {
    if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr int kCUs = 256;
constexpr int kRowBytes = 128;  // bytes of k per stage and row

// One output tile of BM rows x BN columns per workgroup, WM x WN waves.  128 bytes of k per stage, two LDS buffers: while the waves
// multiply out of one, the next stage travels into the other - DIRECT: by load-to-LDS instructions (rows of H and W at 16-byte
// strides, a tile's rows within 2 GB), otherwise through registers (any alignment, H == NULL).  An LDS row's eight 16-byte chunks are permuted by the row
// number, so that eight rows read at one k meet eight bank groups.
// Large products are bound by the matrix pipe and the LDS reads that feed it: int8 8 192 x 4 096 x 4 096 in 119 us (2.3 POP/s, as a large
// library product; pipe busy in 57 % of the cycles, 256 x 256 tiles), bf16 8 192 rows in 8 groups, 2 048 x 4 096 in 149 us (192 x 256).
// Narrow ones are a copy: 100 000 rows int8 128 -> 256 float32 in 24 us (115 MB, 64 x 64).
// A stage is worked off in phases (64 bytes of k x up to four row tiles).  AHEAD (every tile of eight waves, two per SIMD): a phase's
// fragments are requested behind the first MFMAs of the phase in front of it, across the stage's barrier too, so the matrix pipe
// does not wait for LDS; smaller tiles have more waves to hide that.  Row tiles behind the group's last row are skipped four at a time.
template <int KIND, int BM, int BN, int WM, int WN, int NBUF, bool DIRECT>
__device__ __forceinline__ void product_tile(const ProductArgs& a, int slots, int col_tiles, char* smem) {
    constexpr int T = WM * WN * 64, RB = kRowBytes, ES = Elem<KIND>::size;
    constexpr int TM = BM / WM / 16, TN = BN / WN / 16;       // 16 x 16 tiles per wave
    constexpr int NH = BM * 8 / T, NW = (BN * 8 + T - 1) / T;  // chunks per thread and stage
    static_assert(NH * T == BM * 8, "H chunks divide evenly");
    constexpr int RT = TM <= 4 ? TM : TM / 2, HALVES = TM / RT, PHASES = 2 * HALVES;
    static_assert(HALVES * RT == TM, "row tiles divide into phases");
    using Acc = typename Elem<KIND>::Acc;
    constexpr int BUF = (BM + BN) * RB;  // smem: two buffers (one if there is one stage) of [BM rows of H | BN rows of W]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    const int64_t kbytes = (int64_t)a.cin * ES;
    const int steps = (int)((kbytes + RB - 1) / RB);

    const Tile t = find_tile<BM>(a, (int)blockIdx.x, slots, col_tiles);
    if (t.row0 >= t.row1) return;
    const int n0 = t.col * BN;
    const char* Wm = a.W + (int64_t)t.model * a.ctot * kbytes;

    const bool pairs = in_pairs<KIND, TN>(a);
    // this thread's chunks: number c of the buffer lies at byte 16 c, row c / 8, and holds chunk (c % 8) ^ (row's key) of that row
    const char* src[DIRECT ? 1 : NH + NW];
    int at0[DIRECT ? NH + NW : 1];  // DIRECT: byte offset from the tile's first row
    int koff[NH + NW];
    const char* Ht = a.H + (int64_t)t.row0 * a.ldh * ES;
    const char* Wt = Wm + n0 * kbytes;
#pragma unroll
    for (int i = 0; i < NH + NW; ++i) {
        const bool is_h = i < NH;
        const int c = (is_h ? i : i - NH) * T + tid, row = c >> 3;
        koff[i] = ((c & 7) ^ (is_h ? h_key<KIND>(row) : w_key<KIND>(row, pairs))) << 4;
        const int last = is_h ? t.row1 - 1 - t.row0 : a.ctot - 1 - n0;
        const int64_t stride = is_h ? a.ldh * ES : kbytes;
        if constexpr (DIRECT) at0[i] = min(row, last) * (int)stride + koff[i];
        else src[i] = (is_h ? Ht : Wt) + min(row, last) * stride;
    }
    constexpr bool W_PART = NW * T != BN * 8;  // the last W chunk belongs to the first waves only
    i32x4 reg[DIRECT ? 1 : NH + NW];
    __amdgpu_buffer_rsrc_t rH, rW;
    if constexpr (DIRECT) {
        rH = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(Ht), 0, 0x7fffffff, 0x00020000);
        rW = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(Wt), 0, 0x7fffffff, 0x00020000);
    }
    auto fetch = [&](int st, int buf) {
        const bool whole = (int64_t)(st + 1) * RB <= kbytes;
        const int at = st * RB;
        if constexpr (DIRECT) {
            char* base = smem + buf * BUF + wave * 1024;
            if (whole) {
#pragma unroll
                for (int i = 0; i < NH + NW; ++i) {
                    if (W_PART && i == NH + NW - 1 && (i - NH) * T + wave * 64 >= BN * 8) continue;
                    char* d = base + (i < NH ? i * T : BM * 8 + (i - NH) * T) * 16;
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(i < NH ? rH : rW, (__attribute__((address_space(3))) void*)d, 16, at0[i], at, 0, 0);
                }
            } else {  // the rows' ends: chunks behind them come from a line of zeros
#pragma unroll
                for (int i = 0; i < NH + NW; ++i) {
                    if (W_PART && i == NH + NW - 1 && (i - NH) * T + wave * 64 >= BN * 8) continue;
                    const char* p = at + koff[i] < kbytes ? (i < NH ? Ht : Wt) + at0[i] + at : reinterpret_cast<const char*>(g_zeros);
                    char* d = base + (i < NH ? i * T : BM * 8 + (i - NH) * T) * 16;
                    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)d, 16, 0, 0);
                }
            }
        } else {
            auto no_h = [&](int i) { return (KIND == K_F32 || KIND == K_F32P) && i < NH && !a.H; };  // (there is no H: h_const)
#pragma unroll
            for (int i = 0; i < NH + NW; ++i) {
                if (W_PART && i == NH + NW - 1 && (i - NH) * T + wave * 64 >= BN * 8) continue;
                if (no_h(i)) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) reg[i][x] = at + koff[i] + 4 * x < kbytes ? __builtin_bit_cast(int, a.h_const) : 0;
                } else if (kbytes >= 16) {  // (the row's last 16 bytes for a chunk that crosses its end)
                    __builtin_memcpy(&reg[i], src[i] + (whole ? at + koff[i] : min(at + koff[i], (int)kbytes - 16)), 16);
                } else {
                    reg[i] = load_chunk(src[i], at + koff[i], kbytes);
                }
            }
            if (!whole && kbytes >= 16) {
#pragma unroll
                for (int i = 0; i < NH + NW; ++i)
                    if (!no_h(i)) reg[i] = shift_chunk(reg[i], at + koff[i] - ((int)kbytes - 16));
            }
        }
    };
    auto deposit = [&](int buf) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < NH + NW; ++i) {
                if (W_PART && i == NH + NW - 1 && (i - NH) * T + wave * 64 >= BN * 8) continue;
                const int c = (i < NH ? i * T : BM * 8 + (i - NH) * T) + tid;
                *reinterpret_cast<i32x4*>(smem + buf * BUF + c * 16) = reg[i];
            }
        }
    };

    Acc acc[TM][TN] = {};
    constexpr bool AHEAD = WM * WN == 8;
    i32x4 fh[AHEAD ? 2 : 1][RT], fw[AHEAD ? 2 : 1][TN];
    auto read_phase = [&](int buf, int p) {
        const char* sH = smem + buf * BUF;
        const char* sW = sH + BM * RB;
        const int k = p / HALVES, half = p % HALVES;
        if (half == 0) {
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int row = w_row<KIND>(lane & 15, j, pairs);
                fw[AHEAD ? k : 0][j] = lds_frag<KIND, RB>(sW, wn + row, w_key<KIND>(row, pairs), k);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) fh[AHEAD ? p & 1 : 0][i] = lds_frag<KIND, RB>(sH, wm + (half * RT + i) * 16 + (lane & 15), h_key<KIND>(lane & 15), k);
    };
    auto multiply_rows = [&](int p, int from, int to) {
        const int k = p / HALVES, half = p % HALVES;
#pragma unroll
        for (int i = from; i < to; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[half * RT + i][j] = mfma_step<KIND>(fw[AHEAD ? k : 0][j], fh[AHEAD ? p & 1 : 0][i], acc[half * RT + i][j]);
    };

    static_assert(DIRECT || NBUF == 2, "stages that travel through registers are fetched one ahead");
    static_assert(NBUF == 2 || !W_PART, "every wave has the same loads in flight");
    fetch(0, 0);
    if constexpr (DIRECT) {
        if (NBUF == 3 && steps > 1) {
            fetch(1, 1);
            arrive_all<DIRECT, NH + NW>();
        } else {
            arrive_all<DIRECT, 0>();
        }
        if (steps > NBUF - 1) fetch(NBUF - 1, NBUF - 1);
    } else {
        deposit(0);
        if (steps > 1) fetch(1, 1);
        arrive_all<DIRECT, 0>();
    }
    const int live = a.ctot - n0 <= wn ? 0 : min(HALVES, (t.row1 - t.row0 - wm + RT * 16 - 1) / (RT * 16));  // halves with rows
    auto run = [&](auto all) {
        constexpr bool ALL = decltype(all)::value;
        if (AHEAD && (ALL || live > 0)) read_phase(0, 0);
        int cur = 0;  // the buffer of stage st
        for (int st = 0; st < steps; ++st) {
            const int next = cur + 1 == NBUF ? 0 : cur + 1;
#pragma unroll
            for (int p = 0; p < PHASES; ++p) {
                const bool mine = ALL || p % HALVES < live, last = p + 1 == PHASES;
                if (mine) {
                    if (!AHEAD) read_phase(cur, p);
                    multiply_rows(p, 0, AHEAD ? 1 : RT);
                }
                if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
                if (!DIRECT && p == PHASES - 2 && st + 1 < steps) {
                    // (everyone left the buffer of stage st - 1 at the last barrier; a phase is left to hide these writes behind)
                    deposit(next);
                    if (st + 2 < steps) fetch(st + 2, cur);
                }
                if (last && st + 1 < steps) {
                    // stage st + 1 lies in its buffer, everyone has read all of stage st
                    if (NBUF == 3 && st + 2 < steps) arrive_all<DIRECT, NH + NW>();
                    else arrive_all<DIRECT, 0>();
                    if (DIRECT && st + NBUF < steps) fetch(st + NBUF, cur);
                }
                if constexpr (AHEAD) {
                    if (!last ? ALL || (p + 1) % HALVES < live : st + 1 < steps && (ALL || live > 0))
                        read_phase(last ? next : cur, last ? 0 : p + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_setprio(1);
                    if (mine) multiply_rows(p, 1, RT);
                    __builtin_amdgcn_s_setprio(0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            cur = next;
        }
    };
    if (live == HALVES) run(std::true_type{});
    else run(std::false_type{});
    if (live <= 0) return;
    if constexpr (KIND == K_BF16) write_tiles<KIND, __bf16, TM, TN>(a, t, wm, n0 + wn, acc);
    else if constexpr (KIND == K_F16) write_tiles<KIND, _Float16, TM, TN>(a, t, wm, n0 + wn, acc);
    else if constexpr (KIND != K_I8) write_tiles<KIND, float, TM, TN>(a, t, wm, n0 + wn, acc);
    else if (a.out_dtype == DGCN_BF16) write_tiles<KIND, __bf16, TM, TN>(a, t, wm, n0 + wn, acc);
    else if (a.out_dtype == DGCN_F16) write_tiles<KIND, _Float16, TM, TN>(a, t, wm, n0 + wn, acc);
    else write_tiles<KIND, float, TM, TN>(a, t, wm, n0 + wn, acc);
}

// (Stages through registers: five waves per SIMD for the small tiles, not the four that the compiler would choose - short rows are latency:
// 79 002 rows, bf16 30 -> 380 in 378 groups 47 -> 36 us, 100 000 rows int8 127 -> 256 float32 36 -> 30.)
template <int KIND, int BM, int BN, int WM, int WN, int NBUF, bool DIRECT>
__global__ __launch_bounds__(WM* WN * 64, !DIRECT && WM * WN == 4 && BN == 64 && KIND != K_F32P ? 5 : 1) void k_product(ProductArgs a, int slots, int col_tiles) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    product_tile<KIND, BM, BN, WM, WN, NBUF, DIRECT>(a, slots, col_tiles, smem);
}

// Few rows per group: the weights' bytes are the cost.  A workgroup takes 16 rows x 16 NT columns; its waves share the k range in
// interleaved pieces of 128 bytes, read their fragments straight from memory (every weight is used once: LDS would only be a
// detour) and join their sums through LDS in a fixed order.  24 rows in 64 groups, fp16 2 048 x 1 024: 21 us for 97 MB of weights; 5 rows,
// int8 4 096 x 4 096: 6.7 us for 17 MB, most of it one load's and one launch's latency.
template <int KIND, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void k_product_few(ProductArgs a, int slots, int col_tiles) {
    constexpr int ES = Elem<KIND>::size, BM = 16, BN = 16 * NT;
    using Acc = typename Elem<KIND>::Acc;
    __shared__ __attribute__((aligned(16))) Acc part[WAVES][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
    const int64_t kbytes = (int64_t)a.cin * ES;
    const Tile t = find_tile<BM>(a, (int)blockIdx.x, slots, col_tiles);
    if (t.row0 >= t.row1) return;
    const int n0 = t.col * BN;
    const char* h = a.H + (t.row0 + (int64_t)min(lane & 15, t.row1 - 1 - t.row0)) * a.ldh * ES;
    const char* w[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
        w[j] = a.W + ((int64_t)t.model * a.ctot + n0 + min(j * 16 + (lane & 15), a.ctot - 1 - n0)) * kbytes;
    Acc acc[NT] = {};
    const int pieces = (int)((kbytes + 127) >> 7);
    // whole pieces; where rows of W start anywhere, those that are neither first nor last
    const int from = a.dwords_w ? 0 : 1, to = (int)((a.dwords_w ? kbytes : kbytes - 4) >> 7);
    constexpr int U = NT >= 4 ? 2 : 4;
    int c = wave;
    auto checked = [&](int c) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int64_t off = (int64_t)c * 128 + e * 64 + q * 16;
            const i32x4 fh = load_chunk(h, off, kbytes);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j] = mfma_step<KIND>(load_chunk(w[j], off, kbytes), fh, acc[j]);
        }
    };
    auto whole = [&](auto dwords_w, int c, auto count) {
        constexpr bool DW = decltype(dwords_w)::value;
        constexpr int N = decltype(count)::value;
        i32x4 fh[N][2], fw[N][2][NT];
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int64_t off = (int64_t)(c + u * WAVES) * 128 + e * 64 + q * 16;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (DW) __builtin_memcpy(&fw[u][e][j], w[j] + off, 16);
                    else fw[u][e][j] = shift_dwords(load_dwords(w[j] + off), (int)(uintptr_t)w[j] & 3);
                }
                if constexpr (DW) __builtin_memcpy(&fh[u][e], h + off, 16);
                else fh[u][e] = shift_dwords(load_dwords(h + off), (int)(uintptr_t)h & 3);
            }
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j] = mfma_step<KIND>(fw[u][e][j], fh[u][e], acc[j]);
    };
    if (c < from && c < pieces) {
        checked(c);
        c += WAVES;
    }
    auto middle = [&](auto dwords_w) {
        for (; c + (U - 1) * WAVES < to; c += U * WAVES) whole(dwords_w, c, std::integral_constant<int, U>{});
        for (; c < to; c += WAVES) whole(dwords_w, c, std::integral_constant<int, 1>{});
    };
    if (a.dwords_w) middle(std::true_type{});
    else middle(std::false_type{});
    if (c < pieces) checked(c);  // (one of at most two last pieces)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    for (int x = threadIdx.x; x < NT * 64; x += WAVES * 64) {
        const int j = x >> 6, l = x & 63;
        Acc sum = part[0][j][l];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum += part[v][j][l];
        const int64_t r = (int64_t)t.row0 + (l & 15);
        const int n = n0 + j * 16 + 4 * (l >> 4);
        if (r >= t.row1 || n >= a.ctot) continue;
        float ws[4], bias[4], v[4];
        column_values<KIND, 4>(a, t.model, n, ws, bias);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)sum[i];
        const float hs = KIND == K_I8 ? a.hs[r] : 0.f;
        if constexpr (KIND == K_BF16) finish<KIND, __bf16, 4>(a, r, n, v, hs, ws, bias);
        else if constexpr (KIND == K_F16) finish<KIND, _Float16, 4>(a, r, n, v, hs, ws, bias);
        else if (a.out_dtype == DGCN_BF16) finish<KIND, __bf16, 4>(a, r, n, v, hs, ws, bias);
        else if (a.out_dtype == DGCN_F16) finish<KIND, _Float16, 4>(a, r, n, v, hs, ws, bias);
        else finish<KIND, float, 4>(a, r, n, v, hs, ws, bias);
    }
}

// Many rows of a narrow layer (rows of at most KS x 64 bytes, whole 16-byte chunks; at most 16 TN columns): memory-bound, so no LDS and
// no barrier.  Every wave walks a contiguous run of rows in windows of 16 whose loads need no knowledge of the groups and are in flight
// one window ahead; the weights of the group it is in are MFMA fragments in registers.  A window that several groups share is multiplied
// once for each and stored row by row.  800 000 rows of 32 float32 -> 2 in 4 000 groups: 27.5 us for 109 MB.
//
// A lane's 16 bytes of H hold float32 elements 4 q .. 4 q + 3 (q = lane >> 4), the ascending chain needs element 4 s + q in MFMA s: a
// 4 x 4 transpose between the four lane groups and the four registers, in four lane-swap instructions.
template <int KIND> __device__ __forceinline__ i32x4 chain_order(i32x4 v) {
    if constexpr (KIND == K_F32) {
        auto a = __builtin_amdgcn_permlane32_swap((unsigned)v[0], (unsigned)v[2], false, false);
        auto b = __builtin_amdgcn_permlane32_swap((unsigned)v[1], (unsigned)v[3], false, false);
        auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
        auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
        return i32x4{(int)c[0], (int)c[1], (int)d[0], (int)d[1]};
    } else {
        return v;
    }
}

template <int KIND, class O, int TN, int KS>
__device__ __forceinline__ void product_rows(const ProductArgs& a, int run) {
    constexpr int ES = Elem<KIND>::size;
    using Acc = typename Elem<KIND>::Acc;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int64_t kbytes = (int64_t)a.cin * ES;
    const int64_t gw = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto clamp = [&](int p) { return min(max(p, 0), a.rows); };
    if (a.gptr) {  // every table entry is checked by one thread
        for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < a.num_groups; g += (int64_t)gridDim.x * 256)
            if (bad_group(a, a.gptr[g], a.gptr[g + 1], a.mog ? a.mog[g] : (int)g)) atomicOr(a.status, (int)DGCN_FAULT_BAD_GROUP);
    }
    int64_t r = gw * run;  // the next row to compute
    const int64_t end = min(r + run, (int64_t)a.rows);
    if (r >= end) return;
    auto load_h = [&](int64_t window, i32x4 (&h)[KS]) {
        const char* row = a.H + min(window + (lane & 15), (int64_t)a.rows - 1) * a.ldh * ES;
#pragma unroll
        for (int e = 0; e < KS; ++e) {
            h[e] = i32x4{0, 0, 0, 0};
            if (e * 64 + q * 16 < kbytes) __builtin_memcpy(&h[e], row + e * 64 + q * 16, 16);
        }
    };
    int64_t p0 = 0, p1 = 0;  // the group of row r (none yet)
    int e = -1, model = -1;
    auto find_group = [&]() {  // the last group that starts at or in front of row r
        if (!a.gptr) { p1 = a.rows; e = 0; return; }
        int lo = 0, n = a.num_groups;
        while (n > 64) {
            const int step = (n + 63) >> 6;
            const int64_t i = (int64_t)lane * step;
            const unsigned long long m = __ballot(i < n && clamp(a.gptr[lo + (i < n ? (int)i : 0)]) <= r);
            const int k = max(m == ~0ull ? 64 : (int)__builtin_ctzll(~m), 1);
            lo += (k - 1) * step;
            n = min(step, n - (k - 1) * step);
        }
        const int g = lo + min(lane, n - 1);
        const int q0 = clamp(a.gptr[g]), q1 = clamp(a.gptr[g + 1]), qe = a.mog ? a.mog[g] : g;
        const unsigned long long m = __ballot(lane < n && q0 <= r);
        const int at = __builtin_amdgcn_readfirstlane(max(m == ~0ull ? 64 : (int)__builtin_ctzll(~m), 1) - 1);
        p0 = __builtin_amdgcn_readlane(q0, at);
        p1 = __builtin_amdgcn_readlane(q1, at);
        e = __builtin_amdgcn_readlane(qe, at);
        if (r < p0) {  // in front of the first group: rows of no group up to it
            p1 = p0;
            e = -1;
        } else if (r >= p1) {  // behind the last one; in a table that decreases, on by a step
            p1 = lo + at + 1 == a.num_groups ? end : min(r + 16, end);
            e = -1;
        }
    };
    i32x4 w[TN][KS];
    float ws[TN][4], bias[TN][4];
    i32x4 h[KS], ahead[KS];
    load_h(r, h);
    for (int64_t window = r; window < end; window += 16) {
        const int64_t wend = min(window + 16, end);
        if (wend < end) load_h(wend, ahead);
        i32x4 hk[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) hk[k] = chain_order<KIND>(h[k]);
        while (r < wend) {
            if (r >= p1) find_group();
            const int64_t stop = min(p1, wend);
            if (e >= 0 && e < a.num_models) {
                if (e != model) {
                    model = e;
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        const char* row = a.W + ((int64_t)e * a.ctot + min(w_row<KIND>(lane & 15, j, kPairs<TN, O>), a.ctot - 1)) * kbytes;
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            w[j][k] = i32x4{0, 0, 0, 0};
                            if (k * 64 + q * 16 < kbytes) __builtin_memcpy(&w[j][k], row + k * 64 + q * 16, 16);
                            w[j][k] = chain_order<KIND>(w[j][k]);
                        }
                        column_values<KIND, 4>(a, e, min(w_row<KIND>(4 * q, j, kPairs<TN, O>), a.ctot - 1), ws[j], bias[j]);
                    }
                }
                Acc acc[TN] = {};
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[j] = mfma_step<KIND>(w[j][k], hk[k], acc[j]);
                const int64_t row = window + (lane & 15);
                if (row >= r && row < stop) {
                    const float hs = KIND == K_I8 ? a.hs[row] : 0.f;
                    constexpr int PW = kPairs<TN, O> ? 2 : 1, CH = 4 * PW;
#pragma unroll
                    for (int p = 0; p < TN / PW; ++p) {
                        const int n = p * 16 * PW + q * CH;
                        float v[CH], s[CH], b[CH];
#pragma unroll
                        for (int x = 0; x < CH; ++x) {
                            v[x] = (float)acc[p * PW + (x >> 2)][x & 3];
                            s[x] = ws[p * PW + (x >> 2)][x & 3];
                            b[x] = bias[p * PW + (x >> 2)][x & 3];
                        }
                        if (n < a.ctot) finish<KIND, O, CH>(a, row, n, v, hs, s, b);
                    }
                }
            }
            r = stop;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) h[k] = ahead[k];
    }
}

template <int KIND, class O, int TN, int KS>
__global__ __launch_bounds__(256) void k_product_rows(ProductArgs a, int run) { product_rows<KIND, O, TN, KS>(a, run); }

static int64_t row_slots(const ProductArgs& a, int BM) {
    if (!a.gptr) return ((int64_t)a.rows + BM - 1) / BM;
    const int64_t n = (int64_t)a.rows / BM + a.num_groups;
    return a.counted ? min(n, (int64_t)a.rows) : n;  // (a counted tile holds at least one row)
}
constexpr int64_t max_grid(int threads) { return 0xffffffffu / (unsigned)threads; }  // a launch's threads are counted in 32 bits

template <int KIND, int BM, int BN, int WM, int WN, int NBUF, bool DIRECT>
static int launch_tiles_as(const char* family, const ProductArgs& a, hipStream_t s) {
    const int64_t slots = row_slots(a, BM);
    const int col_tiles = (a.ctot + BN - 1) / BN;
    if (slots * col_tiles > max_grid(WM * WN * 64)) return fail(DGCN_ERR_UNSUPPORTED, "%s: %lld tiles in one call", family, (long long)(slots * col_tiles));
    const int lds = (int)min(((int64_t)a.cin * Elem<KIND>::size - 1) / kRowBytes + 1, (int64_t)NBUF) * (BM + BN) * kRowBytes;
    if (lds > 64 * 1024) {
        static std::atomic<int> reserved[64];
        int dev = 0;
        (void)hipGetDevice(&dev);
        if (!reserved[dev & 63].load(std::memory_order_relaxed)) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(&k_product<KIND, BM, BN, WM, WN, NBUF, DIRECT>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, NBUF * (BM + BN) * kRowBytes) != hipSuccess)
                return fail(DGCN_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS", family, lds);
            reserved[dev & 63].store(1, std::memory_order_relaxed);
        }
    }
    TimedLaunch t(family, s);
    DGCN_LAUNCH(t, (k_product<KIND, BM, BN, WM, WN, NBUF, DIRECT>), dim3((unsigned)(slots * col_tiles)), dim3(WM * WN * 64), lds, s, a, (int)slots, col_tiles);
    return check_launch("k_product");
}

// Load-to-LDS instructions take rows at 16-byte strides; a tile's offsets are 31 bits.
template <int KIND> static bool direct_loads(const ProductArgs& a) {
    constexpr int64_t ES = Elem<KIND>::size;
    return a.H && ((uintptr_t)a.H | (uintptr_t)a.W) % 16 == 0 && a.ldh * ES % 16 == 0 && a.cin * ES % 16 == 0 && a.ldh * ES * 256 < 0x7fffffff &&
           a.cin * ES * 256 < 0x7fffffff;
}

template <int KIND, int BM, int BN, int WM, int WN, int NBUF>
static int launch_tiles(const char* family, const ProductArgs& a, hipStream_t s) {
    if (direct_loads<KIND>(a)) return launch_tiles_as<KIND, BM, BN, WM, WN, NBUF, true>(family, a, s);
    return launch_tiles_as<KIND, BM, BN, WM, WN, 2, false>(family, a, s);
}

template <int KIND, int NT, int WAVES> static int launch_few(const char* family, const ProductArgs& a, hipStream_t s) {
    const int64_t slots = row_slots(a, 16);
    const int col_tiles = (a.ctot + 16 * NT - 1) / (16 * NT);
    if (slots * col_tiles > max_grid(WAVES * 64)) return fail(DGCN_ERR_UNSUPPORTED, "%s: %lld tiles in one call", family, (long long)(slots * col_tiles));
    TimedLaunch t(family, s);
    DGCN_LAUNCH(t, (k_product_few<KIND, NT, WAVES>), dim3((unsigned)(slots * col_tiles)), dim3(WAVES * 64), 0, s, a, (int)slots, col_tiles);
    return check_launch("k_product_few");
}

template <int KIND, class O, int TN, int KS> static int launch_rows_as(const char* family, const ProductArgs& a, hipStream_t s) {
    constexpr int waves = kCUs * 24;
    const int64_t tiles = ((int64_t)a.rows + 15) / 16;
    const int run = (int)((tiles + waves - 1) / waves) * 16;
    const int64_t blocks = ((int64_t)a.rows + 4 * (int64_t)run - 1) / (4 * (int64_t)run);
    TimedLaunch t(family, s);
    DGCN_LAUNCH(t, (k_product_rows<KIND, O, TN, KS>), dim3((unsigned)blocks), dim3(256), 0, s, a, run);
    return check_launch("k_product_rows");
}
template <int KIND, int TN, int KS> static int launch_rows(const char* family, const ProductArgs& a, hipStream_t s) {
    if constexpr (KIND == K_F32) return launch_rows_as<KIND, float, TN, KS>(family, a, s);
    else if constexpr (KIND == K_BF16) return launch_rows_as<KIND, __bf16, TN, KS>(family, a, s);
    else if constexpr (KIND == K_F16) return launch_rows_as<KIND, _Float16, TN, KS>(family, a, s);
    else if (a.out_dtype == DGCN_F32) return launch_rows_as<KIND, float, TN, KS>(family, a, s);
    else if (a.out_dtype == DGCN_BF16) return launch_rows_as<KIND, __bf16, TN, KS>(family, a, s);
    else return launch_rows_as<KIND, _Float16, TN, KS>(family, a, s);
}

// What a call launches: kernels by number, tile kernels with DIRECT.
enum Path {
    P_64_64, P_128_128, P_128_256, P_192_256, P_256_256,  // k_product, 8- and 16-bit types' shapes (in kDirect's order); P_64_64 and P_128_128 float32 too
    P_128_16, P_128_32, P_32_64,                          // k_product, float32
    P_FEW_2_4, P_FEW_1_8, P_FEW_1_4,                      // k_product_few<NT, WAVES>
    P_ROWS_16, P_ROWS_32,                                 // k_product_rows, up to 16 / 32 columns
};

// The tile shapes of the 8- and 16-bit products and what they cost, fitted to shapes of 128 .. 100 000 rows, k of 64 .. 4 096 bytes and
// 20 .. 4 096 columns, dense and in 8 .. 300 groups: a stage (128 bytes of k) takes s1 us in a workgroup that has its CU to itself and sc
// us with per_cu of them there, a tile's start and end f us.  The choice is the fastest shape or within 11 % of it on 32 of 36 calls
// (profiles/products_shapes.txt: every shape's time beside its estimate).  The others lose up to 40 %: the host knows how many tiles to
// expect, not how many there are, and two more than a full round of workgroups are another round (16 000 rows of 2 048 bytes in 8 groups,
// 512 columns: 39.5 us with 128 x 256, 28.2 with 192 x 256).
struct Shape { int bm, bn, per_cu; float s1, sc, f; };
constexpr int kShapes = 5;
constexpr float kBytesPerUs = 4.7e6f;  // a large copy, read and written
constexpr Shape kDirect[kShapes] = {{64, 64, 5, .55f, 1.11f, 2.f}, {128, 128, 2, .78f, 1.05f, 3.f}, {128, 256, 1, .98f, .98f, 4.f},
                                    {192, 256, 1, 1.36f, 1.36f, 5.f}, {256, 256, 1, 1.8f, 1.8f, 6.f}};
constexpr Shape kStaged[kShapes] = {{64, 64, 4, .85f, 1.6f, 2.f}, {128, 128, 1, 1.23f, 1.23f, 3.f}, {128, 256, 1, 1.7f, 1.7f, 4.f},
                                    {192, 256, 1, 2.05f, 2.05f, 5.f}, {0, 0, 0, 0.f, 0.f, 0.f}};

// Row tiles a launch is expected to have: the host knows rows and groups, not the groups' sizes.
static float expected_slots(const ProductArgs& a, int BM) {
    if (!a.gptr || a.num_groups == 1) return (float)(((int64_t)a.rows + BM - 1) / BM);
    return (float)a.rows / BM + .5f * min(a.num_groups, a.rows);
}

// Bytes of a call: every model's weights once, every row in and out.
static float weight_bytes(const ProductArgs& a, int64_t row_bytes) { return (float)(a.gptr ? min(a.num_groups, a.rows) : 1) * a.ctot * row_bytes; }
static float out_bytes(const ProductArgs& a) { return (float)a.rows * (a.out_dtype == DGCN_F32 ? 4.f : 2.f) * a.ctot; }

// A call that takes about as long as its bytes do (`compute_us`: without them) and whose bytes are mostly Y stores it past the caches, in
// whole 64-byte sectors (rows of 4 000 bytes, which are not, take twice as long that way): 100 000 rows, int8 128 -> 256 float32 24 us
// against 40 with outputs that the caches do not already hold; the six layers of a 128-wide 8-bit bank over 500 graphs 571 us against
// 588, aggregations included.  Calls that compute for longer lose by it (fp32 128 -> 256: 1 %), and a small Y is better left in the caches for
// the call that reads it (six layers of a float32 bank, aggregations included: 72.4 us against 75.7 with 1.0 MB per layer, 81.0 against
// 81.6 with 2.6; 97.2 against 95.0 with 5.1, 178 against 170 with 20).
constexpr float kStreamsFrom = 4e6f;
static bool streams_out(const ProductArgs& a, int64_t row_bytes, float compute_us) {
    const int os = a.out_dtype == DGCN_F32 ? 4 : 2;
    const float out = out_bytes(a), all = out + weight_bytes(a, row_bytes) + (float)a.rows * row_bytes;
    return out > kStreamsFrom && all / kBytesPerUs > .75f * compute_us && out > .5f * all && a.ldy * os % 64 == 0 && (uintptr_t)a.Y % 64 == 0;
}

static int choose_shape(ProductArgs& a, int64_t row_bytes, bool direct) {
    const Shape* shapes = direct ? kDirect : kStaged;
    const float steps = (float)((row_bytes + kRowBytes - 1) / kRowBytes);
    int best = 0;
    float least = INFINITY;
    for (int i = 0; i < kShapes; ++i) {
        const Shape& p = shapes[i];
        if (!p.bm) continue;
        const float per = expected_slots(a, p.bm) * (float)((a.ctot + p.bn - 1) / p.bn) / kCUs;  // tiles per CU
        const float rounds = floorf(per / p.per_cu), rest = per - rounds * p.per_cu;
        float cost = rounds * (p.sc * steps + p.f);  // (the expected count is a mean: up to .02 tiles per CU behind a round are left out)
        if (rest > .02f || rounds == 0.f) cost += (p.s1 + (p.per_cu > 1 ? (p.sc - p.s1) * (ceilf(rest) - 1.f) / (p.per_cu - 1) : 0.f)) * steps + p.f;
        if (cost < least) { least = cost; best = i; }
    }
    // Where the bytes alone take longer than that, a copy's many small workgroups are best (100 000 rows, int8 127 -> 256: 33 us with 64 x 64
    // when the larger ones took 41 .. 50; 128 -> 256, Y past the caches: 24 against 31 .. 42) - unless nearly all of the bytes are weights of
    // groups with few rows, which 128 x 128 reads more seldom (64 groups, 2 048 rows, 2 048 bytes x 1 024 columns: 28 us against 37).
    a.stream = streams_out(a, row_bytes, least);
    const float weights = weight_bytes(a, row_bytes), others = (float)a.rows * row_bytes + out_bytes(a);
    if (a.stream || (weights + others) / kBytesPerUs > least) best = direct && a.gptr && weights > 4.f * others ? 1 : 0;
    return best;
}

// The kernel of a call; sets a.stream.
template <int KIND> static int choose_path(ProductArgs& a) {
    const int64_t row_bytes = (int64_t)a.cin * Elem<KIND>::size;
    if constexpr (KIND == K_F32P) {
        return P_64_64;
    } else {
        // a narrow layer over very many rows: no tile would be more than a copy (800 000 rows of 32 float32 -> 2: 28 us against 32 of the
        // 128 x 16 tile; 300 000 rows of 32 bf16 -> 32: 12 against 19 of 64 x 64; at 60 000 rows no difference)
        if (a.H && a.dwords_h && a.dwords_w && row_bytes % 16 == 0 && row_bytes <= 128 && a.ctot <= 32 && a.rows >= 1 << 17)
            return a.ctot <= 16 ? P_ROWS_16 : P_ROWS_32;
    }
    const int groups = min(a.num_groups, a.rows);
    if constexpr (KIND == K_F32) {
        a.stream = streams_out(a, row_bytes, (float)a.rows * a.ctot * a.cin * 2.f / 149e6f);
        // float32: the matrix pipe is the bound from some 64 columns on, so the shape matters little but for its waste.  128 x 128 (1 024
        // x 1 024, 8 192 rows: 144 us against 165) where its tiles fill whole rounds of two per CU; 64 x 64 where a row is one stage (32
        // -> 64, 500 graphs: 16.4 against 19.4 of 32 x 64), else 32 x 64 (128 -> 256: 96 against 101; 200 rows in 10 groups: 12 against 15).
        const float rounds = expected_slots(a, 128) * (float)((a.ctot + 127) / 128) / (2 * kCUs);
        if (a.ctot <= 16) return P_128_16;
        if (a.ctot <= 32 && row_bytes > 128) return P_128_32;
        if (groups == 1 && row_bytes >= 1024 && rounds > .9f * ceilf(rounds)) return P_128_128;
        return row_bytes <= 128 && a.rows / groups >= 48 ? P_64_64 : P_32_64;
    } else if constexpr (KIND != K_F32P) {
        // few rows in every group, long rows and not enough tiles to fill the chip: split k over a workgroup's waves (1 row, 4 096 x
        // 4 096 int8: 6 us against 17 of the 64 x 64 tile; 64 rows: 15 against 19; 24 rows in 64 groups, fp16 2 048 x 1 024: 23 against 29)
        const int64_t tiles = (a.gptr ? (int64_t)groups : (a.rows + 63) / 64) * ((a.ctot + 63) / 64);
        if (row_bytes >= 512 && a.rows <= (a.gptr ? 16 * (int64_t)groups : 64) && tiles < 2 * kCUs) {
            if constexpr (KIND == K_I8)  // (the other types' entry point is the grouped one)
                if (!a.gptr && a.rows <= 16) return row_bytes >= 2048 ? P_FEW_1_8 : P_FEW_1_4;
            return P_FEW_2_4;
        }
        return choose_shape(a, row_bytes, direct_loads<KIND>(a));
    }
}

template <int KIND> static int launch_path(int path, const char* family, const ProductArgs& a, hipStream_t s) {
    if constexpr (KIND == K_F32P) {
        return launch_tiles<KIND, 64, 64, 2, 2, 2>(family, a, s);
    } else {
        if (path == P_ROWS_16) return launch_rows<KIND, 1, 2>(family, a, s);
        if (path == P_ROWS_32) return launch_rows<KIND, 2, 2>(family, a, s);
        if (path == P_64_64) return launch_tiles<KIND, 64, 64, 2, 2, 2>(family, a, s);
        if (path == P_128_128) return launch_tiles<KIND, 128, 128, 2, 4, 2>(family, a, s);
        if constexpr (KIND == K_F32) {
            if (path == P_128_16) return launch_tiles<KIND, 128, 16, 4, 1, 2>(family, a, s);
            if (path == P_128_32) return launch_tiles<KIND, 128, 32, 4, 1, 2>(family, a, s);
            return launch_tiles<KIND, 32, 64, 1, 4, 2>(family, a, s);
        } else {
            if (path == P_FEW_2_4) return launch_few<KIND, 2, 4>(family, a, s);
            if constexpr (KIND == K_I8) {
                if (path == P_FEW_1_8) return launch_few<KIND, 1, 8>(family, a, s);
                if (path == P_FEW_1_4) return launch_few<KIND, 1, 4>(family, a, s);
            }
            if (path == P_128_256) return launch_tiles<KIND, 128, 256, 2, 4, 3>(family, a, s);
            if (path == P_192_256) return launch_tiles<KIND, 192, 256, 2, 4, 2>(family, a, s);
            return launch_tiles_as<KIND, 256, 256, 2, 4, 2, true>(family, a, s);
        }
    }
}

static void prepare_args(int kind, ProductArgs& a) {
    const int es = kind == K_I8 ? 1 : kind == K_BF16 || kind == K_F16 ? 2 : 4;
    // Counting pays where a tile is long (16 000 rows of 1 024 bytes in 64 groups, 512 columns, int8: 20 us, searching 31; of 4 096 bytes 58
    // against 91); in short ones its loads are a part of the time (40 000 rows of 128 bytes in 8 groups: 20 against 17; in 250: 29 against 25).
    a.counted = a.gptr && a.num_groups <= kCountedGroups && (int64_t)a.cin * es > 256;
    a.dwords_h = (uintptr_t)a.H % 4 == 0 && a.ldh * es % 4 == 0;
    a.dwords_w = (uintptr_t)a.W % 4 == 0 && (int64_t)a.cin * es % 4 == 0;
}

template <class F> static int with_kind(int kind, F f) {
    switch (kind) {
        case K_I8: return f(std::integral_constant<int, K_I8>{});
        case K_BF16: return f(std::integral_constant<int, K_BF16>{});
        case K_F16: return f(std::integral_constant<int, K_F16>{});
        case K_F32: return f(std::integral_constant<int, K_F32>{});
        default: return f(std::integral_constant<int, K_F32P>{});
    }
}

static int product_dispatch(const char* family, int kind, ProductArgs& a, hipStream_t s) {
    prepare_args(kind, a);
    return with_kind(kind, [&](auto k) {
        constexpr int KIND = decltype(k)::value;
        return launch_path<KIND>(choose_path<KIND>(a), family, a, s);
    });
}

static bool known_dtype(int32_t d) { return d == DGCN_F32 || d == DGCN_BF16 || d == DGCN_F16; }
static bool known_act(int32_t a) { return a == DGCN_ACT_LINEAR || a == DGCN_ACT_LEAKY_RELU || a == DGCN_ACT_RELU; }
constexpr int kMaxExtent = 0x7fffffff - 1023;  // tile corners, and offsets within a row, stay within 32 bits
constexpr int kMaxInt8Depth = 131071;  // 128 * 128 * cin stays below 2^31

static int check_sizes(const char* who, int32_t rows, int32_t cin, int32_t ctot, int size, bool has_h, int64_t ldh, int64_t ldy, int32_t act) {
    if (rows < 0 || cin <= 0 || ctot <= 0 || (has_h && ldh < cin) || ldy < ctot) return fail(DGCN_ERR_ARG, "%s: bad sizes", who);
    if (!known_act(act)) return fail(DGCN_ERR_ARG, "%s: unknown activation %d", who, act);
    if (rows > kMaxExtent || ctot > kMaxExtent) return fail(DGCN_ERR_UNSUPPORTED, "%s: more than %d rows or columns", who, kMaxExtent);
    if ((int64_t)cin * size > kMaxExtent) return fail(DGCN_ERR_UNSUPPORTED, "%s: rows of more than %d bytes", who, kMaxExtent);
    return DGCN_OK;
}

static int product_int8(const char* who, const char* family, ProductArgs& a, hipStream_t s) {
    int rc = check_sizes(who, a.rows, a.cin, a.ctot, 1, true, a.ldh, a.ldy, a.act);
    if (rc) return rc;
    if (!known_dtype(a.out_dtype)) return fail(DGCN_ERR_ARG, "%s: unknown dtype %d", who, a.out_dtype);
    if (a.cin > kMaxInt8Depth) return fail(DGCN_ERR_UNSUPPORTED, "%s: cin %d > %d: the int32 sums could overflow", who, a.cin, kMaxInt8Depth);
    if (a.num_groups < 0 || a.num_models <= 0) return fail(DGCN_ERR_ARG, "%s: bad sizes", who);
    if (a.rows == 0 || a.num_groups == 0) return DGCN_OK;
    if (!a.H || !a.hs || !a.W || !a.ws || !a.Y) return fail(DGCN_ERR_ARG, "%s: null argument", who);
    return product_dispatch(family, K_I8, a, s);
}

}  // namespace dgcn

using namespace dgcn;

extern "C" int dgcn_transform_int8_batch(const int8_t* H, int64_t ldh, const float* h_scale, int32_t rows, int32_t cin, const int8_t* W,
                                         const float* w_scale, int32_t ctot, const float* bias, int32_t act, void* Y, int32_t out_dtype,
                                         int64_t ldy, void* stream) {
    ProductArgs a{};
    a.H = (const char*)H; a.ldh = ldh; a.hs = h_scale; a.rows = rows; a.cin = cin; a.W = (const char*)W; a.ws = w_scale; a.ctot = ctot;
    a.bias = bias; a.act = act; a.Y = Y; a.out_dtype = out_dtype; a.ldy = ldy; a.num_groups = 1; a.num_models = 1;
    return product_int8("dgcn_transform_int8_batch", "transform_int8", a, (hipStream_t)stream);
}

extern "C" int dgcn_transform_grouped_int8_batch(const int8_t* H, int64_t ldh, const float* h_scale, int32_t rows, int32_t cin,
                                                 const int32_t* group_ptr, const int32_t* model_of_group, int32_t num_groups, const int8_t* W,
                                                 const float* w_scale, int32_t num_models, int32_t ctot, const float* bias, int32_t act,
                                                 void* Y, int32_t out_dtype, int64_t ldy, int32_t* status, void* stream) {
    const char* who = "dgcn_transform_grouped_int8_batch";
    ProductArgs a{};
    a.H = (const char*)H; a.ldh = ldh; a.hs = h_scale; a.rows = rows; a.cin = cin; a.W = (const char*)W; a.ws = w_scale; a.ctot = ctot;
    a.bias = bias; a.act = act; a.Y = Y; a.out_dtype = out_dtype; a.ldy = ldy; a.num_groups = num_groups; a.num_models = num_models;
    a.gptr = group_ptr; a.mog = model_of_group; a.status = status;
    if (num_groups > 0 && rows > 0 && (!group_ptr || !status)) return fail(DGCN_ERR_ARG, "%s: null argument", who);
    return product_int8(who, "transform_grouped_int8", a, (hipStream_t)stream);
}

extern "C" int dgcn_transform_grouped_batch(const void* H, int32_t dtype, int64_t ldh, float h_const, int32_t rows, int32_t cin,
                                            const int32_t* group_ptr, const int32_t* model_of_group, int32_t num_groups, const void* W,
                                            int32_t num_models, int32_t ctot, const float* bias, int32_t act, int32_t precise, void* Y,
                                            int64_t ldy, int32_t* status, void* stream) {
    const char* who = "dgcn_transform_grouped_batch";
    int rc = check_sizes(who, rows, cin, ctot, dtype == DGCN_F32 ? 4 : 2, H != nullptr, ldh, ldy, act);
    if (rc) return rc;
    if (!known_dtype(dtype)) return fail(DGCN_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if (num_groups < 0 || num_models <= 0) return fail(DGCN_ERR_ARG, "%s: bad sizes", who);
    if (dtype != DGCN_F32 && precise) return fail(DGCN_ERR_ARG, "%s: precise takes float32", who);
    if (rows == 0 || num_groups == 0) return DGCN_OK;
    if ((!H && dtype != DGCN_F32) || !W || !Y || !group_ptr || !status) return fail(DGCN_ERR_ARG, "%s: null argument", who);
    ProductArgs a{};
    a.H = (const char*)H; a.ldh = ldh; a.h_const = h_const; a.rows = rows; a.cin = cin; a.W = (const char*)W; a.ctot = ctot; a.bias = bias;
    a.act = act; a.Y = Y; a.out_dtype = dtype; a.ldy = ldy; a.num_groups = num_groups; a.num_models = num_models;
    a.gptr = group_ptr; a.mog = model_of_group; a.status = status;
    const int kind = dtype == DGCN_BF16 ? K_BF16 : dtype == DGCN_F16 ? K_F16 : precise ? K_F32P : K_F32;
    return product_dispatch("transform_grouped", kind, a, (hipStream_t)stream);
}

extern "C" int dgcn_product_path(int32_t dtype, int32_t precise, const void* H, int64_t ldh, int32_t rows, int32_t cin, int32_t num_groups,
                                 const void* W, int32_t ctot, const void* Y, int32_t out_dtype, int64_t ldy) {
    static const int32_t table = 0;  // (stands for a group table: nothing reads it)
    const char* who = "dgcn_product_path";
    const bool i8 = dtype == DGCN_I8;
    int rc = check_sizes(who, rows, cin, ctot, i8 ? 1 : dtype == DGCN_F32 ? 4 : 2, H != nullptr, ldh, ldy, DGCN_ACT_LINEAR);
    if (rc) return rc;
    if ((!i8 && !known_dtype(dtype)) || !known_dtype(out_dtype)) return fail(DGCN_ERR_ARG, "%s: unknown dtype %d -> %d", who, dtype, out_dtype);
    if (rows == 0 || num_groups < 0 || !W || !Y || (!H && dtype != DGCN_F32)) return fail(DGCN_ERR_ARG, "%s: no such product", who);
    if (i8 ? precise : out_dtype != dtype || num_groups == 0 || (precise && dtype != DGCN_F32)) return fail(DGCN_ERR_ARG, "%s: no such product", who);
    ProductArgs a{};
    a.H = (const char*)H; a.ldh = ldh; a.rows = rows; a.cin = cin; a.W = (const char*)W; a.ctot = ctot; a.Y = const_cast<void*>(Y);
    a.out_dtype = out_dtype; a.ldy = ldy; a.num_groups = num_groups > 0 ? num_groups : 1; a.gptr = num_groups > 0 ? &table : nullptr;
    const int kind = i8 ? K_I8 : dtype == DGCN_BF16 ? K_BF16 : dtype == DGCN_F16 ? K_F16 : precise ? K_F32P : K_F32;
    prepare_args(kind, a);
    return with_kind(kind, [&](auto k) {
        constexpr int KIND = decltype(k)::value;
        const int path = choose_path<KIND>(a);
        return path | (path < P_FEW_2_4 && direct_loads<KIND>(a) ? DGCN_PRODUCT_DIRECT : 0) | (a.stream ? DGCN_PRODUCT_STREAMS : 0);
    });
}
