// Dense products of batches with several models and of 8-bit matrices (include/dgcn.h: dgcn_transform_grouped_batch,
// dgcn_transform_int8_batch, dgcn_transform_grouped_int8_batch).
//
//   Y[r][n] = act( epilogue( sum_k H[r][k] * W[e(r)][n][k] ) + bias[e(r)][n] )
//
// Every type runs the same tile loop in BYTES: 64 bytes of a row of H and of W feed one step of a 16 x 16 output tile, 16 bytes per
// lane (lane & 15 = the row, lane >> 4 = which 16 of the 64 bytes): one MFMA of int8 (k = 64), bf16 / fp16 (k = 32), four of float32
// (k = 4 each).  W is the MFMA's A operand and H its B operand, so a lane ends with four output columns n of ONE row r.
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
    bool vec_out;        // rows of Y take 16-byte (float32) / 8-byte (half) stores
};

template <int KIND> struct Elem;
template <> struct Elem<K_I8> { static constexpr int size = 1; using Acc = i32x4; };
template <> struct Elem<K_BF16> { static constexpr int size = 2; using Acc = f32x4; };
template <> struct Elem<K_F16> { static constexpr int size = 2; using Acc = f32x4; };
template <> struct Elem<K_F32> { static constexpr int size = 4; using Acc = f32x4; };
template <> struct Elem<K_F32P> { static constexpr int size = 4; using Acc = f64x4; };

// The group of a tile slot without a prefix sum over the groups: group g's row tiles start at slot floor(p_g / BM) + g, which is
// increasing in g, and ceil((p_{g+1} - p_g) / BM) never exceeds the distance to the next group's start.  So a launch of
// floor(rows / BM) + num_groups slots covers every tile (some slots are empty), and a slot finds its group by search: 64-ary, a lane
// per probe.  Pointers are clamped to [0, rows] before use: a bad table cannot lead out of the matrix.
struct Tile { int row0, row1, model; };  // rows [row0, row1) of this slot; row0 >= row1: nothing to do

__device__ __forceinline__ Tile find_tile(const ProductArgs& a, int64_t slot, int BM) {
    Tile t{0, 0, 0};
    if (!a.gptr) {
        const int64_t r = slot * BM;
        t.row0 = (int)min(r, (int64_t)a.rows);
        t.row1 = (int)min(r + BM, (int64_t)a.rows);
        return t;
    }
    const int lane = threadIdx.x & 63;
    auto ptr = [&](int g) { return min(max(a.gptr[g], 0), a.rows); };
    int lo = 0, n = a.num_groups;  // the group is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const int64_t i = (int64_t)lane * step;
        const bool below = i < n && (int64_t)(ptr(lo + (int)i) / BM) + lo + i <= slot;
        const unsigned long long m = __ballot(below);
        const int k = m == ~0ull ? 64 : __builtin_ctzll(~m);
        if (k == 0) return t;  // in front of the first group
        const int at = (k - 1) * step;
        lo += at;
        n = min(step, n - at);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int p0 = ptr(lo), p1 = ptr(lo + 1);
    const int64_t tile = slot - (p0 / BM + (int64_t)lo);
    const int64_t r = p0 + tile * BM;
    if (tile < 0 || r >= p1) return t;
    const int e = a.mog ? a.mog[lo] : lo;
    if (e < 0 || e >= a.num_models) return t;
    t.row0 = (int)r;
    t.row1 = (int)min(r + BM, (int64_t)p1);
    t.model = e;
    return t;
}

// Every slot below num_groups checks the table entry of its own number.
__device__ __forceinline__ void check_group(const ProductArgs& a, int64_t slot) {
    if (!a.gptr || slot >= a.num_groups || threadIdx.x != 0) return;
    const int g = (int)slot, p0 = a.gptr[g], p1 = a.gptr[g + 1], e = a.mog ? a.mog[g] : g;
    if (p0 < 0 || p1 < p0 || p1 > a.rows || e < 0 || e >= a.num_models) atomicOr(a.status, (int)DGCN_FAULT_BAD_GROUP);
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
// the other types take chunk lane >> 4 as it lies.  `row` is the LDS row, `step` the 64-byte step within it.
template <int KIND, int ROW_BYTES>
__device__ __forceinline__ i32x4 lds_frag(const char* base, int row, int step) {
    const int q = (threadIdx.x & 63) >> 4;
    if constexpr (KIND == K_F32 || KIND == K_F32P) {
        i32x4 v;
#pragma unroll
        for (int s = 0; s < 4; ++s) v[s] = *reinterpret_cast<const int*>(base + row * ROW_BYTES + (((step * 4 + s) ^ (row & 7)) << 4) + (q << 2));
        return v;
    } else {
        return *reinterpret_cast<const i32x4*>(base + row * ROW_BYTES + (((step * 4 + q) ^ (row & 7)) << 4));
    }
}

template <class O> __device__ __forceinline__ O round_to(float x) { return (O)x; }

// Four output columns n .. n + 3 of row r.
template <class O>
__device__ __forceinline__ void store4(const ProductArgs& a, int64_t r, int n, const float (&v)[4]) {
    O* y = reinterpret_cast<O*>(a.Y) + r * a.ldy + n;
    if (a.vec_out && n + 4 <= a.ctot) {
        using V = __attribute__((ext_vector_type(4))) O;
        V o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = round_to<O>(v[i]);
        *reinterpret_cast<V*>(y) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.ctot) y[i] = round_to<O>(v[i]);
    }
}

// Columns n .. n + 3 of row r from their accumulators: scales, bias, activation, one rounding.
template <int KIND>
__device__ __forceinline__ void finish4(const ProductArgs& a, const Tile& t, int64_t r, int n, typename Elem<KIND>::Acc acc) {
    const int64_t ch = (int64_t)t.model * a.ctot + n;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = (float)acc[i];
        const bool in = n + i < a.ctot;
        if constexpr (KIND == K_I8) v[i] = (v[i] * a.hs[r]) * (in ? a.ws[ch + i] : 0.f);
        if (a.bias) v[i] += in ? a.bias[ch + i] : 0.f;
        v[i] = apply_act(v[i], a.act);
    }
    if (a.out_dtype == DGCN_F32) store4<float>(a, r, n, v);
    else if (a.out_dtype == DGCN_BF16) store4<__bf16>(a, r, n, v);
    else store4<_Float16>(a, r, n, v);
}

// 16 bytes at byte offset `off` of a row of `row_bytes` bytes; bytes behind the row's end are zero.
template <int KIND>
__device__ __forceinline__ i32x4 load_chunk(const char* row, int64_t off, int64_t row_bytes) {
    i32x4 v = {0, 0, 0, 0};
    if (off + 16 <= row_bytes) {
        __builtin_memcpy(&v, row + off, 16);
    } else if (off < row_bytes) {
        char* d = reinterpret_cast<char*>(&v);
        constexpr int ES = Elem<KIND>::size;
#pragma unroll
        for (int i = 0; i < 16 / ES; ++i)
            if (off + (i + 1) * ES <= row_bytes) __builtin_memcpy(d + i * ES, row + off + i * ES, ES);
    }
    return v;
}

// The general kernel: any alignment, any size.  64 x 64 output tile, four waves of 32 x 32, 128 bytes of k per stage through
// registers into LDS (rows of 128 bytes, their 16-byte chunks permuted by the row number: reads of eight rows meet no bank twice).
template <int KIND>
__global__ __launch_bounds__(256) void k_product_any(ProductArgs a, int64_t slots, int col_tiles) {
    constexpr int BM = 64, BN = 64, RB = 128, ES = Elem<KIND>::size;
    using Acc = typename Elem<KIND>::Acc;
    __shared__ __attribute__((aligned(16))) char sH[BM * RB];
    __shared__ __attribute__((aligned(16))) char sW[BN * RB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    const int64_t kbytes = (int64_t)a.cin * ES;
    const int steps = (int)((kbytes + RB - 1) / RB);
    for (int64_t tile = blockIdx.x; tile < slots * col_tiles; tile += gridDim.x) {
        const int64_t slot = tile / col_tiles;
        const int n0 = (int)(tile - slot * col_tiles) * BN;
        if (n0 == 0) check_group(a, slot);
        const Tile t = find_tile(a, slot, BM);
        if (t.row0 >= t.row1) continue;
        const char* Wm = a.W + (int64_t)t.model * a.ctot * kbytes;
        Acc acc[2][2] = {};
        const int lr = threadIdx.x >> 3, lc = threadIdx.x & 7;  // this thread's chunk of rows lr and lr + 32
        i32x4 h[2], w[2];
        auto load = [&](int st) {
            const int64_t off = (int64_t)st * RB + lc * 16;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = min(t.row0 + lr + 32 * j, t.row1 - 1), n = min(n0 + lr + 32 * j, a.ctot - 1);
                w[j] = load_chunk<KIND>(Wm + (int64_t)n * kbytes, off, kbytes);
                if ((KIND == K_F32 || KIND == K_F32P) && !a.H) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[j][i] = off + 4 * i < kbytes ? __builtin_bit_cast(int, a.h_const) : 0;
                } else {
                    h[j] = load_chunk<KIND>(a.H + (int64_t)r * a.ldh * ES, off, kbytes);
                }
            }
        };
        load(0);
        for (int st = 0; st < steps; ++st) {
            __syncthreads();  // (the last stage's reads are done)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int o = (lr + 32 * j) * RB + ((lc ^ (lr & 7)) << 4);
                *reinterpret_cast<i32x4*>(sH + o) = h[j];
                *reinterpret_cast<i32x4*>(sW + o) = w[j];
            }
            __syncthreads();
            if (st + 1 < steps) load(st + 1);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                i32x4 fh[2], fw[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    fh[j] = lds_frag<KIND, RB>(sH, wm + j * 16 + (lane & 15), k);
                    fw[j] = lds_frag<KIND, RB>(sW, wn + j * 16 + (lane & 15), k);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = mfma_step<KIND>(fw[j], fh[i], acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = t.row0 + wm + i * 16 + (lane & 15);
                if (r >= t.row1) continue;
                if constexpr (KIND == K_F32P) {
                    // (the double instruction returns row 4 i + (lane >> 4) in register i)
                    const int64_t ch = (int64_t)t.model * a.ctot;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int n = n0 + wn + j * 16 + 4 * x + (lane >> 4);
                        if (n >= a.ctot) continue;
                        float v = (float)acc[i][j][x];
                        if (a.bias) v += a.bias[ch + n];
                        reinterpret_cast<float*>(a.Y)[(int64_t)r * a.ldy + n] = apply_act(v, a.act);
                    }
                } else {
                    const int n = n0 + wn + j * 16 + 4 * (lane >> 4);
                    if (n < a.ctot) finish4<KIND>(a, t, r, n, acc[i][j]);
                }
            }
        __syncthreads();  // (the next tile's first stage overwrites the LDS)
    }
}

static size_t dtype_size(int32_t d) { return d == DGCN_F32 ? 4 : 2; }

template <int KIND> static int launch_any(const char* family, const ProductArgs& a, hipStream_t s) {
    const int64_t slots = a.gptr ? (int64_t)a.rows / 64 + a.num_groups : ((int64_t)a.rows + 63) / 64;
    const int col_tiles = ceil_div(a.ctot, 64);
    const int blocks = (int)min(slots * col_tiles, (int64_t)1 << 20);
    TimedLaunch t(family, s);
    DGCN_LAUNCH(t, (k_product_any<KIND>), dim3(blocks), dim3(256), 0, s, a, slots, col_tiles);
    return check_launch("k_product_any");
}

static int product_dispatch(const char* family, int kind, ProductArgs& a, hipStream_t s) {
    const size_t os = dtype_size(a.out_dtype);
    a.vec_out = a.ldy % 4 == 0 && (uintptr_t)a.Y % (4 * os) == 0;
    switch (kind) {
        case K_I8: return launch_any<K_I8>(family, a, s);
        case K_BF16: return launch_any<K_BF16>(family, a, s);
        case K_F16: return launch_any<K_F16>(family, a, s);
        case K_F32: return launch_any<K_F32>(family, a, s);
        default: return launch_any<K_F32P>(family, a, s);
    }
}

static bool known_dtype(int32_t d) { return d == DGCN_F32 || d == DGCN_BF16 || d == DGCN_F16; }
static bool known_act(int32_t a) { return a == DGCN_ACT_LINEAR || a == DGCN_ACT_LEAKY_RELU || a == DGCN_ACT_RELU; }
constexpr int kMaxExtent = 0x7fffffff - 1023;  // tile corners stay within 32 bits
constexpr int kMaxInt8Depth = 131071;  // 128 * 128 * cin stays below 2^31

static int check_sizes(const char* who, int32_t rows, int32_t cin, int32_t ctot, bool has_h, int64_t ldh, int64_t ldy, int32_t act) {
    if (rows < 0 || cin <= 0 || ctot <= 0 || (has_h && ldh < cin) || ldy < ctot) return fail(DGCN_ERR_ARG, "%s: bad sizes", who);
    if (!known_act(act)) return fail(DGCN_ERR_ARG, "%s: unknown activation %d", who, act);
    if (rows > kMaxExtent || ctot > kMaxExtent) return fail(DGCN_ERR_UNSUPPORTED, "%s: more than %d rows or columns", who, kMaxExtent);
    return DGCN_OK;
}

static int product_int8(const char* who, const char* family, ProductArgs& a, hipStream_t s) {
    int rc = check_sizes(who, a.rows, a.cin, a.ctot, true, a.ldh, a.ldy, a.act);
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
    int rc = check_sizes(who, rows, cin, ctot, H != nullptr, ldh, ldy, act);
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
