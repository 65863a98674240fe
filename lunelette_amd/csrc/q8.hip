// Products of 8-bit rows with 8-bit weights (lh_q8_pack, lh_q8_quantize, lh_q8_matvec).
//
// Packed weights: tiles of 16 rows x 64 columns, row tile by row tile, the codes of
// all tiles first. A tile's 1 KiB holds for lane l = 16 g + r of a wave row r's columns
// 16 g .. 16 g + 15: the operand of a 16x16x64 matrix instruction. Then the FP32 scales
// of the rows. Rows and columns past the matrix, to a multiple of 16 and of 128, have
// codes and scales of 0, so what the activations hold past their last column adds nothing.
#include "lh_mfma.h"
#include "lh_serving.h"

namespace lh {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct Q8Shape {
    uint32_t rows, cols, tiles, blocks;   // 16-row tiles, 64-column blocks
};

static Q8Shape q8_shape(uint32_t rows, uint32_t cols)
{
    return {rows, cols, (rows + 15) / 16, (cols + 127) / 128 * 2};
}

__device__ __forceinline__ const float* q8_scales(const uint8_t* packed, const Q8Shape& p)
{
    return reinterpret_cast<const float*>(packed + (size_t)p.tiles * p.blocks * 1024);
}

// Four blocks of a tile, a wave each: grid (tiles, fours of blocks). Bound: the bytes, read and
// written once; 18432 x 3072 21.8 us, 5.2 TB/s (byte by byte 109).
__global__ void __launch_bounds__(256)
k_q8_pack(const int8_t* __restrict__ codes, const float* __restrict__ scales, Q8Shape p,
    uint8_t* __restrict__ packed)
{
    const uint32_t lane = threadIdx.x & 63, tile = blockIdx.x;
    const uint32_t block = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t row = tile * 16 + (lane & 15), col = block * 64 + 16 * (lane >> 4);
    if (block >= p.blocks) {
        return;
    }
    u32x4 word = {0, 0, 0, 0};
    if (row < p.rows) {
        const int8_t* c = codes + (size_t)row * p.cols + col;
        if (col + 16 <= p.cols) {
            __builtin_memcpy(&word, c, 16);   // at any address
        } else {
            for (uint32_t e = 0; e < 16; e++) {
                const uint32_t v = col + e < p.cols ? (uint8_t)c[e] : 0;
                word[e >> 2] |= v << (8 * (e & 3));
            }
        }
    }
    reinterpret_cast<u32x4*>(packed)[((size_t)tile * p.blocks + block) * 64 + lane] = word;
    if (block == 0 && lane < 16) {
        const_cast<float*>(q8_scales(packed, p))[tile * 16 + lane] = row < p.rows ? scales[row] : 0;
    }
}

// Columns c .. c + 3 of a row of `cols`; 0 past its end.
__device__ __forceinline__ float4 q8_quad(const float* x, uint32_t c, uint32_t cols)
{
    if (c + 3 < cols) {
        return load4(x + c);
    }
    return make_float4(c < cols ? x[c] : 0, c + 1 < cols ? x[c + 1] : 0,
        c + 2 < cols ? x[c + 2] : 0, 0);
}

// A workgroup a tile, a wave a row of it, so that the 16-byte pieces of a tile meet in one L2.
// The row's scale first, then its codes: in FP32 as in q8_rows.hip, in 64 bits next to
// a border. Bound: the bytes, of which the row's come twice; 18432 x 3072 90 us (a
// wave a row in 64 bits 320).
__global__ void __launch_bounds__(1024)
k_q8_quantize(const float* __restrict__ w, Q8Shape p, uint8_t* __restrict__ packed)
{
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t in = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x, row = tile * 16 + in;
    const float* x = w + (size_t)row * p.cols;
    const uint32_t cols = row < p.rows ? p.cols : 0;
    // Magnitudes as whole numbers, among which Inf and NaN are the largest. (The compiler forms a
    // vote over `v < infinity` with a comparison that a NaN passes: not equal to it.)
    uint32_t most = 0;
#pragma unroll 4
    for (uint32_t c = 4 * lane; c < cols; c += 256) {
        const float4 v = q8_quad(x, c, cols);
        most = max(max(most, max(__float_as_uint(fabsf(v.x)), __float_as_uint(fabsf(v.y)))),
            max(__float_as_uint(fabsf(v.z)), __float_as_uint(fabsf(v.w))));
    }
    const bool bad = !__all(most < 0x7f800000u);
    const float scale = (float)((double)wave_max64(__uint_as_float(most)) / 127.0);
    if (lane == 0) {
        const_cast<float*>(q8_scales(packed, p))[row] = bad ? __builtin_nanf("") : scale;
    }
    const bool some = !bad && scale > 0;
    const float by = some ? (float)(1.0 / (double)scale) : 0.0f;
    const bool wide = some && !(by >= 0x1p-100f && by <= 0x1p100f);
    const float whole = 0x1.8p23f, border = 0.5f - 0x1p-12f;
    uint8_t* to = packed + (size_t)tile * p.blocks * 1024 + 16 * in + 4 * (lane & 3);
#pragma unroll 4
    for (uint32_t c = 4 * lane; c < p.blocks * 64; c += 256) {
        uint32_t code[4] = {0, 0, 0, 0};
        if (some) {
            const float4 quad = q8_quad(x, c, cols);
            const float v[4] = {quad.x, quad.y, quad.z, quad.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float t = v[e] * by, rounded = t + whole;
                code[e] = __float_as_uint(rounded);
                if (wide || fabsf(t - (rounded - whole)) > border) {
                    code[e] = (uint32_t)(int)rint(
                        fmin(fmax((double)v[e] / (double)scale, -127.0), 127.0));
                }
            }
        }
        *reinterpret_cast<uint32_t*>(to + (size_t)(c >> 4) * 256) = (code[0] & 255) |
            (code[1] & 255) << 8 | (code[2] & 255) << 16 | code[3] << 24;
    }
}

struct Q8Args {
    const uint8_t* packed;
    Q8Shape p;
    const int8_t* x;
    const float* x_scales;
    float* y;
    int32_t* part;                  // [split][token][16 tiles] where columns are split
    size_t x_stride, y_stride;
    uint32_t tokens, splits, per;   // per: 128-column steps of a split
};

// y of four rows' sums v for a token. w: the rows' scales.
__device__ __forceinline__ float4 q8_values(float4 w, i32x4 v, float scale)
{
    return make_float4(scale * (w.x * (float)v[0]), scale * (w.y * (float)v[1]),
        scale * (w.z * (float)v[2]), scale * (w.w * (float)v[3]));
}

// Sums v of rows row .. row + 3 for a token, as y or as a split's part.
__device__ __forceinline__ void q8_put(const Q8Args& a, float4 w, i32x4 v, uint32_t token,
    float scale, uint32_t row, uint32_t split)
{
    if (a.splits > 1) {
        *reinterpret_cast<i32x4*>(a.part + ((size_t)split * a.tokens + token) * (a.p.tiles * 16) +
            row) = v;
        return;
    }
    float* y = a.y + token * a.y_stride + row;
    const float4 r = q8_values(w, v, scale);
    if (row + 3 < a.p.rows) {
        store4(y, r);
        return;
    }
    const float e[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 3; i++) {
        if (row + i < a.p.rows) {
            y[i] = e[i];
        }
    }
}

__device__ __forceinline__ float4 q8_row_scales(const Q8Args& a, uint32_t row)
{
    return *reinterpret_cast<const float4*>(q8_scales(a.packed, a.p) + row);
}

// The product of NT tiles of 16 tokens, one or two. A workgroup takes RT tiles of rows, its
// eight waves a slice of the columns each; a wave asks for U blocks of its slice at once
// and for another whenever it has multiplied one. The sums meet in LDS.
// Bound: the weights' bytes. Measured, cold weights: 18432 x 3072 (57 MB) for one token
// 10.5 us, 5.4 TB/s, 131072 x 3072 for eight 62 us, 6.5 TB/s; 3072 x 9216 6.8 us, of
// which a launch and the first bytes' way are 4. More tokens' words are 16 rows apart each,
// which a request takes half a cache line of: 3072 x 9216 for 16 tokens 10.3 us. Nine
// blocks on their way or three, sixteen waves or four: no gain.
enum { FEW_WAVES = 8 };

template <int RT, int NT>
__global__ void __launch_bounds__(64 * FEW_WAVES)
k_q8_few(Q8Args a)
{
    constexpr int W = FEW_WAVES, U = RT * NT == 4 ? 3 : 6;
    __shared__ i32x4 sums[W][RT * NT][64];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x * RT;
    const uint32_t per = (a.p.blocks + W - 1) / W, first = wave * per;
    const uint32_t end = first + per < a.p.blocks ? first + per : a.p.blocks;
    const uint32_t last_word = (a.p.cols - 1) & ~15u;
    const i32x4* w[RT];
    const int8_t* x[NT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        // Tiles past the last repeat it and are not stored.
        w[t] = reinterpret_cast<const i32x4*>(a.packed) +
            (size_t)(tile + t < a.p.tiles ? tile + t : a.p.tiles - 1) * a.p.blocks * 64 + lane;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t t = n * 16 + (lane & 15);
        x[n] = a.x + (t < a.tokens ? t : a.tokens - 1) * a.x_stride;
    }
    i32x4 wr[U][RT], xr[U][NT], acc[RT][NT];
    auto load = [&](int u, uint32_t b) __attribute__((always_inline)) {
        // Words past the last column meet codes of 0.
        const uint32_t col = b * 64 + 16 * (lane >> 4);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            xr[u][n] = *reinterpret_cast<const i32x4*>(x[n] + (col < last_word ? col : last_word));
        }
#pragma unroll
        for (int t = 0; t < RT; t++) {
            wr[u][t] = __builtin_nontemporal_load(w[t] + (size_t)b * 64);
        }
    };
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (first + u < end) {
            load(u, first + u);
        }
    }
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            acc[t][n] = (i32x4){0, 0, 0, 0};
        }
    }
    for (uint32_t b = first; b < end; b += U) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (b + u >= end) {
                break;
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    acc[t][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wr[u][t], xr[u][n],
                        acc[t][n], 0, 0, 0);
                }
            }
            if (b + u + U < end) {
                load(u, b + u + U);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            sums[wave][t * NT + n][lane] = acc[t][n];
        }
    }
    __syncthreads();
    const uint32_t token = wave % NT * 16 + (lane & 15), mine = tile + wave / NT;
    if (wave >= RT * NT || token >= a.tokens || mine >= a.p.tiles) {
        return;
    }
    i32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int i = 1; i < W; i++) {
        v += sums[i][wave][lane];
    }
    const uint32_t row = mine * 16 + 4 * (lane >> 4);
    q8_put(a, q8_row_scales(a, row), v, token, a.x_scales[token], row, 0);
}

// The workgroup's barrier after a wait that leaves some of the wave's loads into LDS on
// their way (__syncthreads waits for all of them).
template <int WAIT>
__device__ __forceinline__ void q8_meet()
{
    __builtin_amdgcn_s_waitcnt(WAIT);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A wave's own barrier: its lanes' accesses to LDS (which the unit makes in the order of the
// program) stay to their side of it.
__device__ __forceinline__ void wave_meet()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The product of many tokens. A workgroup of WM x WN waves forms the sums of MT = WM * MW
// tiles of rows and NT = WN * NW tiles of tokens, a wave MW x NW of them, over a split
// of the columns. 128 columns (a step) of both operands at a time go to LDS as they are
// multiplied, in B buffers: one is multiplied while the others fill.
// Bound: at large tiles matrix instructions and the operands' way from L2 to LDS, which the
// one barrier a step lets overlap in part. 18432 x 3072 for 2048 tokens takes 115 us, 2.0e15
// operations a second, with cold weights 122, with cold inputs and outputs too 124, and 134 to
// 139 beside a profiler (256 x 256 tiles: without the
// matrix instructions 100, without loads and reads 110, without stores 10 less, cold 20
// less; the matrix instructions alone reach 3.5e15 to 4.1e15 on random codes).
// Measured there, too, with stores of 64 bytes of a row (123, cold 130): tiles of
// 192 x 256 in one workgroup a unit 115, cold 131, but 82
// against 77 for 1024 tokens and 94 against 78 for 3072 x 9216; 256 x 256 125, cold 139
// (8192^3, which they fill: 2.37e15 a second); 128 x 256 in three buffers 144; workgroups
// that go on to their next item 138 (registers); four waves of 96 x 128 172 (registers);
// activations in pieces of 64 columns of 16 tokens 134 (half a cache line of each row a
// request); other starting columns for each workgroup, stores past the caches, priorities
// of waves or of workgroups: no gain.
template <int MW, int NW, int WM, int WN, int B>
__global__ void __launch_bounds__(64 * WM * WN, 2)
k_q8_tiles(Q8Args a, uint32_t mtiles, uint32_t ntiles)
{
    constexpr int W = WM * WN, MT = MW * WM, NT = NW * WN;
    constexpr int AP = 2 * MT / W, BP = 2 * NT / W;   // 1 KiB pieces a wave fetches
    static_assert(2 * MT % W == 0 && 2 * NT % W == 0, "pieces are dealt evenly");
    static_assert((B - 2) * (AP + BP) < 64, "the wait counts pieces");
    constexpr int SIZE = (MT + NT) * 2048;
    __shared__ __attribute__((aligned(1024))) uint8_t buf0[SIZE], buf1[SIZE];
    __shared__ __attribute__((aligned(1024))) uint8_t buf2[B > 2 ? SIZE : 16];
    __shared__ __attribute__((aligned(1024))) uint8_t buf3[B > 3 ? SIZE : 16];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wm = wave % WM, wn = wave / WM;
    // Neighbouring items to an XCD's workgroups (every eighth): they share rows and tokens
    // in its L2.
    uint32_t id = gridDim.x % 8 ? blockIdx.x
        : (blockIdx.x & 7) * (gridDim.x / 8) + (blockIdx.x >> 3);
    const uint32_t split = id % a.splits;
    id /= a.splits;
    const uint32_t group = ntiles >= 8 ? 8 : 32 / ntiles;
    const uint32_t base = id / (group * ntiles) * group, in = id % (group * ntiles);
    const uint32_t rows = mtiles - base < group ? mtiles - base : group;
    const uint32_t tile0 = (base + in % rows) * MT, token0 = in / rows * (NT * 16);
    const uint32_t all = (a.p.blocks + 1) / 2, first = split * a.per;
    const uint32_t end = first + a.per < all ? first + a.per : all;
    const uint32_t last_word = (a.p.cols - 1) & ~15u;
    // Where a wave's pieces come from. Of the activations a piece is 128 columns of 8
    // tokens, a lane's 16-byte word of them turned by its token: so the words that eight
    // lanes read at once lie in different banks. Tiles and tokens past the last repeat it
    // and are not stored; words past the last column meet codes of 0.
    const uint8_t* wfrom[AP];
    const int8_t* xfrom[BP];
#pragma unroll
    for (int n = 0; n < AP; n++) {
        const uint32_t t = tile0 + (AP * wave + n) / 2;
        wfrom[n] = a.packed + (size_t)(t < a.p.tiles ? t : a.p.tiles - 1) * a.p.blocks * 1024 +
            lane * 16;
    }
#pragma unroll
    for (int n = 0; n < BP; n++) {
        const uint32_t t = token0 + 8 * (BP * wave + n) + (lane >> 3);
        xfrom[n] = a.x + (t < a.tokens ? t : a.tokens - 1) * a.x_stride;
    }
    const uint32_t word = 16 * ((lane & 7) ^ (lane >> 3));
    // Steps past the last repeat it, so that the number of pieces on their way is the same
    // at each wait.
    auto fetch = [&](uint32_t step, uint8_t* to) __attribute__((always_inline)) {
        step = step < end ? step : end - 1;
#pragma unroll
        for (int n = 0; n < AP; n++) {
            const uint32_t f = AP * wave + n;
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(wfrom[n] +
                    (size_t)(2 * step + (f & 1)) * 1024),
                (__attribute__((address_space(3))) void*)(to + f * 1024), 16, 0, 0);
        }
        const uint32_t col = 128 * step + word;
#pragma unroll
        for (int n = 0; n < BP; n++) {
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(xfrom[n] +
                    (col < last_word ? col : last_word)),
                (__attribute__((address_space(3))) void*)(to + (2 * MT + BP * wave + n) * 1024), 16,
                0, 0);
        }
    };
    i32x4 acc[MW][NW];
#pragma unroll
    for (int m = 0; m < MW; m++) {
#pragma unroll
        for (int n = 0; n < NW; n++) {
            acc[m][n] = (i32x4){0, 0, 0, 0};
        }
    }
    // A half (64 columns) of a step's operands: of the activations token lane & 15's word
    // of columns 16 (lane >> 4).
    const uint32_t x_at = (lane & 15) * 128 + 16 * ((lane >> 4) ^ (lane & 7));
    auto read = [&](const uint8_t* from, int h, i32x4 (&w)[MW], i32x4 (&x)[NW])
        __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NW; n++) {
            x[n] = *reinterpret_cast<const i32x4*>(from + 2 * (MT + wn * NW + n) * 1024 +
                (h ? x_at ^ 64 : x_at));
        }
#pragma unroll
        for (int m = 0; m < MW; m++) {
            w[m] = *reinterpret_cast<const i32x4*>(from + (2 * (wm * MW + m) + h) * 1024 +
                lane * 16);
        }
    };
    auto multiply = [&](const i32x4 (&w)[MW], const i32x4 (&x)[NW])
        __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < MW; m++) {
#pragma unroll
            for (int n = 0; n < NW; n++) {
                acc[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[m], x[n], acc[m][n], 0, 0, 0);
            }
        }
    };
    // vmcnt(B - 2 steps' pieces), lgkmcnt(0): the next step's pieces, this wave's reads.
    constexpr int LEFT = (B - 2) * (AP + BP);
    constexpr int WAIT = 0x0070 | (LEFT & 15) | (LEFT >> 4) << 14;
    i32x4 w0[MW], x0[NW], w1[MW], x1[NW];
    // The order that the compiler is held to: reads and loads among the matrix instructions,
    // which take 16 cycles each, not all ahead of them (2048 tokens below: 4 us less).
    constexpr int MFMA = 8, LOAD = 16, READ = 256, BETWEEN = MW * NW / (MW + NW);
    // Step s in `now`, whose first half is in registers; the next B - 2 are on their way.
    auto turn = [&](uint32_t s, uint8_t* now, uint8_t* then) __attribute__((always_inline)) {
        read(now, 1, w1, x1);
        multiply(w0, x0);
#pragma unroll
        for (int i = 0; i < MW + NW; i++) {
            __builtin_amdgcn_sched_group_barrier(READ, 1, 0);
            __builtin_amdgcn_sched_group_barrier(MFMA, BETWEEN, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        q8_meet<WAIT>();
        fetch(s + B, now);
        read(then, 0, w0, x0);
        multiply(w1, x1);
#pragma unroll
        for (int i = 0; i < MW + NW; i++) {
            if (i < AP + BP) {
                __builtin_amdgcn_sched_group_barrier(LOAD, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(READ, 1, 0);
            __builtin_amdgcn_sched_group_barrier(MFMA, BETWEEN, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        return s + 1 < end;
    };
    fetch(first, buf0);
    fetch(first + 1, buf1);
    if (B > 2) {
        fetch(first + 2, buf2);
    }
    if (B > 3) {
        fetch(first + 3, buf3);
    }
    constexpr int START = (B - 1) * (AP + BP);
    q8_meet<0x0f70 | (START & 15) | (START >> 4) << 14>();
    read(buf0, 0, w0, x0);
    for (uint32_t s = first;; s += B) {
        if (!turn(s, buf0, buf1)) {
            break;
        }
        if (B == 2) {
            if (!turn(s + 1, buf1, buf0)) {
                break;
            }
        } else {
            if (!turn(s + 1, buf1, buf2) || !turn(s + 2, buf2, B > 3 ? buf3 : buf0) ||
                (B > 3 && !turn(s + 3, buf3, buf0))) {
                break;
            }
        }
    }
    // All scales before the first store, behind which the compiler keeps a load.
    float4 w[MW];
    float scale[NW];
#pragma unroll
    for (int m = 0; m < MW; m++) {
        const uint32_t t = tile0 + wm * MW + m;
        w[m] = q8_row_scales(a, (t < a.p.tiles ? t : a.p.tiles - 1) * 16 + 4 * (lane >> 4));
    }
#pragma unroll
    for (int n = 0; n < NW; n++) {
        const uint32_t token = token0 + (wn * NW + n) * 16 + (lane & 15);
        scale[n] = a.x_scales[token < a.tokens ? token : a.tokens - 1];
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);   // here: between stores it would wait for those too
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MW >= 4) {
        if (a.splits == 1 && (tile0 + MT) * 16 <= a.p.rows) {
            // Through LDS, where all waves are done: a store then takes 256 bytes and more of a
            // token's row in place of 64 (2048 tokens above 123 us -> 116, cold 130 -> 124).
            constexpr int WIDE = MW * 16 + 4;   // floats of a token, in other banks than the next's
            static_assert(W / 2 * 16 * WIDE * 4 <= SIZE, "half of the waves in a buffer");
            __syncthreads();
            float* mine = reinterpret_cast<float*>(wave < W / 2 ? buf0 : buf1) +
                wave % (W / 2) * (16 * WIDE);
            float* y = a.y + (tile0 + wm * MW) * 16;
#pragma unroll
            for (int n = 0; n < NW; n++) {
#pragma unroll
                for (int m = 0; m < MW; m++) {
                    *reinterpret_cast<float4*>(mine + (lane & 15) * WIDE + m * 16 +
                        4 * (lane >> 4)) = q8_values(w[m], acc[m][n], scale[n]);
                }
                wave_meet();
#pragma unroll
                for (int i = 0; i < MW; i++) {
                    const uint32_t t = (i * 64 + lane) / (MW * 4);
                    const uint32_t c = (i * 64 + lane) % (MW * 4) * 4;
                    const uint32_t token = token0 + (wn * NW + n) * 16 + t;
                    const float4 v = *reinterpret_cast<const float4*>(mine + t * WIDE + c);
                    if (token < a.tokens) {
                        store4(y + token * a.y_stride + c, v);
                    }
                }
                wave_meet();
            }
            return;
        }
    }
#pragma unroll
    for (int n = 0; n < NW; n++) {
        const uint32_t token = token0 + (wn * NW + n) * 16 + (lane & 15);
        if (token >= a.tokens) {
            continue;
        }
#pragma unroll
        for (int m = 0; m < MW; m++) {
            const uint32_t tile = tile0 + wm * MW + m;
            if (tile < a.p.tiles) {
                q8_put(a, w[m], acc[m][n], token, scale[n], tile * 16 + 4 * (lane >> 4), split);
            }
        }
    }
}

// Joins the column splits' sums: a thread four rows of a token.
__global__ void __launch_bounds__(256)
k_q8_join(Q8Args a)
{
    const uint32_t row = (blockIdx.x * 256 + threadIdx.x) * 4, token = blockIdx.y;
    if (row >= a.p.rows) {
        return;
    }
    const uint32_t splits = a.splits;
    const size_t wide = a.p.tiles * 16, one = a.tokens * wide;
    const int32_t* from = a.part + token * wide + row;
    i32x4 v = *reinterpret_cast<const i32x4*>(from);
    for (uint32_t i = 1; i < splits; i++) {
        v += *reinterpret_cast<const i32x4*>(from + i * one);
    }
    a.splits = 1;
    q8_put(a, q8_row_scales(a, row), v, token, a.x_scales[token], row, 0);
}

}  // namespace lh

using namespace lh;

extern "C" int lh_launch_q8_pack(const int8_t* codes, const float* scales, uint32_t rows,
    uint32_t cols, uint8_t* packed, hipStream_t s)
{
    const Q8Shape p = q8_shape(rows, cols);
    hipLaunchKernelGGL(k_q8_pack, dim3(p.tiles, (p.blocks + 3) / 4), dim3(256), 0, s, codes,
        scales, p, packed);
    return (int)hipGetLastError();
}

extern "C" int lh_launch_q8_quantize(const float* w, uint32_t rows, uint32_t cols,
    uint8_t* packed, hipStream_t s)
{
    const Q8Shape p = q8_shape(rows, cols);
    hipLaunchKernelGGL(k_q8_quantize, dim3(p.tiles), dim3(1024), 0, s, w, p, packed);
    return (int)hipGetLastError();
}

// Whether k_q8_few runs a product: to 16 tokens, and to 32 where each workgroup's reading of
// their words costs less than tiles in LDS, for few rows and columns. Measured (17, 24, 32
// tokens, cold weights, us; tiles in brackets):
//   3072 x 3072     5.3  6.0  6.6 ( 8.3  8.7  9.1)   3072 x 6144   8.4  9.7 11.0 (10.5 10.7 11.0)
//   6144 x 3072     6.7  7.5  8.2 (10.7 10.8 10.9)   6144 x 6144  11.1 12.3 13.9 (12.8 13.0 13.6)
//   12288 x 3072   10.6 11.9 13.4 (11.6 11.7 11.8)   3072 x 9216  10.7 12.6 14.3 (12.6 12.9 12.9)
//   18432 x 3072   14.5 16.4 18.6 (15.2 15.7 16.3)   1024 x 16384 15.0 17.8 21.0 (12.2 12.5 12.7)
// The limits are those of 24 tokens; 17 tokens would gain 5 to 15% past them, 32 lose as much
// within (12288 x 6144: 24.2 against 20.2).
static bool q8_few(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    return tokens <= 16 || (tokens <= 32 && rows <= 12288 && cols <= 6144);
}

// Other ways to run a product: a workgroup's tile, the 1 / 64 us that a step takes
// it where it is alone on a compute unit, and that it adds where others are there too.
struct Q8Way {
    uint32_t rows, tokens, buffers, alone, shared;
};
static const Q8Way q8_ways[] = {
    {64, 32, 4, 13, 11}, {64, 64, 3, 18, 15}, {64, 128, 3, 24, 24}, {128, 128, 2, 46, 37},
    {192, 128, 2, 64, 50},
};
enum { Q8_WAYS = sizeof q8_ways / sizeof *q8_ways, Q8_SPLITS = 8, UNITS = 256 };

struct Q8Plan {
    uint32_t way, splits, per;
};

// The way and number of column splits of the least estimated time. The estimate adds up the
// steps of a unit's workgroups, as many at once as LDS holds, and for splits a second
// launch with their sums written and read. Fitted to 180 sizes (1024 to 18432 rows, 1024
// to 9216 columns, 17 to 2048 tokens, cold weights): what it picks takes 4% longer on
// average, 31% at worst, than the best measured there of all splits of ten tiles (these
// and 32 x 64, 64 x 64 and 64 x 128 and 128 x 128 in other waves, 192 x 256).
static Q8Plan q8_plan(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    const uint64_t steps = (cols + 127) / 128;
    Q8Plan best = {0, 1, (uint32_t)steps};
    uint64_t least = ~(uint64_t)0;
    for (uint32_t w = 0; w < Q8_WAYS; w++) {
        const Q8Way& way = q8_ways[w];
        const uint64_t tiles = (uint64_t)((rows + way.rows - 1) / way.rows) *
            ((tokens + way.tokens - 1) / way.tokens);
        const uint64_t lds = way.buffers * (way.rows + way.tokens) * 128;
        const uint64_t at_once = 160 * 1024 / lds < 4 ? 160 * 1024 / lds : 4;
        for (uint32_t want = 1; want <= Q8_SPLITS && 2 * want <= steps + 1; want++) {
            const uint64_t per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
            const uint64_t mine = (tiles * splits + UNITS - 1) / UNITS, rest = mine % at_once;
            const auto step = [&](uint64_t n) {
                return n * way.shared > way.alone ? n * way.shared : way.alone;
            };
            uint64_t time = per * (mine / at_once * step(at_once) + (rest ? step(rest) : 0));
            if (splits > 1) {
                // 2.9 us, and 8 bytes a sum at 4.9 TB/s, in 1 / 64 us.
                time += 185 + splits * rows * tokens / 9475;
            }
            if (time < least) {
                least = time;
                best = {w, (uint32_t)splits, (uint32_t)per};
            }
        }
    }
    return best;
}

// The kernel that a product runs: k_q8_few with two tiles of rows (1) or not (0), with two
// of tokens (2 more), or from 4 on one of q8_ways.
// Two tiles of rows share the tokens' words, but leave half the workgroups. Measured, one tile
// against two (us, cold weights): 6144 x 3072 for 4 tokens 5.8 and 5.6, for 8 6.3 and 5.8, for
// 16 7.6 and 6.6, for 24 9.3 and 7.6; 12288 x 3072 for 24 16.0 and 12.0; 131072 x 3072 for 4
// 57.6 and 59.7, for 8 62.7 and 61.7, for 16 89 and 72; below 384 tiles, 4096 x 3072 for 16 5.4
// and 6.3. Not on its side are few tokens over many rows: 18432 x 3072 for 5 to 12 10.8 to 12.9
// and 13.0 to 14.4 (16: 14.7 and 14.4), 8192 x 8192 for 8 13.1 and 15.8.
static Q8Plan q8_kernel(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    if (q8_few(rows, cols, tokens)) {
        const bool two = tokens > 4 && (rows + 15) / 16 >= 384;
        return {two + 2u * (tokens > 16), 1, 0};
    }
    Q8Plan plan = q8_plan(rows, cols, tokens);
    plan.way += 4;
    return plan;
}

template <int MW, int NW, int WM, int WN, int B>
static void q8_tiles(const Q8Args& a, hipStream_t s)
{
    const uint32_t m = (a.p.tiles + MW * WM - 1) / (MW * WM);
    const uint32_t n = (a.tokens + 16 * NW * WN - 1) / (16 * NW * WN);
    hipLaunchKernelGGL((k_q8_tiles<MW, NW, WM, WN, B>), dim3(m * n * a.splits), dim3(64 * WM * WN),
        0, s, a, m, n);
}

template <int RT, int NT>
static void q8_streamed(const Q8Args& a, hipStream_t s)
{
    hipLaunchKernelGGL((k_q8_few<RT, NT>), dim3((a.p.tiles + RT - 1) / RT), dim3(64 * FEW_WAVES),
        0, s, a);
}

extern "C" int lh_q8_way(uint32_t rows, uint32_t cols, uint32_t tokens, uint32_t* splits)
{
    const Q8Plan plan = q8_kernel(rows, cols, tokens);
    *splits = plan.splits;
    return (int)plan.way;
}

extern "C" size_t lh_q8_scratch_bytes(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    uint32_t splits;
    lh_q8_way(rows, cols, tokens, &splits);
    return splits == 1 ? 0 : (size_t)splits * tokens * ((rows + 15) / 16 * 64);
}

extern "C" int lh_launch_q8_matvec(const uint8_t* packed, const int8_t* x, size_t x_stride,
    const float* x_scales, float* y, size_t y_stride, uint32_t rows, uint32_t cols,
    uint32_t tokens, uint8_t* scratch, hipStream_t s)
{
    const Q8Plan plan = q8_kernel(rows, cols, tokens);
    const Q8Args a = {packed, q8_shape(rows, cols), x, x_scales, y,
        reinterpret_cast<int32_t*>(scratch), x_stride, y_stride, tokens, plan.splits, plan.per};
    switch (plan.way) {
    case 0: q8_streamed<1, 1>(a, s); break;
    case 1: q8_streamed<2, 1>(a, s); break;
    case 2: q8_streamed<1, 2>(a, s); break;
    case 3: q8_streamed<2, 2>(a, s); break;
    case 4: q8_tiles<1, 2, 4, 1, 4>(a, s); break;
    case 5: q8_tiles<2, 2, 2, 2, 3>(a, s); break;
    case 6: q8_tiles<2, 2, 2, 4, 3>(a, s); break;
    case 7: q8_tiles<4, 2, 2, 4, 2>(a, s); break;
    default: q8_tiles<6, 4, 2, 2, 2>(a, s); break;
    }
    const hipError_t e = hipGetLastError();
    if (e || a.splits == 1) {
        return (int)e;
    }
    hipLaunchKernelGGL(k_q8_join, dim3((rows + 1023) / 1024, tokens), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}
