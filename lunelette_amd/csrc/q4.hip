// Products with 4-bit weights and BF16 group scales (lh_q4_*).
//
// Packed weights: tiles of 16 rows x 128 columns, row tile by row tile, the
// codes of all tiles first. A tile's 1 KiB of codes holds for lane
// l = 16 g + r of a wave 16 bytes: word j has row r's columns 32 j + 8 g .. + 7,
// the even ones' codes in nibbles 0..3 and the odd ones' in 4..7, so that
// (word >> 4 i) & 0x000f000f is columns 2 i and 2 i + 1 as two 16-bit halves: the
// operand of a 16x16x32 matrix instruction. Then the scales: a tile's hold for g
// and group j the four BF16 scales of rows 4 g .. 4 g + 3, the rows of a lane's
// results. Rows and columns past the matrix have code 8 and scale 0.
#include "lh_nibbles.h"
#include "lh_serving.h"

namespace lh {

struct Q4Shape {
    uint32_t rows, cols, group, tiles, blocks;   // 16-row tiles, 128-column blocks
};

static Q4Shape q4_shape(uint32_t rows, uint32_t cols, uint32_t group)
{
    return {rows, cols, group, (rows + 15) / 16, (cols + 127) / 128};
}

__device__ __forceinline__ size_t q4_scales_at(const Q4Shape& p)
{
    return (size_t)p.tiles * p.blocks * 1024;
}

// Byte of (16-row tile, block)'s scale of row r (0..15) and group j of the block.
__device__ __forceinline__ size_t q4_scale_at(const Q4Shape& p, uint32_t tile, uint32_t block,
    uint32_t r, uint32_t j)
{
    const uint32_t per = 128 / p.group;
    return q4_scales_at(p) + ((size_t)tile * p.blocks + block) * (32 * per) +
        ((r >> 2) * per + j) * 8 + (r & 3) * 2;
}

// One word of packed codes a thread: grid (tiles, blocks), 256 threads.
__global__ void __launch_bounds__(256)
k_q4_pack(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales, Q4Shape p,
    uint8_t* __restrict__ packed)
{
    const uint32_t tile = blockIdx.x, block = blockIdx.y, i = threadIdx.x;
    const uint32_t lane = i >> 2, j = i & 3, row = tile * 16 + (lane & 15);
    const uint32_t col = block * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t word = 0x88888888u;
    if (row < p.rows && col < p.cols) {
        const uint8_t* c = codes + (size_t)row * (p.cols / 2) + col / 2;
        word = 0;
        for (int e = 0; e < 4; e++) {
            const uint32_t two = c[e];
            word |= (two & 15u) << (4 * e) | (two >> 4) << (16 + 4 * e);
        }
    }
    reinterpret_cast<uint32_t*>(packed)[((size_t)tile * p.blocks + block) * 256 + i] = word;
    const uint32_t per = 128 / p.group;
    if (i < 16 * per) {
        const uint32_t r = i / per, g = i % per, srow = tile * 16 + r, gcol = block * per + g;
        const uint16_t v = srow < p.rows && gcol < p.cols / p.group
            ? scales[(size_t)srow * (p.cols / p.group) + gcol] : (uint16_t)0;
        *reinterpret_cast<uint16_t*>(packed + q4_scale_at(p, tile, block, r, g)) = v;
    }
}

// Rounds FP32 weights: 256 threads of a (block, tile) form the scales of its
// groups, then a packed word each.
__global__ void __launch_bounds__(256)
k_q4_quantize(const float* __restrict__ w, Q4Shape p, uint8_t* __restrict__ packed)
{
    __shared__ float scale[16][4];
    const uint32_t tile = blockIdx.x, block = blockIdx.y, i = threadIdx.x;
    const uint32_t per = 128 / p.group;
    if (i < 16 * per) {
        const uint32_t r = i / per, g = i % per, row = tile * 16 + r;
        const uint32_t first = block * 128 + g * p.group;
        uint32_t s = 0;
        if (row < p.rows && first < p.cols) {
            float most = 0;
            bool finite = true;
            for (uint32_t c = 0; c < p.group; c++) {
                const float v = w[(size_t)row * p.cols + first + c];
                finite &= __builtin_isfinite(v);
                most = fmaxf(most, fabsf(v));
            }
            s = finite ? bf16_nearest(most / 7.0f) : 0x7fc0u;
        }
        scale[r][g] = bf16_to_f32(s);
        *reinterpret_cast<uint16_t*>(packed + q4_scale_at(p, tile, block, r, g)) = (uint16_t)s;
    }
    __syncthreads();
    const uint32_t lane = i >> 2, j = i & 3, row = tile * 16 + (lane & 15);
    const uint32_t col = block * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t word = 0x88888888u;
    if (row < p.rows && col < p.cols) {
        const float s = scale[lane & 15][(32 * j) / p.group];
        if (s > 0) {
            word = 0;
            for (uint32_t e = 0; e < 8; e++) {
                const float v = w[(size_t)row * p.cols + col + e] / s;
                const float code = __builtin_rintf(fminf(fmaxf(v, -7.0f), 7.0f)) + 8.0f;
                word |= (uint32_t)code << (4 * (e >> 1) + 16 * (e & 1));
            }
        }
    }
    reinterpret_cast<uint32_t*>(packed)[((size_t)tile * p.blocks + block) * 256 + i] = word;
}

// The product. A wave takes 128-column blocks of RT row tiles for NT tiles of 16
// tokens: y^T tile [16 rows][16 tokens] = W X^T by 16x16x32 FP16 matrix instructions,
// W the codes minus 8 (exact), X two planes h + l of x times a power of two. A
// group's sums are formed from 0 and join the row's by its scale in FP32, so a scale
// never rounds a weight. Eight waves split the columns and meet in LDS. Codes and
// scales of the next block are on their way while one is multiplied.
enum { WAVES = 8 };

struct Q4Args {
    const uint8_t* packed;
    Q4Shape p;
    const float* x;
    float* y;
    size_t x_stride, y_stride;
    uint32_t tokens, per;       // per: blocks of a wave
    const f16x8* planes;        // [token tile][block][32-column step][plane][lane]
    const float* factors;       // [token]: the power of two back
    float* part;                // [split][token][16 tiles] where blockIdx.z splits
};

// A block's codes and scales of RT tiles. PER: scales of a row in a block.
template <int PER, int RT>
struct Q4Block {
    u32x4 w[RT];
    uint32_t s[RT][2 * PER];   // BF16 pairs: group j's rows 4 g .. + 3 in words 2 j, 2 j + 1

    __device__ __forceinline__ void load(const Q4Args& a, uint32_t tile, uint32_t block,
        uint32_t lane)
    {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            // Tiles past the last repeat it and are not stored.
            const uint32_t mine = tile + t < a.p.tiles ? tile + t : a.p.tiles - 1;
            const size_t at = (size_t)mine * a.p.blocks + block;
            w[t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.packed) +
                at * 64 + lane);
            const uint32_t* scale = reinterpret_cast<const uint32_t*>(a.packed +
                q4_scales_at(a.p) + at * (32 * PER)) + (lane >> 4) * (2 * PER);
#pragma unroll
            for (int i = 0; i < 2 * PER; i++) {
                s[t][i] = scale[i];
            }
        }
    }
};

template <int PER, int RT, int NT>
__device__ __forceinline__ void q4_multiply(const Q4Block<PER, RT>& b, const f16x8 (&x)[NT][4][2],
    floatx4 (&acc)[RT][NT], const NibbleMasks& mask)
{
#pragma unroll
    for (int t = 0; t < RT; t++) {
        floatx4 d[NT];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const f16x8 w = codes_minus8(b.w[t][j], mask);
            constexpr int STEPS = 4 / PER;   // 32-column steps of a group
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (j % STEPS == 0) {
                    d[n] = (floatx4){0, 0, 0, 0};
                }
                d[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x[n][j][0], d[n], 0, 0, 0);
                d[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x[n][j][1], d[n], 0, 0, 0);
            }
            if (j % STEPS == STEPS - 1) {
                const uint32_t low = b.s[t][2 * (j / STEPS)], high = b.s[t][2 * (j / STEPS) + 1];
                const float s[4] = {bf16_to_f32(low & 0xffffu),
                    __uint_as_float(low & 0xffff0000u), bf16_to_f32(high & 0xffffu),
                    __uint_as_float(high & 0xffff0000u)};
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[t][n][i] = __builtin_fmaf(s[i], d[n][i], acc[t][n][i]);
                    }
                }
            }
        }
    }
}

// The eight waves' sums of RT tiles (each times its factor) to y.
template <int RT>
__device__ __forceinline__ void q4_store(const Q4Args& a, floatx4* joined,
    const floatx4 (&acc)[RT][1], float factor, uint32_t tile)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        floatx4 v = acc[t][0];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] *= factor;
        }
        joined[(t * WAVES + wave) * 64 + lane] = v;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < RT * 64; i += 64 * WAVES) {
        const uint32_t l = i & 63, t = i >> 6;
        floatx4 v = joined[t * WAVES * 64 + l];
#pragma unroll
        for (int w = 1; w < WAVES; w++) {
            v += joined[(t * WAVES + w) * 64 + l];
        }
        const uint32_t token = l & 15, row = (tile + t) * 16 + 4 * (l >> 4);
        if (token >= a.tokens) {
            continue;
        }
        float* y = a.y + token * a.y_stride + row;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (row + e < a.p.rows) {
                y[e] = v[e];
            }
        }
    }
}

// Few tokens: every wave turns its own columns of x into planes in LDS first (its own
// power of two for each token), with the first block's codes on their way. At most
// STAGED (token, block) pairs a wave, 512 bytes each; no scratch and one launch.
enum { STAGED = 32 };

// LDS: the planes, then the waves' sums.
static size_t q4_few_lds(uint32_t tokens, uint32_t per, uint32_t rt)
{
    const size_t planes = (size_t)WAVES * tokens * per * 512, sums = (size_t)rt * WAVES * 1024;
    return planes > sums ? planes : sums;
}

template <int PER, int RT>
__global__ void __launch_bounds__(64 * WAVES)
k_q4_few(Q4Args a)
{
    extern __shared__ floatx4 shared[];
    __shared__ uint32_t most[WAVES][16];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x * RT, tokens = a.tokens;
    const uint32_t first = wave * a.per;
    // [block][step][plane][g][token]
    f16x8* planes = reinterpret_cast<f16x8*>(shared) + wave * tokens * a.per * 32;
    const uint32_t end = first + a.per < a.p.blocks ? first + a.per : a.p.blocks;
    // Chunks of eight columns: lane l takes chunks l, l + 64 .. of (token, chunk).
    constexpr int EACH = STAGED / 4;
    const uint32_t width = a.per * 16, used = tokens * width;
    const float inverse = 1.0f / (float)width;
    float v[EACH][8];
    uint32_t token[EACH], chunk[EACH];
    if (lane < 16) {
        most[wave][lane] = 0;
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        if (64u * i >= used) {
            break;
        }
        const uint32_t id = 64 * i + lane;
        token[i] = (uint32_t)(((float)id + 0.5f) * inverse);   // exact: ids are below 2^10
        chunk[i] = id - token[i] * width;
        const uint32_t col = first * 128 + chunk[i] * 8;
        if (token[i] < tokens && col < a.p.cols) {
            const float* x = a.x + token[i] * a.x_stride + col;
            const float4 p = load4(x), q = load4(x + 4);
            v[i][0] = p.x, v[i][1] = p.y, v[i][2] = p.z, v[i][3] = p.w;
            v[i][4] = q.x, v[i][5] = q.y, v[i][6] = q.z, v[i][7] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[i][e] = 0;
            }
        }
    }
    Q4Block<PER, RT> now;
    if (first < end) {
        now.load(a, tile, first, lane);
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        if (64u * i >= used) {
            break;
        }
        uint32_t m = 0;   // magnitudes order as their bits; an Inf or NaN is the largest
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t bits = __float_as_uint(v[i][e]) & 0x7fffffffu;
            m = m > bits ? m : bits;
        }
        if (token[i] < tokens) {
            atomicMax(&most[wave][token[i]], m);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        if (64u * i >= used) {
            break;
        }
        if (token[i] < tokens) {
            const float up = exp2i(row_exponent(__uint_as_float(most[wave][token[i]])));
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                s[e] = v[i][e] * up;
            }
            f16x8 hi, lo;
            planes8(s, hi, lo);
            // Chunk: block, step j and g in turn.
            f16x8* to = planes + ((chunk[i] >> 2) * 8 + (chunk[i] & 3)) * tokens + token[i];
            to[0] = hi;
            to[4 * tokens] = lo;
        }
    }
    __syncthreads();
    const NibbleMasks mask;
    const uint32_t mine = (lane & 15) < tokens ? lane & 15 : tokens - 1;
    float factor[1] = {exp2i(-row_exponent(__uint_as_float(most[wave][mine])))};
    floatx4 acc[RT][1];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        acc[t][0] = (floatx4){0, 0, 0, 0};
    }
    for (uint32_t b = first; b < end; b++) {
        Q4Block<PER, RT> next = now;
        if (b + 1 < end) {
            next.load(a, tile, b + 1, lane);
        }
        f16x8 x[1][4][2];
#pragma unroll
        for (int j = 0; j < 4; j++) {
#pragma unroll
            for (int plane = 0; plane < 2; plane++) {
                x[0][j][plane] = planes[(((b - first) * 4 + j) * 8 + plane * 4 + g) * tokens +
                    mine];
            }
        }
        q4_multiply<PER, RT, 1>(now, x, acc, mask);
        now = next;
    }
    __syncthreads();   // the planes are done with
    q4_store<RT>(a, shared, acc, factor[0], tile);
}

// More tokens: planes made once, by one workgroup a token. A thread holds its first
// two chunks of eight columns (all of them up to 16384 columns) between the two passes.
__global__ void __launch_bounds__(1024)
k_q4_planes(Q4Args a, f16x8* planes, float* factors)
{
    __shared__ uint32_t most[16];
    const uint32_t token = blockIdx.x, chunks = a.p.blocks * 16;
    const float* x = a.x + token * a.x_stride;
    auto load = [&](uint32_t chunk, float (&v)[8]) __attribute__((always_inline)) {
        if (chunk * 8 < a.p.cols) {
            const float4 p = load4(x + chunk * 8), q = load4(x + chunk * 8 + 4);
            v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
            v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = 0;
            }
        }
    };
    uint32_t m = 0;
    auto largest = [&](const float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t bits = __float_as_uint(v[e]) & 0x7fffffffu;
            m = m > bits ? m : bits;
        }
    };
    float v0[8], v1[8];
    load(threadIdx.x, v0);
    load(threadIdx.x + 1024, v1);
    largest(v0);
    largest(v1);
    for (uint32_t c = threadIdx.x + 2048; c < chunks; c += 1024) {
        float v[8];
        load(c, v);
        largest(v);
    }
    for (int s = 32; s; s >>= 1) {
        const uint32_t o = __shfl_xor(m, s);
        m = m > o ? m : o;
    }
    if ((threadIdx.x & 63) == 0) {
        most[threadIdx.x >> 6] = m;
    }
    __syncthreads();
    for (int w = 0; w < 16; w++) {
        m = m > most[w] ? m : most[w];
    }
    const int e2 = row_exponent(__uint_as_float(m));
    const float up = exp2i(e2);
    if (threadIdx.x == 0) {
        factors[token] = exp2i(-e2);
    }
    auto store = [&](uint32_t c, const float (&v)[8]) __attribute__((always_inline)) {
        if (c >= chunks) {
            return;
        }
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            s[e] = v[e] * up;
        }
        f16x8 hi, lo;
        planes8(s, hi, lo);
        f16x8* to = planes + ((size_t)(token >> 4) * a.p.blocks * 8 + (c >> 2) * 2) * 64 +
            16 * (c & 3) + (token & 15);
        to[0] = hi;
        to[64] = lo;
    };
    store(threadIdx.x, v0);
    store(threadIdx.x + 1024, v1);
    for (uint32_t c = threadIdx.x + 2048; c < chunks; c += 1024) {
        float v[8];
        load(c, v);
        store(c, v);
    }
}

// Four waves with two row tiles each share the planes of NT token tiles in LDS, which
// is filled a block ahead by loads straight into it; codes come a block ahead too.
// grid (8-tile row groups, token tiles / NT, column splits). Planes of tokens past the
// last hold anything: a column's sums are its own and these are not stored.
template <int PER, int NT>
__global__ void __launch_bounds__(256)
k_q4_many(Q4Args a)
{
    constexpr int RT = 2, BLOCK = NT * 512;   // f16x8 of a block's planes
    __shared__ f16x8 shared[2][BLOCK];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = (blockIdx.x * 4 + wave) * RT, tile0 = blockIdx.y * NT;
    const uint32_t first = blockIdx.z * a.per;
    const uint32_t end = first + a.per < a.p.blocks ? first + a.per : a.p.blocks;
    const uint32_t last = (a.tokens - 1) >> 4;
    auto stage = [&](uint32_t block, f16x8* to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) {
            // 256 f16x8: half a token tile's block; a wave writes 1 KiB in lane order.
            const uint32_t n = i / 2, at = tile0 + n < last ? tile0 + n : last;
            const f16x8* from = a.planes + ((size_t)at * a.p.blocks + block) * 512 +
                (i & 1) * 256 + threadIdx.x;
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)from,
                (__attribute__((address_space(3))) void*)(to + i * 256 + wave * 64), 16, 0, 0);
        }
    };
    floatx4 acc[RT][NT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            acc[t][n] = (floatx4){0, 0, 0, 0};
        }
    }
    const NibbleMasks mask;
    Q4Block<PER, RT> now;
    now.load(a, tile, first, lane);
    stage(first, shared[0]);
    for (uint32_t b = first; b < end; b++) {
        Q4Block<PER, RT> next = now;
        __syncthreads();   // this block's planes are there, the other buffer is free
        if (b + 1 < end) {
            next.load(a, tile, b + 1, lane);
            stage(b + 1, shared[(b + 1 - first) & 1]);
        }
        const f16x8* planes = shared[(b - first) & 1] + lane;
        f16x8 x[NT][4][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[n][j][0] = planes[n * 512 + j * 128];
                x[n][j][1] = planes[n * 512 + j * 128 + 64];
            }
        }
        q4_multiply<PER, RT, NT>(now, x, acc, mask);
        now = next;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t token = (tile0 + n) * 16 + (lane & 15);
        if (token >= a.tokens) {
            continue;
        }
        const float factor = a.factors[token];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const uint32_t row = (tile + t) * 16 + 4 * g;
            if (tile + t >= a.p.tiles) {
                continue;
            }
            floatx4 v = acc[t][n];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] *= factor;
            }
            if (gridDim.z > 1) {
                const size_t width = (size_t)a.p.tiles * 16;
                *reinterpret_cast<floatx4*>(a.part +
                    ((size_t)blockIdx.z * a.tokens + token) * width + row) = v;
                continue;
            }
            float* y = a.y + token * a.y_stride + row;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (row + e < a.p.rows) {
                    y[e] = v[e];
                }
            }
        }
    }
}

// y = the sum of the column splits' parts, in their order.
__global__ void __launch_bounds__(256)
k_q4_join(Q4Args a, uint32_t splits)
{
    const uint32_t row = blockIdx.x * 256 + threadIdx.x, token = blockIdx.y;
    if (row >= a.p.rows) {
        return;
    }
    const size_t width = (size_t)a.p.tiles * 16, step = width * a.tokens;
    const float* part = a.part + token * width + row;
    float v = part[0];
    for (uint32_t i = 1; i < splits; i++) {
        v += part[i * step];
    }
    a.y[token * a.y_stride + row] = v;
}

}  // namespace lh

using namespace lh;

extern "C" int lh_launch_q4_pack(const uint8_t* codes, const uint16_t* scales, uint32_t rows,
    uint32_t cols, uint32_t group, uint8_t* packed, hipStream_t s)
{
    const Q4Shape p = q4_shape(rows, cols, group);
    hipLaunchKernelGGL(k_q4_pack, dim3(p.tiles, p.blocks), dim3(256), 0, s, codes, scales, p,
        packed);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

extern "C" int lh_launch_q4_quantize(const float* w, uint32_t rows, uint32_t cols, uint32_t group,
    uint8_t* packed, hipStream_t s)
{
    const Q4Shape p = q4_shape(rows, cols, group);
    hipLaunchKernelGGL(k_q4_quantize, dim3(p.tiles, p.blocks), dim3(256), 0, s, w, p, packed);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// How a product runs. few: planes in the kernel itself, rt row tiles a workgroup.
// Otherwise nt token tiles a workgroup and `splits` column splits, with scratch for
// planes, factors and parts.
struct Q4Plan {
    bool few;
    uint32_t nt, rt, splits, per;
    size_t planes, factors;   // bytes
};

// Workgroups to aim for, one a unit (down of 45 tokens: 21 us with 256, 25 with 128,
// 24 with 384); the row tiles of a k_q4_many workgroup.
enum { Q4_WORKGROUPS = 256, MANY_TILES = 8 };

static Q4Plan q4_plan(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    const uint32_t blocks = (cols + 127) / 128, tiles = (rows + 15) / 16;
    Q4Plan p = {};
    p.per = (blocks + WAVES - 1) / WAVES;
    p.splits = 1;
    p.few = tokens <= 16 && tokens * p.per <= STAGED;
    if (p.few) {
        // Row tiles of a workgroup: one round of workgroups, two on a unit where their
        // LDS fits twice.
        const uint32_t units = q4_few_lds(tokens, p.per, 1) > 80 * 1024 ? 256 : 512;
        const uint32_t rt = (tiles + units - 1) / units;
        p.rt = rt < 6 ? rt : 6;
        return p;
    }
    const uint32_t tt = (tokens + 15) / 16;
    p.nt = tt < 4 ? tt : 4;
    const uint32_t groups = (tiles + MANY_TILES - 1) / MANY_TILES * ((tt + p.nt - 1) / p.nt);
    uint32_t splits = (Q4_WORKGROUPS + groups - 1) / groups;
    const uint32_t most = (blocks + 3) / 4;   // four blocks at least
    splits = splits < most ? splits : most;
    p.per = (blocks + splits - 1) / splits;
    p.splits = (blocks + p.per - 1) / p.per;
    p.planes = (size_t)tt * blocks * 8192;
    p.factors = lh_round16((size_t)tokens * 4);
    return p;
}

template <int PER>
static void q4_few(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    const dim3 grid((a.p.tiles + p.rt - 1) / p.rt), block(64 * WAVES);
    const size_t lds = q4_few_lds(a.tokens, p.per, p.rt);
    switch (p.rt) {
    case 1: hipLaunchKernelGGL((k_q4_few<PER, 1>), grid, block, lds, s, a); break;
    case 2: hipLaunchKernelGGL((k_q4_few<PER, 2>), grid, block, lds, s, a); break;
    case 3: hipLaunchKernelGGL((k_q4_few<PER, 3>), grid, block, lds, s, a); break;
    case 4: hipLaunchKernelGGL((k_q4_few<PER, 4>), grid, block, lds, s, a); break;
    case 5: hipLaunchKernelGGL((k_q4_few<PER, 5>), grid, block, lds, s, a); break;
    default: hipLaunchKernelGGL((k_q4_few<PER, 6>), grid, block, lds, s, a); break;
    }
}

template <int PER>
static void q4_many(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    const uint32_t tt = (a.tokens + 15) / 16;
    const dim3 grid((a.p.tiles + MANY_TILES - 1) / MANY_TILES, (tt + p.nt - 1) / p.nt, p.splits);
    const dim3 block(256);
    switch (p.nt) {
    case 1: hipLaunchKernelGGL((k_q4_many<PER, 1>), grid, block, 0, s, a); break;
    case 2: hipLaunchKernelGGL((k_q4_many<PER, 2>), grid, block, 0, s, a); break;
    case 3: hipLaunchKernelGGL((k_q4_many<PER, 3>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((k_q4_many<PER, 4>), grid, block, 0, s, a); break;
    }
}

template <int PER>
static void q4_product(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    if (p.few) {
        q4_few<PER>(p, a, s);
    } else {
        q4_many<PER>(p, a, s);
    }
}

// For any number of rows: splits appear below 256 workgroups and bring them to less
// than 512, of eight row tiles and (past 64 tokens more workgroups, not more tokens)
// 64 tokens, so their parts hold at most 512 * 8 * 16 rows of min(tokens, 64).
extern "C" size_t lh_q4_scratch_bytes(uint32_t cols, uint32_t tokens)
{
    const Q4Plan p = q4_plan(1, cols, tokens);
    if (p.few) {
        return 0;
    }
    const size_t parts = cols > 128 * 4 ? (size_t)512 * MANY_TILES * 16 * 4 : 0;
    return p.planes + p.factors + parts * (tokens < 64 ? tokens : 64);
}

extern "C" int lh_launch_q4_matvec(const uint8_t* packed, const float* x, size_t x_stride,
    float* y, size_t y_stride, uint32_t rows, uint32_t cols, uint32_t group, uint32_t tokens,
    uint8_t* scratch, hipStream_t s)
{
    const Q4Plan p = q4_plan(rows, cols, tokens);
    f16x8* planes = reinterpret_cast<f16x8*>(scratch);
    float* factors = reinterpret_cast<float*>(scratch + p.planes);
    const Q4Args a = {packed, q4_shape(rows, cols, group), x, y, x_stride, y_stride, tokens, p.per,
        planes, factors, reinterpret_cast<float*>(scratch + p.planes + p.factors)};
    if (!p.few) {
        hipLaunchKernelGGL(k_q4_planes, dim3(tokens), dim3(1024), 0, s, a, planes, factors);
        if (hipGetLastError() != hipSuccess) {
            return -1;
        }
    }
    switch (group) {
    case 32: q4_product<4>(p, a, s); break;
    case 64: q4_product<2>(p, a, s); break;
    default: q4_product<1>(p, a, s); break;
    }
    if (hipGetLastError() != hipSuccess) {
        return -1;
    }
    if (p.splits > 1) {
        hipLaunchKernelGGL(k_q4_join, dim3((rows + 255) / 256, tokens), dim3(256), 0, s, a,
            p.splits);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
