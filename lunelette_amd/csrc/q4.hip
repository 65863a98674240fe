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
// W the codes minus 8 (exact), X two planes h + l of x times a power of two: 22 bits of
// the largest x that shares the power (of a token's 128 columns, in k_q4_many of all of
// its columns). A group's sums are formed from 0 and join the row's by its scale in FP32,
// so a scale never rounds a weight. Codes and scales of the blocks to come are on their
// way while one is multiplied.
// Bound: the codes' bytes. Measured, cold weights: 131072 x 3072 (214 MB) for one token
// 50 us, 4.3 TB/s, for eight 54 us; 18432 x 3072 with groups of 32 (32 MB) 14 us for one
// token and for eight, 16 to 18 for 16, of which a launch and the first bytes' way are 5.
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
    float* part;                // [split][token][16 tiles] where columns are split
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

// The same of one block whose token columns have powers of two of their own: f[n] takes
// the block's sums back, in FP32 (a product with a power of two is exact). x(n, j, plane)
// reads an operand when it is needed.
template <int PER, int RT, int NT, class X>
__device__ __forceinline__ void q4_multiply_block(const Q4Block<PER, RT>& b, const X& x,
    const float (&f)[NT], floatx4 (&acc)[RT][NT], const NibbleMasks& mask)
{
    constexpr int STEPS = 4 / PER;   // 32-column steps of a group
    floatx4 sum[RT][NT], d[RT][NT];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f16x8 w[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            w[t] = codes_minus8(b.w[t][j], mask);
        }
        // Products that need one another stand four apart where there are as many.
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += 2) {
            constexpr int TWO = NT > 1 ? 2 : 1;
            f16x8 at[TWO][2];
#pragma unroll
            for (int i = 0; i < TWO && n0 + i < NT; i++) {
                at[i][0] = x(n0 + i, j, 0);
                at[i][1] = x(n0 + i, j, 1);
            }
#pragma unroll
            for (int plane = 0; plane < 2; plane++) {
#pragma unroll
                for (int i = 0; i < TWO && n0 + i < NT; i++) {
#pragma unroll
                    for (int t = 0; t < RT; t++) {
                        floatx4& to = d[t][n0 + i];
                        if (j % STEPS == 0 && plane == 0) {
                            to = (floatx4){0, 0, 0, 0};
                        }
                        to = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[t], at[i][plane], to, 0, 0,
                            0);
                    }
                }
            }
        }
        if (j % STEPS != STEPS - 1) {
            continue;
        }
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const uint32_t low = b.s[t][2 * (j / STEPS)], high = b.s[t][2 * (j / STEPS) + 1];
            const float s[4] = {bf16_to_f32(low & 0xffffu), __uint_as_float(low & 0xffff0000u),
                bf16_to_f32(high & 0xffffu), __uint_as_float(high & 0xffff0000u)};
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (PER * RT * NT > 24) {
                        // No registers for a block's sums. (The scale meets the sum first, as
                        // below: with f it may leave FP32's range where the sum is 0.)
                        acc[t][n][i] = __builtin_fmaf(s[i] * d[t][n][i], f[n], acc[t][n][i]);
                        continue;
                    }
                    sum[t][n][i] = j < STEPS ? s[i] * d[t][n][i]
                        : __builtin_fmaf(s[i], d[t][n][i], sum[t][n][i]);
                    if (j == 3) {
                        acc[t][n][i] = __builtin_fmaf(f[n], sum[t][n][i], acc[t][n][i]);
                    }
                }
            }
        }
    }
}

// Four rows of a token: to y, or to the split's part.
__device__ __forceinline__ void q4_put(const Q4Args& a, floatx4 v, uint32_t token, uint32_t row,
    uint32_t split, uint32_t splits)
{
    if (splits > 1) {
        *reinterpret_cast<floatx4*>(a.part +
            ((size_t)split * a.tokens + token) * a.p.tiles * 16 + row) = v;
        return;
    }
    float* y = a.y + token * a.y_stride + row;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (row + e < a.p.rows) {
            y[e] = v[e];
        }
    }
}

__device__ __forceinline__ void load_chunk(const float* x, float (&v)[8])
{
    const float4 p = load4(x), q = load4(x + 4);
    v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
    v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
}

// Planes of a token's chunk of eight columns (0 if it has none), where 16 lanes side by
// side have those of a block; its power of two back.
__device__ __forceinline__ float chunk_planes(float (&v)[8], bool used, f16x8& hi, f16x8& lo)
{
    if (!__all(used)) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = used ? v[e] : 0.0f;
        }
    }
    // A NaN takes no part and stays one in its plane.
    float f;
    asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(f) : "v"(v[0]), "v"(v[1]), "v"(v[2]));
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(f) : "v"(v[3]), "v"(v[4]));
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(f) : "v"(v[5]), "v"(v[6]));
    asm("v_max_f32 %0, %0, |%1|" : "+v"(f) : "v"(v[7]));
    uint32_t m = __float_as_uint(f);   // magnitudes order as their bits
    uint32_t o;   // the row's other lanes by rotations of 8, 4, 2 and 1
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x128, 0xf, 0xf, false), m = m > o ? m : o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x124, 0xf, 0xf, false), m = m > o ? m : o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x122, 0xf, 0xf, false), m = m > o ? m : o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x121, 0xf, 0xf, false), m = m > o ? m : o;
    const int e2 = row_exponent(__uint_as_float(m));
    const float up = exp2i(e2);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        v[e] *= up;
    }
    planes8(v, hi, lo);
    return exp2i(-e2);
}

// Few tokens: every wave turns its own columns of x into planes in LDS first, with the
// first DEPTH blocks' codes on their way, then takes row tiles in turn: the codes of
// the blocks to come, of the next tiles too, stay DEPTH ahead. At most STAGED (token,
// block) pairs a wave; no scratch and one launch.
// A pair's 512 bytes of planes are followed by 16 with its power of two back, which
// shifts the next token's to other banks.
enum { STAGED = 32, PAIR = 33 };   // PAIR: f16x8 of one

static size_t q4_few_lds(uint32_t tokens, uint32_t per, uint32_t rt)
{
    // The waves' sums of two turns, then the pairs.
    return (size_t)2 * rt * WAVES * 1024 + (size_t)WAVES * tokens * per * PAIR * 16;
}

template <int PER, int RT, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES)
k_q4_few(Q4Args a)
{
    extern __shared__ floatx4 shared[];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, tokens = a.tokens;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t first = wave * a.per;
    const uint32_t left = first < a.p.blocks ? a.p.blocks - first : 0;
    const uint32_t blocks = left < a.per ? left : a.per;
    floatx4* joined = shared;   // [turn][tile][wave][lane]
    // [block][token][step][plane][g] of the wave
    f16x8* planes = reinterpret_cast<f16x8*>(shared + 2 * RT * WAVES * 64) +
        wave * tokens * a.per * PAIR;
    const uint32_t pairs = tokens * blocks, stride = gridDim.x * RT;
    const float inverse = 1.0f / (float)tokens;
    Q4Block<PER, RT> ring[DEPTH];
    uint32_t load_tile = blockIdx.x * RT, load_block = 0;
    // Unconditional, as all loads here: after one that may not have been issued the
    // compiler can only wait for everything. Past the end the last tile comes again, a
    // wave without columns takes those of the first block and drops them.
    auto ask = [&](Q4Block<PER, RT>& to) __attribute__((always_inline)) {
        to.load(a, load_tile, blocks ? first + load_block : 0, lane);
        if (++load_block >= blocks) {
            load_block = 0;
            load_tile += load_tile + stride < a.p.tiles ? stride : 0;
        }
    };
    float v[4][8];
    bool used[4];
    auto load_x = [&](uint32_t base) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t pair = base + 4 * i + g;
            // Exact: pairs are below 2^10.
            const uint32_t block = (uint32_t)(((float)pair + 0.5f) * inverse);
            const uint32_t token = pair - block * tokens;
            const uint32_t col = (first + block) * 128 + (lane & 15) * 8;
            used[i] = pair < pairs && col < a.p.cols;
            load_chunk(a.x + (used[i] ? token * a.x_stride + col : 0), v[i]);
        }
    };
    auto make = [&](uint32_t base) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f16x8 hi, lo;
            const float back = chunk_planes(v[i], used[i], hi, lo);
            const uint32_t pair = base + 4 * i + g;
            if (pair < pairs) {
                // Chunk: step j and g in turn.
                f16x8* to = planes + pair * PAIR + (lane & 12) * 2 + (lane & 3);
                to[0] = hi;
                to[4] = lo;
                if ((lane & 15) == 0) {
                    *reinterpret_cast<float*>(planes + pair * PAIR + 32) = back;
                }
            }
        }
    };
    load_x(0);
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
        __builtin_amdgcn_sched_barrier(0);   // in their order, which the waits go by
        ask(ring[d]);
    }
    make(0);
    for (uint32_t base = 16; base < pairs; base += 16) {
        load_x(base);
        make(base);
    }
    // Only this wave reads them.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const NibbleMasks mask;
    const uint32_t mine = (lane & 15) < tokens ? lane & 15 : tokens - 1;
    const f16x8* planes_mine = planes + mine * PAIR;
    uint32_t tile = blockIdx.x * RT, block = 0;
    floatx4 acc[RT][1];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        acc[t][0] = (floatx4){0, 0, 0, 0};
    }
    // The eight waves' sums of the tiles to y.
    auto store = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            joined[(t * WAVES + wave) * 64 + lane] = acc[t][0];
            acc[t][0] = (floatx4){0, 0, 0, 0};
        }
        // Waits for LDS alone, not for the codes on their way. The next turn writes the
        // other half; by the one after it all have read this one.
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        if (wave < RT) {
            floatx4 v = joined[wave * WAVES * 64 + lane];
#pragma unroll
            for (int w = 1; w < WAVES; w++) {
                v += joined[(wave * WAVES + w) * 64 + lane];
            }
            const uint32_t token = lane & 15, row = (tile + wave) * 16 + 4 * g;
            float* y = a.y + token * a.y_stride + row;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (token < tokens && row + e < a.p.rows) {
                    y[e] = v[e];
                }
            }
        }
        joined = joined == shared ? shared + RT * WAVES * 64 : shared;
        tile += stride;
    };
    if (blocks == 0) {
        while (tile < a.p.tiles) {
            store();
        }
        return;
    }
    while (true) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const f16x8* pair = planes_mine + block * tokens * PAIR;
            auto x = [&](int, int j, int plane) __attribute__((always_inline)) {
                return pair[j * 8 + plane * 4 + g];
            };
            const float f[1] = {*reinterpret_cast<const float*>(pair + 32)};
            q4_multiply_block<PER, RT, 1>(ring[d], x, f, acc, mask);
            // The scales are done with before they are loaded over: moved to registers of
            // their own, the loop's end would wait for the loads to move them back.
            __builtin_amdgcn_sched_barrier(0);
            ask(ring[d]);
            if (++block == blocks) {
                store();
                block = 0;
                if (tile >= a.p.tiles) {
                    return;
                }
            }
        }
    }
}

// Some tokens: eight waves, two row tiles each, in two halves that take every
// second block. The blocks' planes are shared in LDS, made for the next two blocks while
// two are multiplied, with codes two turns ahead. grid (8-tile row groups, column
// splits, NT token tiles). Token t of step j's g is at place (t + g + 4 j) % 16 of its
// sixteen, so that a token's sixteen chunks go to different banks.
// Bound by its vector instructions, half of which make the planes: 45 tokens, 3072 x 9216
// (14 MB) 14 us and 4 for the join.
template <int PER, int NT>
__global__ void __launch_bounds__(512, NT == 1 ? 4 : 2)
k_q4_some(Q4Args a)
{
    constexpr int RT = 2, BLOCK = NT * 512;   // f16x8 of a block's planes
    extern __shared__ floatx4 shared[];
    f16x8* planes = reinterpret_cast<f16x8*>(shared);                   // [turn][half][BLOCK]
    float* factors = reinterpret_cast<float*>(planes + 4 * BLOCK);      // [turn][half][NT * 16]
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave >> 2;
    const uint32_t tile = (blockIdx.x * 4 + (wave & 3)) * RT;
    const uint32_t first = blockIdx.y * a.per;
    const uint32_t end = first + a.per < a.p.blocks ? first + a.per : a.p.blocks;
    const uint32_t chunk = threadIdx.x & 15, row = (threadIdx.x >> 4) & 15;
    const uint32_t token0 = blockIdx.z * NT * 16;
    float v[NT][8];
    bool used[NT];
    auto load_x = [&](uint32_t block) __attribute__((always_inline)) {
        const uint32_t col = (block + half) * 128 + chunk * 8;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint32_t token = token0 + n * 16 + row;
            const bool real = token < a.tokens && block + half < end && col < a.p.cols;
            load_chunk(a.x + (real ? token * a.x_stride + col : 0), v[n]);
            used[n] = real;
        }
    };
    auto make = [&](uint32_t turn) __attribute__((always_inline)) {
        f16x8* to = planes + (turn * 2 + half) * BLOCK + (chunk >> 2) * 128 + (chunk & 3) * 16 +
            ((row + (chunk & 3) + 4 * (chunk >> 2)) & 15);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            f16x8 hi, lo;
            const float back = chunk_planes(v[n], used[n], hi, lo);
            to[n * 512] = hi;
            to[n * 512 + 64] = lo;
            if (chunk == 0) {
                factors[(turn * 2 + half) * NT * 16 + n * 16 + row] = back;
            }
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
    // Loads are unconditional, as in k_q4_few: blocks past the end are the last one again.
    auto ask = [&](Q4Block<PER, RT>& to, uint32_t block) __attribute__((always_inline)) {
        to.load(a, tile, block + half < end ? block + half : end - 1, lane);
    };
    load_x(first);
    Q4Block<PER, RT> ring[2];
    __builtin_amdgcn_sched_barrier(0);   // in their order, which the waits go by
    ask(ring[0], first);
    __builtin_amdgcn_sched_barrier(0);
    ask(ring[1], first + 2);
    __builtin_amdgcn_sched_barrier(0);
    make(0);
    for (uint32_t b = first; b < end; b += 4) {
#pragma unroll
        for (int d = 0; d < 2; d++) {
            const uint32_t at = b + 2 * d;
            if (at >= end) {
                break;
            }
            // Planes of this turn are there and the other turn's are done with; codes on
            // their way go on.
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            load_x(at + 2);
            if (at + half < end) {
                const f16x8* from = planes + (d * 2 + half) * BLOCK + g * 16;
                auto x = [&](int n, int j, int plane) __attribute__((always_inline)) {
                    return from[n * 512 + j * 128 + plane * 64 + ((lane + g + 4 * j) & 15)];
                };
                float f[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    f[n] = factors[(d * 2 + half) * NT * 16 + n * 16 + (lane & 15)];
                }
                q4_multiply_block<PER, RT, NT>(ring[d], x, f, acc, mask);
            }
            __builtin_amdgcn_sched_barrier(0);   // as in k_q4_few
            ask(ring[d], at + 4);
            make(1 - d);
        }
    }
    // The second half's sums join the first's.
    __syncthreads();
    floatx4* joined = shared + (wave & 3) * RT * NT * 64 + lane;
    if (half == 1) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                joined[(t * NT + n) * 64] = acc[t][n];
            }
        }
    }
    __syncthreads();
    if (half == 1) {
        return;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t token = token0 + n * 16 + (lane & 15);
        if (token >= a.tokens) {
            continue;
        }
#pragma unroll
        for (int t = 0; t < RT; t++) {
            if (tile + t < a.p.tiles) {
                q4_put(a, acc[t][n] + joined[(t * NT + n) * 64], token, (tile + t) * 16 + 4 * g,
                    blockIdx.y, gridDim.y);
            }
        }
    }
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

// Four waves with two row tiles each share the planes of four token tiles in LDS, which
// is filled a block ahead by loads straight into it; codes come a block ahead too.
// grid (8-tile row groups, token tiles / 4, column splits). Planes of tokens past the
// last hold anything: a column's sums are its own and these are not stored.
template <int PER>
__global__ void __launch_bounds__(256)
k_q4_many(Q4Args a)
{
    constexpr int RT = 2, NT = 4, BLOCK = NT * 512;   // f16x8 of a block's planes
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
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's part of the planes
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
            q4_put(a, v, token, row, blockIdx.z, gridDim.z);
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
    return (int)hipGetLastError();
}

extern "C" int lh_launch_q4_quantize(const float* w, uint32_t rows, uint32_t cols, uint32_t group,
    uint8_t* packed, hipStream_t s)
{
    const Q4Shape p = q4_shape(rows, cols, group);
    hipLaunchKernelGGL(k_q4_quantize, dim3(p.tiles, p.blocks), dim3(256), 0, s, w, p, packed);
    return (int)hipGetLastError();
}

// How a product runs: few tokens, some, or many. rt row tiles a workgroup of
// k_q4_few, of which there are `groups`; otherwise nt token tiles a workgroup and `splits`
// column splits, with scratch for their parts and, past 64 tokens, planes and factors.
enum Q4Way { Q4_FEW, Q4_SOME, Q4_MANY };
struct Q4Plan {
    Q4Way way;
    uint32_t nt, rt, groups, splits, per;
    size_t planes, factors;   // bytes
};

// The row tiles of a k_q4_some or k_q4_many workgroup. The first makes its planes again
// for every 8 row tiles and 64 tokens, the second reads those of a launch of its own: the
// first up to 64 tokens (64 tokens, 3072 x 4096: 16.5 us against 19.8), and up to 128 where
// there are at most SOME_TILES row tiles (100 tokens: 6144 x 3072 26 us against 28, 18432 x
// 3072 88 against 68).
// START and JOIN: what a workgroup's start and the launch that joins splits cost, in
// blocks (2 to 8 give the same times).
enum { MANY_TILES = 8, SOME_TILES = 512, START = 3, JOIN = 3 };

static Q4Plan q4_plan(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    const uint32_t blocks = (cols + 127) / 128, tiles = (rows + 15) / 16;
    Q4Plan p = {};
    p.per = (blocks + WAVES - 1) / WAVES;
    p.splits = 1;
    if (tokens <= 16 && tokens * p.per <= STAGED) {
        p.way = Q4_FEW;
        // Two row tiles use an operand twice, which pays once a workgroup has many turns
        // (8 tokens, 131072 rows of 3072: 54 us against 58; 18432 rows: 14 both; 4 tokens,
        // 3072 rows of 4096: 5.6 with one, 6.7 with two). More than 24 pairs leave no room
        // for their sums.
        p.rt = tiles > 2048 && tokens * p.per <= 24 ? 2 : 1;
        // One round of workgroups, two on a unit where their LDS fits twice, with as many
        // turns each.
        const uint32_t units = q4_few_lds(tokens, p.per, p.rt) > 80 * 1024 ? 256 : 512;
        const uint32_t groups = (tiles + p.rt - 1) / p.rt, turns = (groups + units - 1) / units;
        p.groups = (groups + turns - 1) / turns;
        return p;
    }
    const uint32_t tt = (tokens + 15) / 16, token_groups = (tt + 3) / 4;
    p.way = token_groups == 1 || (token_groups == 2 && tiles <= SOME_TILES) ? Q4_SOME : Q4_MANY;
    p.nt = p.way == Q4_SOME ? (tt + token_groups - 1) / token_groups : 4;
    const uint32_t groups = (tiles + MANY_TILES - 1) / MANY_TILES * token_groups;
    // Workgroups that run at once: registers leave room for one of k_q4_some's on a unit
    // past one token tile.
    const uint32_t slots = p.way == Q4_SOME && p.nt > 1 ? 256 : 512;
    uint32_t best = ~0u;
    const uint32_t most = (blocks + 3) / 4;   // four blocks at least
    for (uint32_t i = 1; i <= most && (i == 1 || groups * i <= 512); i++) {
        const uint32_t per = (blocks + i - 1) / i;
        const uint32_t cost = (groups * i + slots - 1) / slots * (per + START) + (i > 1 ? JOIN : 0);
        if (cost < best) {
            best = cost;
            p.per = per;
        }
    }
    p.splits = (blocks + p.per - 1) / p.per;
    if (token_groups > 1) {   // (whatever the rows are: scratch is sized without them)
        p.planes = (size_t)tt * blocks * 8192;
        p.factors = lh_round16((size_t)tokens * 4);
    }
    return p;
}

template <int PER>
static void q4_few(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    const dim3 grid(p.groups), block(64 * WAVES);
    const size_t lds = q4_few_lds(a.tokens, p.per, p.rt);
    if (p.rt == 1) {
        hipLaunchKernelGGL((k_q4_few<PER, 1, 4>), grid, block, lds, s, a);
    } else {
        hipLaunchKernelGGL((k_q4_few<PER, 2, 2>), grid, block, lds, s, a);
    }
}

template <int PER, int NT>
static void q4_some_of(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    const size_t lds = (size_t)4 * NT * (8192 + 64);
    hipLaunchKernelGGL((k_q4_some<PER, NT>), dim3((a.p.tiles + MANY_TILES - 1) / MANY_TILES,
        p.splits, (a.tokens + NT * 16 - 1) / (NT * 16)), dim3(512), lds, s, a);
}

template <int PER>
static void q4_some(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    switch (p.nt) {
    case 1: q4_some_of<PER, 1>(p, a, s); break;
    case 2: q4_some_of<PER, 2>(p, a, s); break;
    case 3: q4_some_of<PER, 3>(p, a, s); break;
    default: q4_some_of<PER, 4>(p, a, s); break;
    }
}

template <int PER>
static void q4_many(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    const uint32_t tt = (a.tokens + 15) / 16;
    const dim3 grid((a.p.tiles + MANY_TILES - 1) / MANY_TILES, (tt + p.nt - 1) / p.nt, p.splits);
    const dim3 block(256);
    hipLaunchKernelGGL((k_q4_many<PER>), grid, block, 0, s, a);
}

template <int PER>
static void q4_product(const Q4Plan& p, const Q4Args& a, hipStream_t s)
{
    switch (p.way) {
    case Q4_FEW: q4_few<PER>(p, a, s); break;
    case Q4_SOME: q4_some<PER>(p, a, s); break;
    default: q4_many<PER>(p, a, s); break;
    }
}

// For any number of rows: with column splits there are at most 512 workgroups, of eight
// row tiles and (past 64 tokens more workgroups, not more tokens) 64 tokens, so their
// parts hold at most 512 * 8 * 16 rows of min(tokens, 64).
extern "C" size_t lh_q4_scratch_bytes(uint32_t cols, uint32_t tokens)
{
    const Q4Plan p = q4_plan(1, cols, tokens);
    if (p.way == Q4_FEW) {
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
    if (p.way == Q4_MANY) {
        hipLaunchKernelGGL(k_q4_planes, dim3(tokens), dim3(1024), 0, s, a, planes, factors);
        if (const hipError_t e = hipGetLastError()) {
            return (int)e;
        }
    }
    switch (group) {
    case 32: q4_product<4>(p, a, s); break;
    case 64: q4_product<2>(p, a, s); break;
    default: q4_product<1>(p, a, s); break;
    }
    if (const hipError_t e = hipGetLastError()) {
        return (int)e;
    }
    if (p.splits > 1) {
        hipLaunchKernelGGL(k_q4_join, dim3((rows + 255) / 256, tokens), dim3(256), 0, s, a,
            p.splits);
    }
    return (int)hipGetLastError();
}
