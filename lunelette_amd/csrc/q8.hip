// Products of 8-bit rows with 8-bit weights (lh_q8_pack, lh_q8_quantize, lh_q8_matvec).
//
// Packed weights: tiles of 16 rows x 64 columns, row tile by row tile, the codes of
// all tiles first. A tile's 1 KiB holds for lane l = 16 g + r of a wave row r's columns
// 16 g .. 16 g + 15: the operand of a 16x16x64 matrix instruction. Then the FP32 scales
// of the rows. Rows and columns past the matrix have codes and scales of 0, so what
// the activations hold past their last column adds nothing.
#include "lh_mfma.h"
#include "lh_serving.h"

namespace lh {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct Q8Shape {
    uint32_t rows, cols, tiles, blocks;   // 16-row tiles, 64-column blocks
};

static Q8Shape q8_shape(uint32_t rows, uint32_t cols)
{
    return {rows, cols, (rows + 15) / 16, (cols + 63) / 64};
}

__device__ __forceinline__ const float* q8_scales(const uint8_t* packed, const Q8Shape& p)
{
    return reinterpret_cast<const float*>(packed + (size_t)p.tiles * p.blocks * 1024);
}

// A wave a tile: grid (tiles, blocks).
__global__ void __launch_bounds__(64)
k_q8_pack(const int8_t* __restrict__ codes, const float* __restrict__ scales, Q8Shape p,
    uint8_t* __restrict__ packed)
{
    const uint32_t lane = threadIdx.x, tile = blockIdx.x, block = blockIdx.y;
    const uint32_t row = tile * 16 + (lane & 15), col = block * 64 + 16 * (lane >> 4);
    u32x4 word = {0, 0, 0, 0};
    if (row < p.rows) {
        const int8_t* c = codes + (size_t)row * p.cols + col;
        for (uint32_t e = 0; e < 16; e++) {
            const uint32_t v = col + e < p.cols ? (uint8_t)c[e] : 0;
            word[e >> 2] |= v << (8 * (e & 3));
        }
    }
    reinterpret_cast<u32x4*>(packed)[((size_t)tile * p.blocks + block) * 64 + lane] = word;
    if (block == 0 && lane < 16) {
        const_cast<float*>(q8_scales(packed, p))[tile * 16 + lane] = row < p.rows ? scales[row] : 0;
    }
}

// A wave a row of the tiles, whose scale it forms first.
__global__ void __launch_bounds__(64)
k_q8_quantize(const float* __restrict__ w, Q8Shape p, uint8_t* __restrict__ packed)
{
    const uint32_t lane = threadIdx.x, row = blockIdx.x;
    const float* x = w + (size_t)row * p.cols;
    float most = 0;
    bool finite = true;
    if (row < p.rows) {
        for (uint32_t c = lane; c < p.cols; c += 64) {
            finite &= __builtin_isfinite(x[c]);
            most = fmaxf(most, fabsf(x[c]));
        }
    }
    const bool bad = !__all(finite);
    const float scale = (float)((double)wave_max64(most) / 127.0);
    if (lane == 0) {
        const_cast<float*>(q8_scales(packed, p))[row] = bad ? __builtin_nanf("") : scale;
    }
    for (uint32_t word = lane; word < p.blocks * 4; word += 64) {
        u32x4 v = {0, 0, 0, 0};
        if (row < p.rows && !bad && scale > 0) {
            for (uint32_t e = 0; e < 16; e++) {
                const uint32_t c = word * 16 + e;
                const double q = c < p.cols ? (double)x[c] / (double)scale : 0;
                const int code = (int)rint(fmin(fmax(q, -127.0), 127.0));
                v[e >> 2] |= (uint32_t)(uint8_t)code << (8 * (e & 3));
            }
        }
        reinterpret_cast<u32x4*>(packed)[((size_t)(row >> 4) * p.blocks + (word >> 2)) * 64 +
            16 * (word & 3) + (row & 15)] = v;
    }
}

struct Q8Args {
    const uint8_t* packed;
    Q8Shape p;
    const int8_t* x;
    const float* x_scales;
    float* y;
    size_t x_stride, y_stride;
    uint32_t tokens;
};

// A wave a tile of 16 rows and 16 tokens.
__global__ void __launch_bounds__(64)
k_q8_matvec(Q8Args a)
{
    const uint32_t lane = threadIdx.x, tile = blockIdx.x;
    const uint32_t token = blockIdx.y * 16 + (lane & 15), g = lane >> 4;
    const uint32_t mine = token < a.tokens ? token : a.tokens - 1;
    const int8_t* x = a.x + mine * a.x_stride;
    const i32x4* w = reinterpret_cast<const i32x4*>(a.packed) + (size_t)tile * a.p.blocks * 64;
    i32x4 acc = {0, 0, 0, 0};
    for (uint32_t b = 0; b < a.p.blocks; b++) {
        const uint32_t col = b * 64 + g * 16;
        // Words past the row's last meet codes of 0.
        const i32x4 v = *reinterpret_cast<const i32x4*>(x + (col < a.p.cols ? col : 0));
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b * 64 + lane], v, acc, 0, 0, 0);
    }
    if (token >= a.tokens) {
        return;
    }
    const float scale = a.x_scales[token];
    const float* ws = q8_scales(a.packed, a.p);
    for (uint32_t e = 0; e < 4; e++) {
        const uint32_t row = tile * 16 + 4 * g + e;
        if (row < a.p.rows) {
            a.y[token * a.y_stride + row] = scale * (ws[row] * (float)acc[e]);
        }
    }
}

}  // namespace lh

using namespace lh;

extern "C" int lh_launch_q8_pack(const int8_t* codes, const float* scales, uint32_t rows,
    uint32_t cols, uint8_t* packed, hipStream_t s)
{
    const Q8Shape p = q8_shape(rows, cols);
    hipLaunchKernelGGL(k_q8_pack, dim3(p.tiles, p.blocks), dim3(64), 0, s, codes, scales, p,
        packed);
    return (int)hipGetLastError();
}

extern "C" int lh_launch_q8_quantize(const float* w, uint32_t rows, uint32_t cols,
    uint8_t* packed, hipStream_t s)
{
    const Q8Shape p = q8_shape(rows, cols);
    hipLaunchKernelGGL(k_q8_quantize, dim3(p.tiles * 16), dim3(64), 0, s, w, p, packed);
    return (int)hipGetLastError();
}

extern "C" size_t lh_q8_scratch_bytes(uint32_t rows, uint32_t cols, uint32_t tokens)
{
    return 0;
}

extern "C" int lh_launch_q8_matvec(const uint8_t* packed, const int8_t* x, size_t x_stride,
    const float* x_scales, float* y, size_t y_stride, uint32_t rows, uint32_t cols,
    uint32_t tokens, uint8_t* scratch, hipStream_t s)
{
    const Q8Args a = {packed, q8_shape(rows, cols), x, x_scales, y, x_stride, y_stride, tokens};
    hipLaunchKernelGGL(k_q8_matvec, dim3(a.p.tiles, (tokens + 15) / 16), dim3(64), 0, s, a);
    return (int)hipGetLastError();
}
