// Rows of FP32 values rounded to 8-bit codes with a scale each (lh_q8_rows, lh_q8_silu,
// lh_q8_norm).
//
// v = x, SiLU(x) * second, or gamma (h / sqrt(mean h^2 + 1e-5)) with h = x + second;
// scale = max |v| / 127, code = rint(v / scale). A code next to a border between two hangs
// on v's last bits, so scales and codes are those of v in 64 bits. But 64 bits are
// formed only where they decide: a quotient in FP32 is off by less than 2^-13, so
// only one within 2^-12 of a border (one of 2000 to 4000) is formed again.
// Bound: a row's bytes, read once into registers and written once. Measured: the norm with
// the addition of 4096 rows of 3072 32.6 us, 5.0 TB/s (a large copy makes 4.7 to 5.2),
// 4096 plain rows of 4096 15.8 us, 5.3 TB/s, SwiGLU of 2048 rows of 9216 38.7 us, 4.4 TB/s
// (its exponential and two joins); one row of the norm 4.0. A row in memory twice, and in
// 64 bits throughout, took the norm 77 us. Rows that FP32 does not decide are in 64 bits
// here as well: SwiGLU with a gate below -80 in each row 106 us.
#include "lh_serving.h"
#include "lh_topk.h"

namespace lh {

// Over groups of 2 J lanes, the same bits in each.
template <int J>
__device__ __forceinline__ double add_lanes(double v, uint32_t lane)
{
    v += xor_double<J>(v, lane);
    if constexpr (J > 1) {
        v = add_lanes<J / 2>(v, lane);
    }
    return v;
}

template <int J>
__device__ __forceinline__ double most_lanes(double v, uint32_t lane)
{
    v = fmax(v, xor_double<J>(v, lane));
    if constexpr (J > 1) {
        v = most_lanes<J / 2>(v, lane);
    }
    return v;
}

template <int J>
__device__ __forceinline__ float most_lanes(float v, uint32_t lane)
{
    v = fmaxf(v, __uint_as_float(xor_word<J>(__float_as_uint(v), lane)));
    if constexpr (J > 1) {
        v = most_lanes<J / 2>(v, lane);
    }
    return v;
}

// The maximum (of values that are not NaN) over a row's W waves and, if asked for, the sum,
// in every lane. Each call of a workgroup has `shared` of its own.
template <int W, bool SUM, typename T>
__device__ __forceinline__ void join_row(double& sum, T& most, double (&shared)[2][W],
    uint32_t lane, uint32_t wave)
{
    sum = SUM ? add_lanes<32>(sum, lane) : sum;
    most = most_lanes<32>(most, lane);
    if constexpr (W > 1) {
        if (lane == 0) {
            shared[0][wave] = sum;
            shared[1][wave] = most;
        }
        __syncthreads();
        sum = SUM ? add_lanes<W / 2>(shared[0][lane % W], lane) : sum;
        most = most_lanes<W / 2>((T)shared[1][lane % W], lane);
    }
}

// SiLU(g) * u with an error below 2^-20 of itself or of 2^-60, for g above -80, |u| below
// 2^66 and results below 2^120. (Where g times the factor is subnormal it loses up to
// 2^-150, of which u makes 2^-84; the factor itself is no less than 2^-117.)
__device__ __forceinline__ float silu_near(float g, float u)
{
    const float e = exp_near(-fabsf(g)), part = __builtin_amdgcn_rcpf(1.0f + e);
    return g * (g < 0 ? e * part : part) * u;
}

__device__ __forceinline__ double silu_wide(float g, float u)
{
    return (double)g / (1.0 + exp(-(double)g)) * (double)u;
}

// A row's value at column c in 64 bits, r the norm's factor.
template <int KIND>
__device__ __forceinline__ double q8_wide(const lh_q8_source& a, size_t row, uint32_t c, float h,
    double r)
{
    if (KIND == LH_Q8_SILU) {
        return silu_wide(a.x[row * a.x_stride + c], a.second[row * a.second_stride + c]);
    }
    return KIND == LH_Q8_NORM ? (double)a.gamma[c] * (double)h * r : (double)h;
}

// The code, its sign in the bits above.
__device__ __forceinline__ uint32_t q8_code_wide(double v, float scale)
{
    return (uint32_t)(int)rint(fmin(fmax(v / (double)scale, -127.0), 127.0));
}

// Columns c .. c + 3 of a row; 0 past its end.
__device__ __forceinline__ void load_quad(const float* row, uint32_t c, uint32_t width,
    float (&v)[4])
{
    if (c + 3 < width) {
        const float4 f = load4(row + c);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[e] = c + e < width ? row[c + e] : 0.0f;
    }
}

__device__ __forceinline__ void store_codes(int8_t* to, uint32_t c, uint32_t width,
    const uint32_t (&code)[4])
{
    if (c + 3 < width) {
        // Byte 0 of each: the second operand's bytes have indexes 0 to 3, the first's 4 to 7.
        *reinterpret_cast<uint32_t*>(to + c) =
            __builtin_amdgcn_perm(__builtin_amdgcn_perm(code[3], code[2], 0x0c0c0400u),
                __builtin_amdgcn_perm(code[1], code[0], 0x0c0c0400u), 0x05040100u);
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; e++) {
        if (c + e < width) {
            to[c + e] = (int8_t)code[e];
        }
    }
}

// The row's h: x, or x + second.
template <int KIND>
__device__ __forceinline__ void load_h(const lh_q8_source& a, size_t row, uint32_t c,
    float (&h)[4])
{
    load_quad(a.x + row * a.x_stride, c, a.width, h);
    if (KIND == LH_Q8_NORM && a.second) {
        float s[4];
        load_quad(a.second + row * a.second_stride, c, a.width, s);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            h[e] += s[e];
        }
    }
}

__device__ __forceinline__ void store_h(const lh_q8_source& a, size_t row, uint32_t c,
    const float (&h)[4])
{
    float* to = a.sum + row * a.sum_stride;
    if (c + 3 < a.width) {
        store4(to + c, make_float4(h[0], h[1], h[2], h[3]));
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; e++) {
        if (c + e < a.width) {
            to[c + e] = h[e];
        }
    }
}

// Whether a maximum of magnitudes is below `to` and no NaN: by their bits, which are above
// infinity's for a NaN.
__device__ __forceinline__ bool below(float most, float to)
{
    return __float_as_uint(most) < __float_as_uint(to);
}

// A row in W waves, Q quads of columns a lane, all in registers.
template <int KIND, int W, int Q>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W)
k_q8_rows(lh_q8_source a)
{
    constexpr uint32_t ROWS = W == 1 ? 4 : 1, STEP = 256 * W;
    __shared__ double shared[KIND == LH_Q8_SILU ? 2 : 1][ROWS][2][W];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wave = all % W, mine = all / W;
    const uint32_t first = 256 * wave + 4 * lane;
    const size_t row = (size_t)blockIdx.x * ROWS + mine;
    if (row >= a.tokens) {
        return;   // of several rows in a workgroup, which meet at no barrier
    }
    float v[Q][4];
    double sum = 0, most = 0;
    bool bad = false;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        load_h<KIND>(a, row, first + q * STEP, v[q]);
    }
    // The norm's weights, from L2 a second time where registers do not hold them.
    constexpr bool HELD = KIND == LH_Q8_NORM && Q <= 4;
    float g[HELD ? Q : 1][4], u[KIND == LH_Q8_SILU ? Q : 1][4];
#pragma unroll
    for (int q = 0; q < Q; q++) {
        if (HELD) {
            load_quad(a.gamma, first + q * STEP, a.width, g[q]);
        }
        if (KIND == LH_Q8_SILU) {
            load_quad(a.second + row * a.second_stride, first + q * STEP, a.width, u[q]);
        }
    }
    // Largest magnitudes in FP32, NaN where there is one; the least gate, the largest up.
    float near = 0, quad[Q], least = 0, most_up = 0;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const uint32_t c = first + q * STEP;
        quad[q] = 0;
        if (KIND == LH_Q8_NORM && a.sum && c < a.width) {
            store_h(a, row, c, v[q]);
        }
        float (&w)[4] = g[HELD ? q : 0];
        if (KIND == LH_Q8_NORM && !HELD) {
            load_quad(a.gamma, c, a.width, w);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (KIND == LH_Q8_NORM) {
                const double h = v[q][e], value = (double)w[e] * h;
                sum += h * h;
                most = fmax(most, fabs(value));
                bad |= !(fabs(value) <= 1e300);
            } else {
                if (KIND == LH_Q8_SILU) {
                    least = fminf(least, v[q][e]);
                    most_up = fmaxf(most_up, fabsf(u[q][e]));
                    v[q][e] = silu_near(v[q][e], u[q][e]);
                }
                quad[q] = __builtin_elementwise_maximum(quad[q], fabsf(v[q][e]));
            }
        }
        near = __builtin_elementwise_maximum(near, quad[q]);
    }
    if (KIND == LH_Q8_NORM && W == 16) {
        // The codes' rare 64-bit values begin with the conversions that the sums took. The
        // compiler is not to see it: it would hold all of these until then, in 18 to 32
        // registers more. Up to 64 registers (four quads) a unit takes two rows at once: the
        // norm of 2048 rows of 9216 46.2 us, 55.4 with 70 registers. In fewer waves, of which
        // a unit takes several rows anyway, it was 11% faster (one wave) to 4% slower (eight).
#pragma unroll
        for (int q = 0; q < Q; q++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                asm("" : "+v"(v[q][e]));
            }
        }
    }
    const double inf = __builtin_inf();
    double r = 1;
    bool wide = false;   // the whole row in 64 bits
    if (KIND == LH_Q8_NORM) {
        most = bad ? inf : most;
        join_row<W, true>(sum, most, shared[0][mine], lane, wave);
        wide = !(most >= 0x1p-90 && most < 0x1p120);
        r = 1.0 / sqrt(sum / a.width + 1e-5);
        most = sum < inf ? most * r : inf;   // a NaN too
    } else if (KIND == LH_Q8_ROWS) {
        near = below(near, __builtin_inff()) ? near : __builtin_inff();
        join_row<W, false>(sum, near, shared[0][mine], lane, wave);
        most = near;
    } else {
        // First the largest in FP32 (beside what silu_near does not take, an Inf or NaN a larger
        // one still), then those near it in 64 bits. There an Inf or NaN gives one.
        const bool taken = least >= -80.0f && most_up < 0x1p66f && below(near, 0x1p120f);
        near = taken ? near : 0x1p121f;
        join_row<W, false>(sum, near, shared[0][mine], lane, wave);
        wide = !(near >= 0x1p-60f && near < 0x1p120f);
        const float from = near * (1 - 0x1p-18f);
        most = 0;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            if (wide || quad[q] >= from) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t c = first + q * STEP + e;
                    if ((wide || fabsf(v[q][e]) >= from) && c < a.width) {
                        const double value = fabs(q8_wide<KIND>(a, row, c, 0, 1));
                        most = fmax(most, value <= 1e300 ? value : inf);
                    }
                }
            }
        }
        join_row<W, false>(sum, most, shared[1][mine], lane, wave);
    }
    const float scale = (float)(most / 127.0);
    const bool fine = scale < __builtin_inff();
    if (lane == 0 && wave == 0) {
        a.scales[row] = fine ? scale : __builtin_nanf("");
    }
    // v times this is the quotient, off by a few parts of 2^23; where that leaves FP32's
    // range all of the row takes 64 bits.
    const bool some = fine && scale > 0;
    const float by = some ? (float)(r / (double)scale) : 0.0f;
    wide |= !(by >= 0x1p-100f && by <= 0x1p100f) || !(scale >= 0x1p-100f);
    wide &= some;
    // Added and taken away again it rounds to whole numbers, whose bits are then the lowest
    // of the sum.
    const float whole = 0x1.8p23f;
    int8_t* codes = a.codes + row * a.code_stride;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const uint32_t c = first + q * STEP;
        if (c >= a.width) {
            continue;
        }
        float (&weight)[4] = g[HELD ? q : 0];
        if (KIND == LH_Q8_NORM && !HELD) {
            load_quad(a.gamma, c, a.width, weight);
        }
        uint32_t code[4];
        float off[4], most_off = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float w = KIND == LH_Q8_NORM ? weight[e] * v[q][e] : v[q][e];
            const float t = w * by, rounded = t + whole;
            code[e] = some ? __float_as_uint(rounded) : 0;
            off[e] = fabsf(t - (rounded - whole));
            most_off = fmaxf(most_off, off[e]);
        }
        const float border = 0.5f - 0x1p-12f;
        if (wide || (some && most_off > border)) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if ((wide || off[e] > border) && c + e < a.width) {
                    code[e] = q8_code_wide(q8_wide<KIND>(a, row, c + e, v[q][e], r), scale);
                }
            }
        }
        store_codes(codes, c, a.width, code);
    }
}

// Rows that registers do not hold, column by column in 64 bits, twice.
template <int KIND>
__global__ void __launch_bounds__(1024)
k_q8_wide_rows(lh_q8_source a)
{
    __shared__ double shared[2][16];
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.x;
    double sum = 0, most = 0;
    for (uint32_t c = threadIdx.x; c < a.width; c += 1024) {
        float h = a.x[row * a.x_stride + c];
        float odd = h;
        if (KIND == LH_Q8_NORM) {
            h = a.second ? h + a.second[row * a.second_stride + c] : h;
            odd = h;
            if (a.sum) {
                a.sum[row * a.sum_stride + c] = h;
            }
            sum += (double)h * (double)h;
        } else if (KIND == LH_Q8_SILU) {
            odd = odd * 0.0f + a.second[row * a.second_stride + c] * 0.0f;
        }
        const double v = fabs(q8_wide<KIND>(a, row, c, h, 1));
        most = fmax(most, __builtin_isfinite(odd) && v <= 1e300 ? v : __builtin_inf());
    }
    join_row<16, true>(sum, most, shared, lane, wave);
    const double r = KIND == LH_Q8_NORM ? 1.0 / sqrt(sum / a.width + 1e-5) : 1.0;
    const float scale = (float)(most * r / 127.0);
    const bool fine = scale < __builtin_inff();
    if (threadIdx.x == 0) {
        a.scales[row] = fine ? scale : __builtin_nanf("");
    }
    // The same thread's columns as before: a sum in place is its own.
    for (uint32_t c = threadIdx.x; c < a.width; c += 1024) {
        uint32_t code = 0;
        if (fine && scale > 0) {
            float h = 0;
            if (KIND == LH_Q8_NORM && a.sum) {
                h = a.sum[row * a.sum_stride + c];
            } else if (KIND != LH_Q8_SILU) {
                h = a.x[row * a.x_stride + c];
                h = KIND == LH_Q8_NORM && a.second ? h + a.second[row * a.second_stride + c] : h;
            }
            code = q8_code_wide(q8_wide<KIND>(a, row, c, h, r), scale);
        }
        a.codes[row * a.code_stride + c] = (int8_t)code;
    }
}

template <int KIND, int W, int Q>
static void q8_rows(const lh_q8_source& a, hipStream_t s)
{
    constexpr uint32_t rows = W == 1 ? 4 : 1;
    hipLaunchKernelGGL((k_q8_rows<KIND, W, Q>), dim3((a.tokens + rows - 1) / rows),
        dim3(64 * W * rows), 0, s, a);
}

// Few waves with up to four quads a lane, where sixteen hold no row up to eight: 4096 rows of
// 3072 columns in four waves take 33.1 us (norm), 24.9 (SwiGLU) and 13.0 (plain), in twelve
// with one quad 35.0, 34.1 and 17.9. Waves that the four SIMDs do not share evenly take
// longer, three by 11%, nine by 29%.
template <int KIND>
static void q8_rows(const lh_q8_source& a, hipStream_t s)
{
    const uint32_t quads = (a.width + 255) / 256;   // of a lane in one wave
    switch (quads) {
    case 1: q8_rows<KIND, 1, 1>(a, s); return;
    case 2: q8_rows<KIND, 1, 2>(a, s); return;
    case 3: q8_rows<KIND, 1, 3>(a, s); return;
    case 4: q8_rows<KIND, 1, 4>(a, s); return;
    }
    if (quads <= 8) {
        q8_rows<KIND, 4, 2>(a, s);
    } else if (quads <= 12) {
        q8_rows<KIND, 4, 3>(a, s);
    } else if (quads <= 16) {
        q8_rows<KIND, 4, 4>(a, s);
    } else if (quads <= 24) {
        q8_rows<KIND, 8, 3>(a, s);
    } else if (quads <= 32) {
        q8_rows<KIND, 8, 4>(a, s);
    } else if (quads <= 48) {
        q8_rows<KIND, 16, 3>(a, s);
    } else if (quads <= 64) {
        q8_rows<KIND, 16, 4>(a, s);
    } else if (quads <= 96) {
        q8_rows<KIND, 16, 6>(a, s);
    } else {
        if constexpr (KIND != LH_Q8_NORM) {   // the norm's 64-bit values leave no registers
            if (quads <= 128) {
                q8_rows<KIND, 16, 8>(a, s);
                return;
            }
        }
        hipLaunchKernelGGL(k_q8_wide_rows<KIND>, dim3(a.tokens), dim3(1024), 0, s, a);
    }
}

}  // namespace lh

using namespace lh;

extern "C" int lh_launch_q8_rows(int kind, const lh_q8_source* rows, hipStream_t s)
{
    if (kind == LH_Q8_SILU) {
        q8_rows<LH_Q8_SILU>(*rows, s);
    } else if (kind == LH_Q8_NORM) {
        q8_rows<LH_Q8_NORM>(*rows, s);
    } else {
        q8_rows<LH_Q8_ROWS>(*rows, s);
    }
    return (int)hipGetLastError();
}
