// MXFP4 (microscaled 4-bit floating point): quantisation, dequantisation and
// products with a 4-bit weight, on gfx950.
//
// A block is 32 consecutive values of a row in 17 bytes: byte 0 the biased
// exponent e of the scale 2^(e - 127) (255: NaN), bytes 1..16 the codes, byte
// 1 + j holding value j in its low and value j + 16 in its high half.  A code
// is sign, two exponent bits and one mantissa bit: {0, .5, 1, 1.5, 2, 3, 4, 6}.
// gfx950 converts two codes of a byte at once in both directions and takes the
// scale's exponent field alone, so (e << 23) is the scale operand for every e
// (checked on the device: e = 0 is 2^-127; the down conversion rounds half to
// even and saturates at 6).
#include "../internal.h"
#include "device.h"

#include <algorithm>
#include <type_traits>

namespace wamx {

constexpr int kMxBytes = kMxBlockBytes;  // of one block

// 16 and 8 bytes at any address: one global load each.
struct __attribute__((packed, aligned(1))) any16 {
    uint32_t v[4];
};
struct __attribute__((packed, aligned(1))) any8 {
    uint32_t v[2];
};

// A block read as the five aligned dwords that hold its 17 bytes, `mis` bytes
// into the first (every dword holds a byte of the block, so none lies outside
// the tensor's pages).  As 16 + 1 bytes at their odd addresses the few-token
// products took 34% and 19% longer (4096 x 1 x 4096, 14336 x 48 x 4096).  Blocks
// four apart have one `mis`.
struct __attribute__((packed, aligned(4))) dwords4 {
    uint32_t v[4];
};
struct MxBlock {
    dwords4 lo;
    uint32_t hi;
};
__device__ __forceinline__ MxBlock mx_load(const void * aligned) {
    return {*(const dwords4 *) aligned, ((const uint32_t *) aligned)[4]};
}
__device__ __forceinline__ uint32_t mx_select(uint32_t mis) { return 0x04030201u + mis * 0x01010101u; }
__device__ __forceinline__ uint32_t mx_exponent(const MxBlock & b, uint32_t mis) {
    return (b.lo.v[0] >> (8 * mis)) & 255u;
}
// Dword i of the codes.
__device__ __forceinline__ uint32_t mx_codes(const MxBlock & b, int i, uint32_t select) {
    return __builtin_amdgcn_perm(i < 3 ? b.lo.v[i + 1] : b.hi, b.lo.v[i], select);
}

__device__ __forceinline__ float mx_scale(uint32_t e) { return __uint_as_float(e << 23); }

// Eight consecutive values as f32.
template <typename T>
__device__ __forceinline__ void load8(const T * p, float * v) {
    if constexpr (sizeof(T) == 4) {
        const any16 a = *(const any16 *) p, b = *(const any16 *) (p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(a.v[i]);
            v[4 + i] = __uint_as_float(b.v[i]);
        }
    } else {
        const any16 a = *(const any16 *) p;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t h = (uint16_t) (a.v[i >> 1] >> (16 * (i & 1)));
            v[i] = std::is_same<T, _Float16>::value ? (float) __builtin_bit_cast(_Float16, h) : bf16_to_f32(h);
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T * p, const float * v) {
    any16 a;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a.v[i] = __float_as_uint(v[i]);
        *(any16 *) p = a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a.v[i] = __float_as_uint(v[4 + i]);
        *(any16 *) (p + 4) = a;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if constexpr (std::is_same<T, _Float16>::value)
                a.v[i] = (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) v[2 * i]) |
                         (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) v[2 * i + 1]) << 16;
            else
                a.v[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        *(any16 *) p = a;
    }
}

// ---------------------------------------------------------------------------
// Quantisation.  With top = max |x| of a block, e = floor(log2 top) - 2 (the
// exponent field of top, clamped to the scale's range) puts the largest value
// into [4, 8), and every value becomes the nearest code of x 2^-e, halves to
// the even code, 6 the largest.  A block of zeros has e = -127; one with an
// Inf or NaN is NaN (scale byte 255, codes 0).
//
// Memory bound (read s bytes, write 17/32 per value): four lanes take one
// block, eight values each, and the 17-byte blocks of a workgroup meet in LDS
// and leave as 16-byte rows of memory; a 256-thread workgroup makes kQBlocks
// blocks, 17 x 256 bytes, so its part of an aligned result is aligned too.
// ---------------------------------------------------------------------------
constexpr int kQBlocks = 256, kQThreads = 256;

template <typename T>
__global__ __launch_bounds__(kQThreads) void mx_quantize(const T * __restrict__ x, int64_t ldx, uint8_t * __restrict__ q,
                                                         int64_t blocks, int64_t row_blocks) {
    __shared__ __align__(16) uint8_t out[kQBlocks * kMxBytes];
    const int64_t b0 = (int64_t) blockIdx.x * kQBlocks;
    const int lane4 = threadIdx.x & 3;
    constexpr int kPass = kQThreads / 4;
    float v[kQBlocks / kPass][8];
#pragma unroll
    for (int i = 0; i < kQBlocks / kPass; ++i) {
        const int64_t b = min(b0 + i * kPass + (threadIdx.x >> 2), blocks - 1);
        const int64_t row = ldx == row_blocks * 32 ? 0 : b / row_blocks;
        load8(x + row * ldx + (b - row * row_blocks) * 32 + lane4 * 8, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kQBlocks / kPass; ++i) {
        // |x| as bits: their order is the values' order, Inf and NaN on top.
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
        top = max(top, (uint32_t) __shfl_xor((int) top, 1));
        top = max(top, (uint32_t) __shfl_xor((int) top, 2));
        const uint32_t field = top >> 23;
        const bool nan = field == 255;
        const uint32_t e = nan ? 255 : field > 2 ? field - 2 : 0;
        uint32_t code = 0;  // eight codes, value j in bits 4j
        const float s = mx_scale(e);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[i][0], v[i][1], s, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[i][2], v[i][3], s, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[i][4], v[i][5], s, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[i][6], v[i][7], s, 3);
        if (nan) code = 0;
        // Lanes 0, 1 hold values 0..15, lanes 2, 3 values 16..31: lane l < 2
        // joins its codes with lane l + 2's, byte by byte.
        const uint32_t other = (uint32_t) __shfl_xor((int) code, 2);
        uint8_t * blk = out + (i * kPass + (threadIdx.x >> 2)) * kMxBytes;
        if (lane4 == 0) blk[0] = (uint8_t) e;
        if (lane4 < 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                blk[1 + lane4 * 8 + j] = (uint8_t) (((code >> (4 * j)) & 15) | ((other >> (4 * j)) & 15) << 4);
        }
    }
    __syncthreads();
    const int64_t n = min((int64_t) kQBlocks, blocks - b0) * kMxBytes;
    uint8_t * dst = q + b0 * kMxBytes;
    for (int i = threadIdx.x * 16; i < n; i += kQThreads * 16) {
        if (i + 16 <= n) {
            *(any16 *) (dst + i) = *(const any16 *) (out + i);
        } else {
            for (int j = i; j < n; ++j) dst[j] = out[j];
        }
    }
}

// Values of packed blocks: the reverse path, four lanes to a block, eight codes
// read and eight values written by each.  ldy is the row stride of y in
// elements; qs the byte stride of packed rows (row_blocks * 17 when they follow
// each other); rows (nullable) picks row rows[r] of `qrows` packed rows
// (negative or past the end: NaN).  Bound by its writes: 14336 x 4096 values to
// f32 71 us (bf16 34), quantised from it 50 (bf16 26); one after the other 116,
// 4.3 TB/s (bf16 58).
template <typename T>
__global__ __launch_bounds__(kQThreads) void mx_dequantize(const uint8_t * __restrict__ q, int64_t qs,
                                                           const int32_t * __restrict__ rows, int64_t qrows,
                                                           T * __restrict__ y, int64_t ldy, int64_t blocks,
                                                           int64_t row_blocks) {
    const int64_t b0 = (int64_t) blockIdx.x * kQBlocks;
    const int lane4 = threadIdx.x & 3;
    constexpr int kPass = kQThreads / 4;
    any8 code[kQBlocks / kPass];
    uint8_t e[kQBlocks / kPass];
    int64_t yo[kQBlocks / kPass];
#pragma unroll
    for (int i = 0; i < kQBlocks / kPass; ++i) {
        const int64_t b = min(b0 + i * kPass + (threadIdx.x >> 2), blocks - 1);
        const int64_t row = b / row_blocks, kb = b - row * row_blocks;
        int64_t from = row;
        bool ok = true;
        if (rows) {
            from = rows[row];
            ok = from >= 0 && from < qrows;
        }
        const uint8_t * blk = q + (ok ? from : 0) * qs + kb * kMxBytes;
        e[i] = ok ? blk[0] : 255;
        code[i] = *(const any8 *) (blk + 1 + 8 * (lane4 & 1));
        yo[i] = row * ldy + kb * 32 + lane4 * 8;
    }
#pragma unroll
    for (int i = 0; i < kQBlocks / kPass; ++i) {
        if (b0 + i * kPass + (threadIdx.x >> 2) >= blocks) break;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // Sign, then the code's three magnitude bits as the top of an f32
            // times 2^126: exact, the half through a subnormal.
            const uint32_t c = code[i].v[j >> 2] >> (8 * (j & 3) + 4 * (lane4 >> 1));
            v[j] = __uint_as_float((c & 8) << 28 | (c & 7) << 22) * 0x1p126f;
            v[j] = e[i] == 255 ? __uint_as_float(0x7fc00000u)
                               : v[j] * (e[i] ? mx_scale(e[i]) : __uint_as_float(0x00400000u));
        }
        store8(y + yo[i], v);
    }
}

// ---------------------------------------------------------------------------
// Products.
// ---------------------------------------------------------------------------
struct MxParams {
    const uint8_t * w;
    int64_t ws;  // bytes of a weight row
    const void * x;
    int64_t ldx;
    void * y;
    int64_t ldy;
    const uint16_t * bias;
    const uint16_t * res;
    int64_t ldres;
    const float * gate;
    int64_t M, N;
    int kb;  // blocks of a row
    int32_t y_f32, epi;
    int64_t plane;  // bytes from one K split's f32 plane to the next's (y is the first), or 0
    int steps;      // K steps of 128 of one split
};

// Four outputs y[n][m .. m + 3] with the rounding points of the LINEAR
// epilogues: the product to bf16, the bias sum to bf16, then the rest.
__device__ __forceinline__ void mx_store4(const MxParams & p, int64_t n, int64_t m, const float * acc) {
    if (p.y_f32) {
        float * y = (float *) p.y + n * p.ldy + m;
        if (m + 4 <= p.M) {
            any16 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o.v[r] = __float_as_uint(acc[r]);
            *(any16 *) y = o;
            return;
        }
        for (int r = 0; r < 4; ++r)
            if (m + r < p.M) y[r] = acc[r];
        return;
    }
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        v[r] = acc[r];
        if (p.epi == WAMX_EPI_NONE || m + r >= p.M) continue;
        v[r] = round_bf16(v[r]) + bf16_to_f32(p.bias[m + r]);
        if (p.epi == WAMX_EPI_BIAS_GELU) v[r] = gelu_tanh(v[r]);
        if (p.epi == WAMX_EPI_BIAS_GATED)
            v[r] = fmaf(round_bf16(v[r]), p.gate[m + r], bf16_to_f32(p.res[n * p.ldres + m + r]));
        if (p.epi == WAMX_EPI_BIAS_RESIDUAL) v[r] = bf16_to_f32(p.res[n * p.ldres + m + r]) + round_bf16(v[r]);
    }
    uint16_t * y = (uint16_t *) p.y + n * p.ldy + m;
    if (m + 4 <= p.M) {
        any8 o;
        o.v[0] = pack_bf16x2(v[0], v[1]);
        o.v[1] = pack_bf16x2(v[2], v[3]);
        *(any8 *) y = o;
        return;
    }
    for (int r = 0; r < 4; ++r)
        if (m + r < p.M) y[r] = f32_to_bf16(v[r]);
}

// Eight weights for one MFMA: the four bytes of a dword give values (j, j + 16)
// of their block in pairs.
__device__ __forceinline__ bf16x8_t mx_frag(uint32_t d, float scale) {
    union {
        bf16x2_t p[4];
        bf16x8_t v;
    } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 0);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 1);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 2);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, scale, 3);
    return u.v;
}

// The codes of a block with value j in nibble j: dword g holds 8g .. 8g + 7.
__device__ __forceinline__ uint4 mx_natural(const any16 & b) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // Four nibbles to bytes 0 and 2.
        const uint32_t l = b.v[i] & 0x0f0f0f0fu, h = (b.v[i] >> 4) & 0x0f0f0f0fu;
        lo[i] = l | l >> 4;
        hi[i] = h | h >> 4;
    }
    return make_uint4(__builtin_amdgcn_perm(lo[1], lo[0], 0x06040200u), __builtin_amdgcn_perm(lo[3], lo[2], 0x06040200u),
                      __builtin_amdgcn_perm(hi[1], hi[0], 0x06040200u), __builtin_amdgcn_perm(hi[3], hi[2], 0x06040200u));
}

// The activations of mx_frag(dword i): values 4i .. 4i + 3 (lo) and 16 + 4i ..
// (hi) of the block, paired in the same order.
__device__ __forceinline__ bf16x8_t mx_pair(uint32_t lo0, uint32_t lo1, uint32_t hi0, uint32_t hi1) {
    union {
        uint32_t d[4];
        bf16x8_t v;
    } u;
    u.d[0] = __builtin_amdgcn_perm(hi0, lo0, 0x05040100u);
    u.d[1] = __builtin_amdgcn_perm(hi0, lo0, 0x07060302u);
    u.d[2] = __builtin_amdgcn_perm(hi1, lo1, 0x05040100u);
    u.d[3] = __builtin_amdgcn_perm(hi1, lo1, 0x07060302u);
    return u.v;
}

// Few tokens: every byte of the weight is read once, in 16-byte pieces, and goes
// straight into matrix operands.  What it takes beyond those bytes' time is not
// the expansion of the codes (with the bits as they are instead, which computes
// something else, every size takes as long) but x, which each workgroup reads and
// passes through LDS (without: 14336 x 48 x 4096 13.4 us for 18.1, 20000 x 1 x
// 4096 14.8 for 17.4, where all 16 token rows are copies of the one), and the
// latency of the few K steps that a wave has.  A workgroup takes
// RG groups of 16 weight rows and NT tiles of 16 tokens; its waves take the K
// steps of 128 in turn (a row's 68 bytes of a step lie next to the next
// wave's) and their sums meet in LDS in wave order.  Lane (r, g) holds block g
// of the step for weight row r, and the same 32 values of x for token r.
constexpr int kMxWaves = 8, kMxAhead = 2;

template <int RG, int NT, bool XF32>
__global__ __launch_bounds__(kMxWaves * 64) void mx_few(MxParams p) {
    // A wave's x of one step, [token][16-byte piece]; after the last step the
    // waves' sums.
    constexpr int XB = NT * 16 * 256, RB = RG * NT * 64 * 16;
    __shared__ __align__(16) uint8_t lds[kMxWaves * (XB > RB ? XB : RB)];
    f32x4_t (*red)[RG * NT][64] = (f32x4_t (*)[RG * NT][64]) lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int64_t m0 = (int64_t) blockIdx.x * (16 * RG), n0 = (int64_t) blockIdx.y * (16 * NT);
    const int s0 = (int) blockIdx.z * p.steps, s1 = min(s0 + p.steps, (p.kb + 3) / 4);
    p.y = (char *) p.y + blockIdx.z * p.plane;

    const char * w[RG];
    uint32_t mis[RG];
    uint32_t x[NT * 4];
    constexpr int xs = XF32 ? 4 : 2;
    const char * xbase = (const char *) p.x + n0 * p.ldx * xs;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
        // Rows of fewer than four blocks: their last one for the lanes past it.
        w[i] = (const char *) p.w + min(m0 + i * 16 + r, p.M - 1) * p.ws + min(g, p.kb - 1) * (int) kMxBytes;
        mis[i] = (uint32_t) (uintptr_t) w[i] & 3;
        w[i] -= mis[i];
    }
    // Sixteen lanes read the 256 bytes of a token's step (twice that in f32), a
    // lane four tokens, at 32-bit offsets (launch_mx_product sees to that).
#pragma unroll
    for (int j = 0; j < NT * 4; ++j)
        x[j] = (uint32_t) ((min(n0 + j * 4 + g, p.N - 1) - n0) * p.ldx + r * 8) * xs;
    uint4 * mine = (uint4 *) (lds + wave * XB);

    // x of the next step is requested when this one's lies in LDS, the weights
    // kMxAhead steps before their use (one: 14336 x 48 x 4096 19.0 us for 18.1,
    // 14336 x 32 x 4096 16.2 for 15.8, but 20000 x 1 x 4096 17.0 for 17.7; three:
    // spills).
    MxBlock wr[kMxAhead + 1][RG];
    any16 xr[NT * 4][XF32 ? 2 : 1];
    auto load_w = [&](int s, MxBlock * t) {
        // A lane past the row's last block repeats its block of the step before.
        const int64_t o = (int64_t) (s - (s > 0 && 4 * s + g >= p.kb)) * (4 * kMxBytes);
#pragma unroll
        for (int i = 0; i < RG; ++i) t[i] = mx_load(w[i] + o);
    };
    auto load_x = [&](int s) {
        const uint32_t xo = (uint32_t) (4 * s + (r >> 2) < p.kb ? s * 128 : -r * 8) * (uint32_t) xs;  // past the row: its start
#pragma unroll
        for (int j = 0; j < NT * 4; ++j)
#pragma unroll
            for (int v = 0; v < (XF32 ? 2 : 1); ++v) xr[j][v] = *(const any16 *) (xbase + (x[j] + xo) + 16 * v);
    };
    f32x4_t acc[RG][NT];
#pragma unroll
    for (int i = 0; i < RG; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};
    auto multiply = [&](int s, int next, int next_w, MxBlock * t, MxBlock * tn) {
        // Through LDS into operand order: piece q of token n in slot q ^ (n % 16),
        // so that the 16 tokens of a read lie in different banks.
        const bool tail = 4 * s + 4 > p.kb;
#pragma unroll
        for (int j = 0; j < NT * 4; ++j) {
            uint4 v;
            if constexpr (XF32) {
                const any16 &a = xr[j][0], &b = xr[j][1];
                v = make_uint4(pack_bf16x2(__uint_as_float(a.v[0]), __uint_as_float(a.v[1])),
                               pack_bf16x2(__uint_as_float(a.v[2]), __uint_as_float(a.v[3])),
                               pack_bf16x2(__uint_as_float(b.v[0]), __uint_as_float(b.v[1])),
                               pack_bf16x2(__uint_as_float(b.v[2]), __uint_as_float(b.v[3])));
            } else {
                v = make_uint4(xr[j][0].v[0], xr[j][0].v[1], xr[j][0].v[2], xr[j][0].v[3]);
            }
            const int n = j * 4 + g;
            mine[n * 16 + (r ^ (n & 15))] = v;
        }
        if (tail && 4 * s + (r >> 2) >= p.kb) {  // past the row's last block: nothing times nothing
#pragma unroll
            for (int j = 0; j < NT * 4; ++j) mine[(j * 4 + g) * 16 + (r ^ ((j * 4 + g) & 15))] = make_uint4(0, 0, 0, 0);
        }
        if (tail && 4 * s + g >= p.kb) {
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                t[i].hi = 0;
#pragma unroll
                for (int d = 0; d < 4; ++d) t[i].lo.v[d] = 0;
            }
        }
        if (next >= 0) load_x(next);
        if (next_w >= 0) load_w(next_w, tn);
        __builtin_amdgcn_wave_barrier();
        // Dwords 2h and 2h + 1 of the codes meet pieces h and h + 2 of block g.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 lo[NT], hi[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                lo[j] = mine[(j * 16 + r) * 16 + ((4 * g + h) ^ r)];
                hi[j] = mine[(j * 16 + r) * 16 + ((4 * g + h + 2) ^ r)];
            }
#pragma unroll
            for (int d = 2 * h; d < 2 * h + 2; ++d) {
                bf16x8_t b[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    b[j] = d & 1 ? mx_pair(lo[j].z, lo[j].w, hi[j].z, hi[j].w) : mx_pair(lo[j].x, lo[j].y, hi[j].x, hi[j].y);
#pragma unroll
                for (int i = 0; i < RG; ++i) {
                    const bf16x8_t a = mx_frag(mx_codes(t[i], d, mx_select(mis[i])), mx_scale(mx_exponent(t[i], mis[i])));
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[j], acc[i][j], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    };
    // Workgroups begin at different steps: rows of x lie a power of two apart as
    // often as not, where one step of all rows is one channel of the L2.
    const int ns = s1 - s0, turn = (int) (blockIdx.x % (uint32_t) ns);
    auto at = [&](int k) { return s0 + (k + turn < ns ? k + turn : k + turn - ns); };
    int k = wave;
    if (k < ns) load_x(at(k));
#pragma unroll
    for (int d = 0; d < kMxAhead; ++d)
        if (k + d * kMxWaves < ns) load_w(at(k + d * kMxWaves), wr[d]);
    while (k < ns) {
#pragma unroll
        for (int q = 0; q <= kMxAhead; ++q) {
            if (k >= ns) break;
            multiply(at(k), k + kMxWaves < ns ? at(k + kMxWaves) : -1,
                     k + kMxAhead * kMxWaves < ns ? at(k + kMxAhead * kMxWaves) : -1, wr[q],
                     wr[(q + kMxAhead) % (kMxAhead + 1)]);
            k += kMxWaves;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RG; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int t = threadIdx.x; t < RG * NT * 64; t += kMxWaves * 64) {
        const int tile = t >> 6, l = t & 63;
        f32x4_t v = red[0][tile][l];
#pragma unroll
        for (int u = 1; u < kMxWaves; ++u) v += red[u][tile][l];
        const int64_t n = n0 + (tile % NT) * 16 + (l & 15), m = m0 + (tile / NT) * 16 + (l >> 4) * 4;
        if (n >= p.N || m >= p.M) continue;
        const float o[4] = {v[0], v[1], v[2], v[3]};
        mx_store4(p, n, m, o);
    }
}

// Many tokens: WM waves along the weight rows by WN along the tokens, each RG x
// NT tiles of 16 x 16.  Every wave expands its rows' codes itself, so 128 x 128
// tiles take 4 x 2 waves of 2 x 4 tiles (10250 x 333 x 2048: 24.6 us, 2 x 4
// waves of 4 x 2 tiles 28.6).  The weight stays in its 4 bits down to the
// register that becomes the operand: a step of 128 values is 4 blocks a row,
// whose codes are put into the order of their values on the way to LDS and lie
// there as [block][row][g], so that a wave's read of dword g of its rows is 256
// bytes in a row and expands to values 8g .. 8g + 7 of its block.  x lies in LDS
// as it is, half a step at a time.  (With x interleaved in the codes' own order
// instead, and the blocks read at odd addresses for want of registers: 4096 x
// 1100 x 4096 67.7 us for 63.5, 14336 x 2048 x 4096 215 for 210, 10250 x 333 x
// 2048 28.9 for 27.7.)  Both go through registers, requested a step before their
// use, into one of two LDS buffers while the other is multiplied: one barrier
// per half step, the writes behind the first row tile's products.  x straight
// into LDS, three buffers, took as long or longer: 221 us for 2048 tokens.
template <int RG, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void mx_tile(MxParams p) {
    constexpr int TH = 64 * WM * WN, BM = RG * 16 * WM, BN = NT * 16 * WN;
    constexpr int XP = BN * 8 / TH;             // 16-byte x pieces of a thread per half step
    constexpr int WB = (BM * 4 + TH - 1) / TH;  // weight blocks of a thread per step
    // The four blocks of a row, written by four neighbouring lanes, lie a
    // quarter of the banks apart.
    constexpr int WS = (BM + 15) / 16 * 16 + 4, SS = (BM + 63) / 64 * 64 + 16;
    __shared__ __align__(16) uint32_t wl[2][WS * 16];
    __shared__ __align__(16) float sl[2][SS * 4];
    __shared__ __align__(16) uint32_t xl[2][BN * 32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4, wm = wave / WN, wn = wave % WN;
    const int64_t m0 = (int64_t) blockIdx.x * BM, n0 = (int64_t) blockIdx.y * BN;
    const int s0 = (int) blockIdx.z * p.steps, s1 = min(s0 + p.steps, (p.kb + 3) / 4);
    p.y = (char *) p.y + blockIdx.z * p.plane;
    // Sources: one address for the workgroup, 32-bit offsets for the lanes (a
    // tile's rows lie within 4 GB, see launch_mx_product).
    const char * wbase = (const char *) p.w + m0 * p.ws;
    const char * xbase = (const char *) p.x + n0 * p.ldx * 2;

    // Weight blocks: thread t takes block t % 4 of rows t / 4, t / 4 + TH / 4, ...
    const int wkb = threadIdx.x & 3, wrow = threadIdx.x >> 2;
    uint32_t woff[WB];
    const uint32_t wlow = (uint32_t) (uintptr_t) wbase;
#pragma unroll
    for (int j = 0; j < WB; ++j)
        woff[j] = (uint32_t) min((int64_t) (wrow + j * (TH / 4)), p.M - 1 - m0) * (uint32_t) p.ws;
    MxBlock wr[WB];
    uint32_t wmis[WB];
    auto request_w = [&](int s, MxBlock * r, uint32_t * e) {
        const uint32_t at = (uint32_t) min(4 * s + wkb, p.kb - 1) * (uint32_t) kMxBytes;
#pragma unroll
        for (int j = 0; j < WB; ++j) {
            const uint32_t o = woff[j] + at;
            e[j] = (wlow + o) & 3;
            r[j] = mx_load(wbase + (int64_t) o - e[j]);
        }
    };
    auto deposit_w = [&](int s, int buf, const MxBlock * r, const uint32_t * e) {
#pragma unroll
        for (int j = 0; j < WB; ++j) {
            const int row = wrow + j * (TH / 4);
            if (BM % (TH / 4) != 0 && row >= BM) break;
            any16 c;
#pragma unroll
            for (int i = 0; i < 4; ++i) c.v[i] = mx_codes(r[j], i, mx_select(e[j]));
            ((uint4 *) wl[buf])[wkb * WS + row] = mx_natural(c);
            sl[buf][wkb * SS + row] = mx_scale(mx_exponent(r[j], e[j]));
        }
        if (4 * s + 4 > p.kb && 4 * s + wkb >= p.kb) {  // past a row's last block: zeros
#pragma unroll
            for (int j = 0; j < WB; ++j) {
                const int row = wrow + j * (TH / 4);
                if (BM % (TH / 4) != 0 && row >= BM) break;
                ((uint4 *) wl[buf])[wkb * WS + row] = make_uint4(0, 0, 0, 0);
                sl[buf][wkb * SS + row] = 1.0f;
            }
        }
    };
    // Activations: eight lanes read the 128 bytes of a row's half step.
    const int xc = threadIdx.x & 7;
    any16 xr[2][XP];
    uint32_t xoff[XP];
    int xpos[XP];
#pragma unroll
    for (int q = 0; q < XP; ++q) {
        const int row = (threadIdx.x >> 3) + q * (TH / 8);
        xoff[q] = ((uint32_t) min((int64_t) row, p.N - 1 - n0) * (uint32_t) p.ldx + (uint32_t) (xc & 3) * 8) * 2;
        xpos[q] = row * 8 + (xc ^ ((row >> 1) & 7));
    }
    auto request_x = [&](int h, any16 * r) {  // half step h: blocks 2h, 2h + 1
        const uint32_t at = (uint32_t) min(2 * h + (xc >> 2), p.kb - 1) * 64u;
#pragma unroll
        for (int q = 0; q < XP; ++q) r[q] = *(const any16 *) (xbase + (xoff[q] + at));
    };
    auto deposit_x = [&](int h, int buf, const any16 * r) {
        uint4 * dst = (uint4 *) xl[buf];
#pragma unroll
        for (int q = 0; q < XP; ++q) dst[xpos[q]] = make_uint4(r[q].v[0], r[q].v[1], r[q].v[2], r[q].v[3]);
        if (2 * h + 2 > p.kb && 2 * h + (xc >> 2) >= p.kb) {
#pragma unroll
            for (int q = 0; q < XP; ++q) dst[xpos[q]] = make_uint4(0, 0, 0, 0);
        }
    };

    f32x4_t acc[RG][NT];
#pragma unroll
    for (int i = 0; i < RG; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};
    auto multiply = [&](int wbuf, int half, auto && middle) {
        bf16x8_t b[2][NT];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int row = (wn * NT + j) * 16 + c16;
                b[i][j] = ((const bf16x8_t *) xl[half])[row * 8 + ((i * 4 + g) ^ ((row >> 1) & 7))];
            }
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            if (r == 1) middle();
            const int row = (wm * RG + r) * 16 + c16, k = half * 2;
            const bf16x8_t a0 = mx_frag(wl[wbuf][(k * WS + row) * 4 + g], sl[wbuf][k * SS + row]);
            const bf16x8_t a1 = mx_frag(wl[wbuf][((k + 1) * WS + row) * 4 + g], sl[wbuf][(k + 1) * SS + row]);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b[0][j], acc[r][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b[1][j], acc[r][j], 0, 0, 0);
        }
    };
    // Requests past the last step repeat its addresses (requested, not used).
    const int last = s1 - 1;
    if (s0 < s1) {
        request_w(s0, wr, wmis);
        request_x(2 * s0, xr[0]);
        request_x(2 * s0 + 1, xr[1]);
        deposit_w(s0, 0, wr, wmis);
        deposit_x(2 * s0, 0, xr[0]);
        request_w(min(s0 + 1, last), wr, wmis);
        request_x(2 * min(s0 + 1, last), xr[0]);
    }
    lds_barrier();
    for (int s = s0; s < s1; ++s) {
        const int wb = (s - s0) & 1;
        multiply(wb, 0, [&]() {
            deposit_x(2 * s + 1, 1, xr[1]);
            request_x(2 * min(s + 1, last) + 1, xr[1]);
        });
        lds_barrier();
        multiply(wb, 1, [&]() {
            deposit_x(2 * s + 2, 0, xr[0]);
            deposit_w(s + 1, wb ^ 1, wr, wmis);
            request_x(2 * min(s + 2, last), xr[0]);
            request_w(min(s + 2, last), wr, wmis);
        });
        lds_barrier();
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = n0 + (wn * NT + j) * 16 + c16;
        if (n >= p.N) continue;
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            const int64_t m = m0 + (wm * RG + r) * 16 + 4 * g;
            if (m >= p.M) continue;
            const float o[4] = {acc[r][j][0], acc[r][j][1], acc[r][j][2], acc[r][j][3]};
            mx_store4(p, n, m, o);
        }
    }
}

// f32 rows rounded to bf16, one after another.
__global__ __launch_bounds__(256) void mx_round_rows(const float * __restrict__ x, int64_t ldx, uint16_t * __restrict__ y,
                                                     int64_t rows, int row_pieces) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * row_pieces) return;
    const int64_t r = i / row_pieces;
    float v[8];
    load8(x + r * ldx + (i - r * row_pieces) * 8, v);
    store8(y + i * 8, v);
}

// The K splits' planes, added in order, with the product's epilogue.
__global__ __launch_bounds__(256) void mx_reduce(MxParams p, const float * __restrict__ part, int splits) {
    const int64_t quads = (p.M + 3) / 4, i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= p.N * quads) return;
    const int64_t n = i / quads, m = (i - n * quads) * 4;
    float v[4] = {0, 0, 0, 0};
    for (int s = 0; s < splits; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (m + r < p.M) v[r] += part[(s * p.N + n) * p.M + m + r];
    mx_store4(p, n, m, v);
}

template <int RG, int NT>
static void launch_few(const MxParams & p, bool xf32, int splits, hipStream_t s) {
    const dim3 grid((unsigned) ((p.M + 16 * RG - 1) / (16 * RG)), (unsigned) ((p.N + 16 * NT - 1) / (16 * NT)),
                    (unsigned) splits);
    // f32 rows of two token tiles at most are rounded on the way.
    if constexpr (NT <= 2)
        if (xf32) {
            hipLaunchKernelGGL((mx_few<RG, NT, true>), grid, dim3(kMxWaves * 64), 0, s, p);
            return;
        }
    hipLaunchKernelGGL((mx_few<RG, NT, false>), grid, dim3(kMxWaves * 64), 0, s, p);
}
template <int NT>
static void launch_few_rows(const MxParams & p, bool xf32, int rg, int splits, hipStream_t s) {
    if (rg == 1) launch_few<1, NT>(p, xf32, splits, s);
    else if (rg == 2) launch_few<2, NT>(p, xf32, splits, s);
    else launch_few<4, NT>(p, xf32, splits, s);
}

template <int RG, int NT, int WM, int WN>
static void launch_tile(const MxParams & p, int splits, hipStream_t s) {
    constexpr int BM = RG * 16 * WM, BN = NT * 16 * WN;
    const dim3 grid((unsigned) ((p.M + BM - 1) / BM), (unsigned) ((p.N + BN - 1) / BN), (unsigned) splits);
    hipLaunchKernelGGL((mx_tile<RG, NT, WM, WN>), grid, dim3(64 * WM * WN), 0, s, p);
}

// A plan for the tiles: the variant and K splits of the least modelled time
// (us, 256 CUs).  A step of 128 values of c workgroups on a CU takes `base` +
// c * `more` (measured: 224 x 256 tiles 3.4 each, 128 x 256 2.2 each, 128 x 128
// 1.4 alone and 2.4 in pairs, 64 x 64 0.69, 1.03 and with five 2.5); the planes
// of the splits are written and read at 4 TB/s, and they cost one more launch.
// Modelled and measured: 14336 x 128 x 4096 in 128 x 128 tiles and 2 splits 35
// and 33, in 64 x 64 unsplit 38 and 38; 4096 x 128 x 4096 in 64 x 64 and 4
// splits 19 and 20; 4096 x 70 x 14336 in 128 x 128 and 8 splits 29 and 29, in
// 64 x 64 and 4 splits 41 and 37.
struct TilePlan {
    int kind, splits;
};
static TilePlan tile_plan(int64_t M, int64_t N, int steps, size_t ws_bytes) {
    static const struct {
        int bm, bn;
        double base, more;
    } kinds[] = {{224, 256, 0, 3.4}, {128, 256, 0, 2.2}, {128, 128, 0.3, 1.1}, {64, 64, 0.35, 0.42}};
    TilePlan best{2, 1};
    double least = 0;
    for (int k = 0; k < 4; ++k)
        for (int splits = 1; splits <= 8; splits *= 2) {
            const double planes = (double) splits * (double) N * (double) M * 4;
            if (splits > 1 && (steps / splits < 4 || planes > (double) ws_bytes)) break;
            const int64_t tiles = ((M + kinds[k].bm - 1) / kinds[k].bm) * ((N + kinds[k].bn - 1) / kinds[k].bn);
            const double c = (double) ((tiles * splits + 255) / 256);
            const double t = (steps + splits - 1) / splits * (kinds[k].base + c * kinds[k].more) +
                             (splits > 1 ? 5 + 2 * planes / 4e6 : 0);
            if (least == 0 || t < least) {
                least = t;
                best = {k, splits};
            }
        }
    return best;
}

// One product with bf16 activations, or f32 ones for at most 32 tokens.
static void run_product(MxParams p, bool xf32, void * ws, size_t ws_bytes, hipStream_t s) {
    const int steps = (p.kb + 3) / 4;
    const int64_t groups = (p.M + 15) / 16;
    // Few tokens: groups of 16 rows to a workgroup by how many workgroups a CU
    // then has to run and what each costs, two for a group's weights and one for
    // a tile's x (us with 1, 2 and 4 groups: 4096 x 1 x 4096 6.2, 7.8, 12.0;
    // 20000 x 1 x 4096 21.2, 17.7, 22.5; 14336 x 32 x 4096 24.2, 20.0, 15.8;
    // 14336 x 48 x 4096 35.7, 24.0, 18.1).  49 to 64 tokens come here while 512
    // groups, a workgroup per CU, hold the rows (6400 x 64 x 4096 14.6 us, in
    // tiles 20.4).
    const bool near = std::max(p.ws, p.ldx * 2) < (1ll << 23);  // a tile's 256 rows within 32-bit offsets
    const bool few = p.N <= 48 || (p.N <= 64 && groups <= 512) || !near;
    // Four token tiles leave registers for two groups.
    const int most = p.N > 48 ? 2 : 4;
    int rg = 1, splits = 1;
    int64_t least = 0;
    for (int c = 1; c <= most; c *= 2) {
        const int64_t t = (groups + 256 * c - 1) / (256 * c) * (2 * c + (std::min<int64_t>(p.N, 64) + 15) / 16);
        if (least && t > least) continue;
        least = t;
        rg = c;
    }
    TilePlan plan{};
    if (!few) {
        plan = tile_plan(p.M, p.N, steps, ws_bytes);
        splits = plan.splits;
    } else if (p.N > 32 && steps >= 96 && groups <= 256 && 16 * (size_t) p.N * (size_t) p.M <= ws_bytes) {
        // Long rows, few of them: four K splits of 256 workgroups in all
        // (2048 x 64 x 14336: 17.5 us, unsplit in as many row groups 39; 4096 x 48
        // x 14336: 20.7, 47).
        splits = 4;
        rg = std::min(most, groups > 128 ? 4 : groups > 64 ? 2 : 1);
    }
    p.steps = (steps + splits - 1) / splits;
    splits = (steps + p.steps - 1) / p.steps;
    const MxParams whole = p;
    if (splits > 1) {
        p.y = ws;
        p.y_f32 = 1;
        p.ldy = p.M;
        p.epi = WAMX_EPI_NONE;
        p.plane = p.N * p.M * 4;
    }
    if (few) {
        if (p.N <= 16) launch_few_rows<1>(p, xf32, rg, splits, s);
        else if (p.N <= 32) launch_few_rows<2>(p, xf32, rg, splits, s);
        else if (p.N <= 48) launch_few_rows<3>(p, xf32, rg, splits, s);
        else if (rg == 1) launch_few<1, 4>(p, xf32, splits, s);
        else launch_few<2, 4>(p, xf32, splits, s);
    } else if (plan.kind == 0) {
        launch_tile<7, 4, 2, 4>(p, splits, s);
    } else if (plan.kind == 1) {
        launch_tile<4, 4, 2, 4>(p, splits, s);
    } else if (plan.kind == 2) {
        launch_tile<2, 4, 4, 2>(p, splits, s);
    } else {
        launch_tile<2, 2, 2, 2>(p, splits, s);
    }
    if (splits > 1)
        hipLaunchKernelGGL(mx_reduce, dim3((unsigned) ((p.N * ((p.M + 3) / 4) + 255) / 256)), dim3(256), 0, s, whole,
                           (const float *) ws, splits);
}

hipError_t launch_mx_quantize(const void * x, int32_t x_type, int64_t ldx, void * q, int64_t rows, int64_t cols,
                              hipStream_t s) {
    const int64_t rb = cols / 32, blocks = rows * rb;
    if (blocks <= 0) return hipSuccess;
    const int64_t wgs = (blocks + kQBlocks - 1) / kQBlocks;
    if (wgs > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned) wgs), wg(kQThreads);
    uint8_t * o = (uint8_t *) q;
    switch (x_type) {
        case WAMX_TYPE_F32: hipLaunchKernelGGL(mx_quantize<float>, grid, wg, 0, s, (const float *) x, ldx, o, blocks, rb); break;
        case WAMX_TYPE_F16: hipLaunchKernelGGL(mx_quantize<_Float16>, grid, wg, 0, s, (const _Float16 *) x, ldx, o, blocks, rb); break;
        case WAMX_TYPE_BF16: hipLaunchKernelGGL(mx_quantize<uint16_t>, grid, wg, 0, s, (const uint16_t *) x, ldx, o, blocks, rb); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const void * q, int64_t qs, const int32_t * rows, int64_t qrows, void * y,
                                int32_t y_type, int64_t ldy, int64_t nrows, int64_t cols, hipStream_t s) {
    const int64_t rb = cols / 32, blocks = nrows * rb;
    if (blocks <= 0) return hipSuccess;
    const int64_t wgs = (blocks + kQBlocks - 1) / kQBlocks;
    if (wgs > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned) wgs), wg(kQThreads);
    const uint8_t * i = (const uint8_t *) q;
    switch (y_type) {
        case WAMX_TYPE_F32: hipLaunchKernelGGL(mx_dequantize<float>, grid, wg, 0, s, i, qs, rows, qrows, (float *) y, ldy, blocks, rb); break;
        case WAMX_TYPE_F16: hipLaunchKernelGGL(mx_dequantize<_Float16>, grid, wg, 0, s, i, qs, rows, qrows, (_Float16 *) y, ldy, blocks, rb); break;
        case WAMX_TYPE_BF16: hipLaunchKernelGGL(mx_dequantize<uint16_t>, grid, wg, 0, s, i, qs, rows, qrows, (uint16_t *) y, ldy, blocks, rb); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_mx_product(const MxArgs & a, hipStream_t s) {
    if (a.M <= 0 || a.N <= 0) return hipSuccess;
    if (a.K <= 0 || a.K % 32 != 0 || a.K >= 1 << 30) return hipErrorInvalidValue;
    MxParams p{};
    p.w = (const uint8_t *) a.w;
    p.ws = a.w_stride;
    p.x = a.x;
    p.ldx = a.ldx;
    p.y = a.y;
    p.ldy = a.ldy;
    p.bias = (const uint16_t *) a.bias;
    p.res = (const uint16_t *) a.res;
    p.ldres = a.ldres;
    p.gate = a.gate;
    p.M = a.M;
    p.N = a.N;
    p.kb = (int) (a.K / 32);
    p.y_f32 = a.y_type == WAMX_TYPE_F32;
    p.epi = a.epi;
    p.steps = (p.kb + 3) / 4;
    const bool xf32 = a.x_type == WAMX_TYPE_F32;
    // Tokens in parts that a grid takes.  Rows so long or so far apart that 64 of
    // them pass 32-bit offsets go one by one.
    int64_t part = std::max(a.ldx, a.K) > 1 << 23 ? 1 : 1 << 20;
    // f32 activations of more than 32: rounded once into half of the workspace, as
    // many rows at a time as it holds (two at least); single rows on their way.
    const size_t row = (size_t) a.K * 2, half = a.ws_bytes / 2;
    static_assert(kBackendWorkspaceBytes / 2 >= (2u << 23), "a row of 2^23 values fits");
    const bool round = xf32 && a.N > 32 && part > 1;
    if (round) part = std::min<int64_t>(std::min<int64_t>(part, (int64_t) (half / row)), 0x3fffffff / (a.K / 8) * 256);
    for (int64_t n = 0; n < a.N; n += part) {
        MxParams q = p;
        q.N = std::min(part, a.N - n);
        q.x = (const char *) p.x + n * p.ldx * (xf32 ? 4 : 2);
        q.y = (char *) p.y + n * p.ldy * (p.y_f32 ? 4 : 2);
        q.res = p.res ? p.res + n * p.ldres : nullptr;
        if (round) {
            hipLaunchKernelGGL(mx_round_rows, dim3((unsigned) ((q.N * (a.K / 8) + 255) / 256)), dim3(256), 0, s,
                               (const float *) q.x, a.ldx, (uint16_t *) a.ws, q.N, (int) (a.K / 8));
            q.x = a.ws;
            q.ldx = a.K;
        }
        run_product(q, xf32 && !round, (char *) a.ws + (round ? half : 0), round ? half : a.ws_bytes, s);
    }
    return hipGetLastError();
}

}  // namespace wamx
