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

// A barrier that waits for this wave's LDS accesses alone: loads into registers
// stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), other counters untouched
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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

// Values of packed blocks: the reverse path (blocks through LDS, eight values
// per lane).  ldy is the row stride of y in elements; qs the byte stride of
// packed rows (row_blocks * 17 when they follow each other); rows (nullable)
// picks row rows[r] of `qrows` packed rows (negative or past the end: NaN).
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
    float * part;  // K-split planes [split][N][M], or null
    int steps;     // K steps of 128 of one split
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

// Few tokens: the weight bytes bound it, so every one is read once, in
// 16-byte pieces, and goes straight into matrix operands.  A workgroup takes
// RG groups of 16 weight rows and NT tiles of 16 tokens; its waves take the K
// steps of 128 in turn (a row's 68 bytes of a step lie next to the next
// wave's) and their sums meet in LDS in wave order.  Lane (r, g) holds block g
// of the step for weight row r, and the same 32 values of x for token r.
constexpr int kMxWaves = 8;

template <int RG, int NT, bool XF32>
__global__ __launch_bounds__(kMxWaves * 64) void mx_few(MxParams p) {
    __shared__ __align__(16) f32x4_t red[kMxWaves][RG * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int64_t m0 = (int64_t) blockIdx.x * (16 * RG), n0 = (int64_t) blockIdx.y * (16 * NT);
    const int s0 = (int) blockIdx.z * p.steps, s1 = min(s0 + p.steps, (p.kb + 3) / 4);

    const uint8_t * w[RG];
    const char * x[NT];
    constexpr int xs = XF32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < RG; ++i) w[i] = p.w + min(m0 + i * 16 + r, p.M - 1) * p.ws;
#pragma unroll
    for (int j = 0; j < NT; ++j) x[j] = (const char *) p.x + min(n0 + j * 16 + r, p.N - 1) * p.ldx * xs;

    struct Step {
        any16 w[RG];
        uint32_t e[RG];
        uint32_t x[NT][16];
    };
    auto load = [&](int s, Step & t) {
        const int kb = 4 * s + g;
        const bool in = kb < p.kb;
        const int64_t at = in ? kb : p.kb - 1;
#pragma unroll
        for (int i = 0; i < RG; ++i) {
            const uint8_t * b = w[i] + at * kMxBytes;
            t.w[i] = *(const any16 *) (b + 1);
            t.e[i] = b[0];
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if constexpr (XF32) {
                const char * b = x[j] + at * 128;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const any16 a = *(const any16 *) (b + 16 * c);
                    t.x[j][2 * c] = pack_bf16x2(__uint_as_float(a.v[0]), __uint_as_float(a.v[1]));
                    t.x[j][2 * c + 1] = pack_bf16x2(__uint_as_float(a.v[2]), __uint_as_float(a.v[3]));
                }
            } else {
                const char * b = x[j] + at * 64;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const any16 a = *(const any16 *) (b + 16 * c);
#pragma unroll
                    for (int d = 0; d < 4; ++d) t.x[j][4 * c + d] = a.v[d];
                }
            }
        }
        if (!in) {
            // Past the row's last block: nothing times nothing.
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                t.e[i] = 0;
#pragma unroll
                for (int d = 0; d < 4; ++d) t.w[i].v[d] = 0;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int d = 0; d < 16; ++d) t.x[j][d] = 0;
        }
    };

    f32x4_t acc[RG][NT];
#pragma unroll
    for (int i = 0; i < RG; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};
    Step cur;
    for (int s = s0 + wave; s < s1; s += kMxWaves) {
        load(s, cur);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            bf16x8_t b[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                b[j] = mx_pair(cur.x[j][2 * d], cur.x[j][2 * d + 1], cur.x[j][8 + 2 * d], cur.x[j][8 + 2 * d + 1]);
#pragma unroll
            for (int i = 0; i < RG; ++i) {
                const bf16x8_t a = mx_frag(cur.w[i].v[d], mx_scale(cur.e[i]));
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[j], acc[i][j], 0, 0, 0);
            }
        }
    }
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

template <int RG, int NT>
static void launch_few(const MxParams & p, bool xf32, hipStream_t s) {
    const dim3 grid((unsigned) ((p.M + 16 * RG - 1) / (16 * RG)), (unsigned) ((p.N + 16 * NT - 1) / (16 * NT)), 1);
    if (xf32) hipLaunchKernelGGL((mx_few<RG, NT, true>), grid, dim3(kMxWaves * 64), 0, s, p);
    else hipLaunchKernelGGL((mx_few<RG, NT, false>), grid, dim3(kMxWaves * 64), 0, s, p);
}

// Many tokens: matrix-core bound.  Eight waves, 2 along the weight rows by 4
// along the tokens, each RG x NT tiles of 16 x 16 (so RG * 32 rows by NT * 64
// tokens a workgroup).  The weight stays in its 4 bits down to the register
// that becomes the operand: a step of 128 values is 4 blocks a row, whose codes
// lie in LDS as [row][pair of blocks][g][block of the pair], so that one
// 8-byte read gives lane (r, g) dword g of both blocks of a pair.  Such a dword
// expands to values (4g + t, 16 + 4g + t), t = 0..3, of its block, and x is
// written to LDS in that order (two 16-byte pieces 16 values apart, interleaved
// on the way), half a step at a time.  Both go through registers into one of
// two buffers while the other is multiplied: one barrier per half step.
template <bool XF32>
struct MxPiece {  // eight consecutive activations
    any16 v[XF32 ? 2 : 1];
};

template <int RG, int NT, bool XF32>
__global__ __launch_bounds__(512) void mx_tile(MxParams p) {
    constexpr int BM = RG * 32, BN = NT * 64, XP = BN * 8 / 512;  // x pieces of a thread per half step
    constexpr int WB = (BM * 4 + 511) / 512;                      // weight blocks of a thread per step
    static_assert(XP % 2 == 0, "pieces come in pairs");
    __shared__ __align__(16) uint32_t wl[2][BM * 16];
    __shared__ __align__(16) float sl[2][BM * 4];
    __shared__ __align__(16) uint32_t xl[2][BN * 32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4, wm = wave >> 2, wn = wave & 3;
    const int64_t m0 = (int64_t) blockIdx.x * BM, n0 = (int64_t) blockIdx.y * BN;
    const int s0 = (int) blockIdx.z * p.steps, s1 = min(s0 + p.steps, (p.kb + 3) / 4);
    constexpr int xs = XF32 ? 4 : 2;

    // Weight blocks: thread t takes block t % 4 of rows t / 4, t / 4 + 128, ...
    const int wkb = threadIdx.x & 3, wrow = threadIdx.x >> 2;
    const uint8_t * wsrc[WB];
#pragma unroll
    for (int j = 0; j < WB; ++j) wsrc[j] = p.w + min(m0 + wrow + j * 128, p.M - 1) * p.ws;
    any16 wr[WB];
    uint32_t wsc[WB];
    auto request_w = [&](int s) {
        const int kb = 4 * s + wkb;
        const int64_t at = min(kb, p.kb - 1) * (int64_t) kMxBytes;
#pragma unroll
        for (int j = 0; j < WB; ++j) {
            wr[j] = *(const any16 *) (wsrc[j] + at + 1);
            wsc[j] = wsrc[j][at];
            if (kb >= p.kb) {
                wsc[j] = 0;
#pragma unroll
                for (int d = 0; d < 4; ++d) wr[j].v[d] = 0;
            }
        }
    };
    auto deposit_w = [&](int buf) {
#pragma unroll
        for (int j = 0; j < WB; ++j) {
            const int row = wrow + j * 128;
            if (BM % 128 != 0 && row >= BM) break;
#pragma unroll
            for (int d = 0; d < 4; ++d) wl[buf][row * 16 + (wkb >> 1) * 8 + d * 2 + (wkb & 1)] = wr[j].v[d];
            sl[buf][row * 4 + wkb] = mx_scale(wsc[j]);
        }
    };
    // Activations: pair q of a thread is the pieces at 8c and 16 + 8c of a
    // 32-value block, c = 0, 1.
    MxPiece<XF32> xr[XP];
    const char * xsrc[XP / 2];
    int xpos[XP / 2];
#pragma unroll
    for (int q = 0; q < XP / 2; ++q) {
        const int e = threadIdx.x + q * 512, row = e >> 2, i = (e >> 1) & 1, c = e & 1;
        xsrc[q] = (const char *) p.x + (min(n0 + row, p.N - 1) * p.ldx + i * 32 + c * 8) * xs;
        xpos[q] = row * 8 + ((i * 4 + c * 2) ^ ((row >> 1) & 7));  // 16-byte slot of operand g = 2c; g + 1 in slot ^ 1
    }
    auto request_x = [&](int h) {  // half step h: blocks 2h, 2h + 1
#pragma unroll
        for (int q = 0; q < XP / 2; ++q) {
            const int kb = 2 * h + ((threadIdx.x >> 1) & 1);
            const bool in = kb < p.kb;
            const char * a = xsrc[q] + (in ? (int64_t) h * 64 : 0) * xs - (in ? 0 : ((threadIdx.x >> 1) & 1) * 32 * xs);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < (XF32 ? 2 : 1); ++v) {
                    xr[2 * q + u].v[v] = *(const any16 *) (a + u * 16 * xs + v * 16);
                    if (!in) {
#pragma unroll
                        for (int d = 0; d < 4; ++d) xr[2 * q + u].v[v].v[d] = 0;
                    }
                }
        }
    };
    auto deposit_x = [&](int buf) {
#pragma unroll
        for (int q = 0; q < XP / 2; ++q) {
            uint32_t lo[4], hi[4];
            if constexpr (XF32) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const any16 &a = xr[2 * q].v[d >> 1], &b = xr[2 * q + 1].v[d >> 1];
                    lo[d] = pack_bf16x2(__uint_as_float(a.v[2 * (d & 1)]), __uint_as_float(a.v[2 * (d & 1) + 1]));
                    hi[d] = pack_bf16x2(__uint_as_float(b.v[2 * (d & 1)]), __uint_as_float(b.v[2 * (d & 1) + 1]));
                }
            } else {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    lo[d] = xr[2 * q].v[0].v[d];
                    hi[d] = xr[2 * q + 1].v[0].v[d];
                }
            }
            bf16x8_t * dst = (bf16x8_t *) xl[buf];
            dst[xpos[q]] = mx_pair(lo[0], lo[1], hi[0], hi[1]);
            dst[xpos[q] ^ 1] = mx_pair(lo[2], lo[3], hi[2], hi[3]);
        }
    };

    f32x4_t acc[RG][NT];
#pragma unroll
    for (int i = 0; i < RG; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4_t){0, 0, 0, 0};
    auto multiply = [&](int wbuf, int half, int xbuf) {
        bf16x8_t b[2][NT];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int row = (wn * NT + j) * 16 + c16;
                b[i][j] = ((const bf16x8_t *) xl[xbuf])[row * 8 + ((i * 4 + g) ^ ((row >> 1) & 7))];
            }
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            const int row = (wm * RG + r) * 16 + c16;
            const uint2 d = *(const uint2 *) &wl[wbuf][row * 16 + half * 8 + g * 2];
            const float2 sc = *(const float2 *) &sl[wbuf][row * 4 + half * 2];
            const bf16x8_t a0 = mx_frag(d.x, sc.x), a1 = mx_frag(d.y, sc.y);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b[0][j], acc[r][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b[1][j], acc[r][j], 0, 0, 0);
        }
    };
    if (s0 < s1) {
        request_w(s0);
        request_x(2 * s0);
        deposit_w(0);
        deposit_x(0);
    }
    lds_barrier();
    for (int s = s0; s < s1; ++s) {
        const int wb = (s - s0) & 1;
        request_x(2 * s + 1);
        if (s + 1 < s1) request_w(s + 1);
        multiply(wb, 0, 0);
        deposit_x(1);
        lds_barrier();
        if (s + 1 < s1) request_x(2 * s + 2);
        multiply(wb, 1, 1);
        if (s + 1 < s1) {
            deposit_x(0);
            deposit_w(wb ^ 1);
        }
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

template <int RG, int NT>
static void launch_tile(const MxParams & p, bool xf32, hipStream_t s) {
    const dim3 grid((unsigned) ((p.M + RG * 32 - 1) / (RG * 32)), (unsigned) ((p.N + NT * 64 - 1) / (NT * 64)), 1);
    if (xf32) hipLaunchKernelGGL((mx_tile<RG, NT, true>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((mx_tile<RG, NT, false>), grid, dim3(512), 0, s, p);
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
    if (a.K <= 0 || a.K % 32 != 0 || a.K / 32 > 0x7fffffff) return hipErrorInvalidValue;
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
    if (a.N <= 16) launch_few<1, 1>(p, xf32, s);
    else if (a.N <= 32) launch_few<1, 2>(p, xf32, s);
    else if (a.N <= 64) launch_few<2, 4>(p, xf32, s);
    else if (a.N <= 600) launch_tile<4, 2>(p, xf32, s);
    else launch_tile<8, 4>(p, xf32, s);
    return hipGetLastError();
}

}  // namespace wamx
