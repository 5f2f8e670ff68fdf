// Per-head RMSNorm of queries and keys with the rotation by position, and the
// append to the resident K / V^T cache, in one launch.
//
//   q_h = rot(x_h * rsqrt(mean x_h^2 + eps) * w, pos)      head by head, f32,
//   k_h likewise, v_h unchanged; each result rounded to bf16 once.
//
// rot turns the first n_dims of a head: pair i by pos * base^(-2i / n_dims),
// pairs of neighbours (mode 0) or of the halves (mode 2).  The angle is formed
// in f64 as a fraction of a turn, so positions of any size keep it; v_sin and
// v_cos take turns.
#include "../internal.h"
#include "device.h"

#include <algorithm>
#include <cmath>

namespace wamx {

struct __attribute__((packed, aligned(2))) loose_bf16x8 {
    uint32_t v[4];
};
struct __attribute__((packed, aligned(2))) loose_bf16x4 {
    uint32_t v[2];
};

// The sum over groups of N neighbouring lanes, in each of them: exchanges within
// a row of 16 lanes ride on the additions.
template <int N>
__device__ __forceinline__ float lanes_sum(float x) {
    static_assert(N == 8 || N == 16 || N == 32, "");
#define WAMX_DPP_ADD(ctrl) \
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, false))
    WAMX_DPP_ADD(0xB1);   // quad_perm 1,0,3,2
    WAMX_DPP_ADD(0x4E);   // quad_perm 2,3,0,1
    WAMX_DPP_ADD(0x141);  // row_half_mirror: the other four of eight
    if constexpr (N >= 16) WAMX_DPP_ADD(0x140);  // row_mirror: the other eight
#undef WAMX_DPP_ADD
    if constexpr (N == 32) x = sum_xor16(x);
    return x;
}

struct HeadNormParams {
    const uint16_t * x;
    int64_t ldx;
    const uint16_t * wq;
    const uint16_t * wk;
    const int32_t * pos;
    const int32_t * past;
    uint16_t * q;
    uint16_t * k;
    uint16_t * vt;
    int64_t k_rows, vt_ld;
    int64_t rows;        // batch * tokens
    int32_t tokens, heads, kv_heads, q_col, k_col, v_col;
    int32_t mode, n_dims, pass_heads, chunks;
    int64_t v_wgs;       // workgroups of the value part, the first ones
    int32_t v_tiles;     // slot tiles of a sequence
    float eps;
    double turn[128];    // base^(-2i / n_dims) / 2 pi
};

constexpr int kHnThreads = 256, kHnTile = 64;

// The query and key part is a wave per token and group of pass_heads heads:
// DH / 8 lanes hold a head, each two groups of four values that are turned
// against each other, so the sum of squares stays in registers, a lane forms
// four angles for all heads of a token, and no value changes lanes.  The value
// part, whose workgroups come first, transposes tiles of 64 slots through LDS;
// tiles begin at multiples of 64, so eight slots are one aligned store.
//
// The bytes bound it: 4002 tokens of (32 + 8 + 8) heads of 128 take 23 to 25 us,
// 3.9 to 4.3 TB/s with the launch; one token 4.5 us, which is a launch and three
// dependent reads.  With 16-byte pieces, whose halves' partners lie in other
// lanes, the exchanges and twice the angles took 31.6 us.
template <int DH>
__global__ __launch_bounds__(kHnThreads) void head_norm_rope(HeadNormParams p) {
    constexpr int LPH = DH / 8, HPW = 64 / LPH;
    __shared__ uint16_t tile[kHnTile][DH + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int64_t) blockIdx.x < p.v_wgs) {
        const int64_t id = (int64_t) blockIdx.x;
        const int tt = (int) (id % p.v_tiles);
        const int64_t bh = id / p.v_tiles;
        const int64_t b = bh / p.kv_heads, h = bh - b * p.kv_heads;
        // Tokens [t0, t1) of this tile, whose first slot is a multiple of 64.
        const int64_t past = p.past ? p.past[b] : 0;
        const int shift = (int) (past & (kHnTile - 1));
        const int64_t ta = (int64_t) tt * kHnTile - shift;
        const int64_t t0 = max(ta, (int64_t) 0), t1 = min(ta + kHnTile, (int64_t) p.tokens);
        const uint16_t * src = p.x + (b * p.tokens + ta) * p.ldx + p.v_col + h * DH;
        for (int i = threadIdx.x; i < kHnTile * LPH; i += kHnThreads) {
            const int t = i / LPH, c = i % LPH;
            if (ta + t < t0 || ta + t >= t1) continue;
            const loose_bf16x8 a = *(const loose_bf16x8 *) (src + t * p.ldx + c * 8);
            uint32_t * d = (uint32_t *) &tile[t][c * 8];
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = a.v[j];
        }
        __syncthreads();
        uint16_t * dst = p.vt + bh * DH * p.vt_ld;
        for (int i = threadIdx.x; i < DH * (kHnTile / 8); i += kHnThreads) {
            const int d = i / (kHnTile / 8), t8 = i % (kHnTile / 8) * 8;
            const int64_t t = ta + t8, slot = past + t;
            if (t >= t0 && t + 8 <= t1 && slot >= 0 && slot + 8 <= p.k_rows) {
                loose_bf16x8 o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o.v[j] = tile[t8 + 2 * j][d] | (uint32_t) tile[t8 + 2 * j + 1][d] << 16;
                *(loose_bf16x8 *) (dst + d * p.vt_ld + slot) = o;
            } else {
                for (int j = 0; j < 8; ++j)
                    if (t + j >= t0 && t + j < t1 && slot + j >= 0 && slot + j < p.k_rows)
                        dst[d * p.vt_ld + slot + j] = tile[t8 + j][d];
            }
        }
        return;
    }
    const int64_t w = ((int64_t) blockIdx.x - p.v_wgs) * (kHnThreads / 64) + wave;
    const int64_t row = w / p.chunks;
    if (row >= p.rows) return;
    const int h0 = (int) (w - row * p.chunks) * p.pass_heads;
    const int total = (p.q ? p.heads : 0) + (p.k ? p.kv_heads : 0);
    const int h1 = min(h0 + p.pass_heads, total);
    const int64_t b = row / p.tokens;
    const int t = (int) (row - b * p.tokens);
    // This lane's values: four from da on, four from db on.
    const int l8 = lane % LPH, half = p.n_dims / 2;
    const bool turns = l8 * 8 < p.n_dims, halves = turns && p.mode != 0;
    const int da = halves ? l8 * 4 : l8 * 8, db = halves ? half + l8 * 4 : l8 * 8 + 4;
    const double pos = p.pos ? (double) p.pos[row] : 0.0;
    const int64_t slot = (p.past ? p.past[b] : 0) + (int64_t) t;
    const bool slot_ok = slot >= 0 && slot < p.k_rows;
    const uint16_t * x = p.x + row * p.ldx;
    float cs[4], sn[4];
    if (turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = pos * p.turn[l8 * 4 + i];
            const float f = (float) (a - floor(a));
            cs[i] = __builtin_amdgcn_cosf(f);
            sn[i] = __builtin_amdgcn_sinf(f);
        }
    }

    for (int hb = h0; hb < h1; hb += HPW) {
        const int hh = hb + lane / LPH;
        const int h = min(hh, h1 - 1);  // lanes past the end repeat the last head
        const bool is_q = p.q && h < p.heads;
        const int hk = is_q ? h : h - (p.q ? p.heads : 0);
        const uint16_t * src = x + (is_q ? p.q_col : p.k_col) + hk * DH;
        const uint16_t * wt = is_q ? p.wq : p.wk;
        const loose_bf16x4 in[2] = {*(const loose_bf16x4 *) (src + da), *(const loose_bf16x4 *) (src + db)};
        const loose_bf16x4 wg[2] = {*(const loose_bf16x4 *) (wt + da), *(const loose_bf16x4 *) (wt + db)};
        float v[2][4], ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[e][i] = bf16_to_f32((uint16_t) (in[e].v[i >> 1] >> (16 * (i & 1))));
                ss = fmaf(v[e][i], v[e][i], ss);
            }
        const float r = rsqrtf(lanes_sum<LPH>(ss) * (1.0f / DH) + p.eps);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[e][i] = v[e][i] * r * bf16_to_f32((uint16_t) (wg[e].v[i >> 1] >> (16 * (i & 1))));
        if (turns) {
            // Pair i: (a, b) -> (a cos - b sin, a sin + b cos).
            auto turn = [&](float & a, float & b, int i) {
                const float u = a * cs[i] - b * sn[i];
                b = a * sn[i] + b * cs[i];
                a = u;
            };
            if (p.mode == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(v[i >> 1][2 * (i & 1)], v[i >> 1][2 * (i & 1) + 1], i);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(v[0][i], v[1][i], i);
            }
        }
        if (hh >= h1 || (!is_q && !slot_ok)) continue;
        uint16_t * dst = is_q ? p.q + ((b * p.heads + hk) * p.tokens + t) * DH
                              : p.k + ((b * p.kv_heads + hk) * p.k_rows + slot) * DH;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            loose_bf16x4 out;
            out.v[0] = pack_bf16x2(v[e][0], v[e][1]);
            out.v[1] = pack_bf16x2(v[e][2], v[e][3]);
            *(loose_bf16x4 *) (dst + (e ? db : da)) = out;
        }
    }
}

template <int DH>
static hipError_t run(const HeadNormArgs & a, HeadNormParams & p, hipStream_t s) {
    constexpr int HPW = 64 / (DH / 8);
    const int64_t total = (a.q ? a.heads : 0) + (a.k ? a.kv_heads : 0);
    int64_t qk_wgs = 0;
    p.chunks = 1;
    p.pass_heads = HPW;
    if (total > 0) {
        // One pass of a wave per HPW heads until there are enough waves, then
        // more heads to a wave, evenly: the angles are formed once for them
        // (4002 tokens of 40 heads of 128: a pass a wave 27.6 us, all ten 22.5).
        const int64_t groups = (total + HPW - 1) / HPW, passes = std::max<int64_t>(p.rows * groups / 4096, 1);
        p.chunks = (int32_t) ((groups + passes - 1) / passes);
        p.pass_heads = (int32_t) ((groups + p.chunks - 1) / p.chunks * HPW);
        p.chunks = (int32_t) ((total + p.pass_heads - 1) / p.pass_heads);
        const int64_t per = kHnThreads / 64;
        qk_wgs = (p.rows * p.chunks + per - 1) / per;
    }
    // A first slot inside a tile makes the tokens reach one tile more.
    p.v_tiles = (int32_t) (((int64_t) p.tokens + kHnTile - 1 + (a.past ? kHnTile - 1 : 0)) / kHnTile);
    p.v_wgs = a.vt ? a.batch * a.kv_heads * p.v_tiles : 0;
    const int64_t wgs = qk_wgs + p.v_wgs;
    if (wgs <= 0) return hipSuccess;
    if (wgs > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL(head_norm_rope<DH>, dim3((unsigned) wgs), dim3(kHnThreads), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_head_norm_rope(const HeadNormArgs & a, hipStream_t s) {
    if (a.tokens <= 0 || a.batch <= 0) return hipSuccess;
    if (a.tokens > 0x7fffffff || a.heads > 65535 || a.kv_heads > 65535) return hipErrorInvalidValue;
    HeadNormParams p{};
    p.x = (const uint16_t *) a.x;
    p.ldx = a.ldx;
    p.wq = (const uint16_t *) a.wq;
    p.wk = (const uint16_t *) a.wk;
    p.pos = a.pos;
    p.past = a.past;
    p.q = (uint16_t *) a.q;
    p.k = (uint16_t *) a.k;
    p.vt = (uint16_t *) a.vt;
    p.k_rows = a.k_rows;
    p.vt_ld = a.vt_ld;
    p.rows = a.batch * a.tokens;
    p.tokens = (int32_t) a.tokens;
    p.heads = (int32_t) a.heads;
    p.kv_heads = (int32_t) a.kv_heads;
    p.q_col = (int32_t) a.q_col;
    p.k_col = (int32_t) a.k_col;
    p.v_col = (int32_t) a.v_col;
    p.mode = a.rope_mode;
    p.n_dims = a.n_dims;
    p.eps = a.eps;
    const double ratio = a.n_dims > 0 ? std::pow((double) a.freq_base, -2.0 / a.n_dims) : 1.0;
    double f = 0.15915494309189535;  // 1 / 2 pi
    for (int i = 0; i < a.n_dims / 2; ++i, f *= ratio) p.turn[i] = f;
    switch (a.head_dim) {
        case 64: return run<64>(a, p, s);
        case 128: return run<128>(a, p, s);
        case 256: return run<256>(a, p, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace wamx
