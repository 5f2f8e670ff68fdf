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
    int64_t qk_wgs;      // workgroups of the query and key part
    int32_t v_tiles;     // token tiles of a sequence
    float eps;
    double turn[128];    // base^(-2i / n_dims) / 2 pi
};

constexpr int kHnThreads = 256, kHnTile = 64;

// The query and key part is a wave per token and group of pass_heads heads:
// DH / 8 lanes hold a head, eight values each, so the sum of squares stays in
// registers and the angles of a token are formed once for all its heads.  The
// value part transposes tiles of 64 tokens through LDS.
template <int DH>
__global__ __launch_bounds__(kHnThreads) void head_norm_rope(HeadNormParams p) {
    constexpr int LPH = DH / 8, HPW = 64 / LPH;
    __shared__ uint16_t tile[kHnTile][DH + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int64_t) blockIdx.x >= p.qk_wgs) {
        const int64_t id = (int64_t) blockIdx.x - p.qk_wgs;
        const int tt = (int) (id % p.v_tiles);
        const int64_t bh = id / p.v_tiles;
        const int64_t b = bh / p.kv_heads, h = bh - b * p.kv_heads;
        const int t0 = tt * kHnTile, nt = min(p.tokens - t0, kHnTile);
        const uint16_t * src = p.x + (b * p.tokens + t0) * p.ldx + p.v_col + h * DH;
        for (int i = threadIdx.x; i < nt * LPH; i += kHnThreads) {
            const int t = i / LPH, c = i % LPH;
            const loose_bf16x8 a = *(const loose_bf16x8 *) (src + t * p.ldx + c * 8);
            uint32_t * d = (uint32_t *) &tile[t][c * 8];
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = a.v[j];
        }
        __syncthreads();
        const int64_t slot0 = (p.past ? p.past[b] : 0) + (int64_t) t0;
        uint16_t * dst = p.vt + bh * DH * p.vt_ld;
        for (int i = threadIdx.x; i < nt * DH; i += kHnThreads) {
            const int d = i / nt, t = i - d * nt;
            const int64_t slot = slot0 + t;
            if (slot >= 0 && slot < p.k_rows) dst[d * p.vt_ld + slot] = tile[t][d];
        }
        return;
    }
    const int64_t w = (int64_t) blockIdx.x * (kHnThreads / 64) + wave;
    const int64_t row = w / p.chunks;
    if (row >= p.rows) return;
    const int h0 = (int) (w - row * p.chunks) * p.pass_heads;
    const int total = (p.q ? p.heads : 0) + (p.k ? p.kv_heads : 0);
    const int h1 = min(h0 + p.pass_heads, total);
    const int64_t b = row / p.tokens;
    const int t = (int) (row - b * p.tokens);
    const int d0 = (lane % LPH) * 8;

    // Angles of this lane's values.
    const double pos = p.pos ? (double) p.pos[row] : 0.0;
    const bool turns = d0 < p.n_dims;
    const int half = p.n_dims / 2;
    float cs[8], sn[8];
    if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (p.mode == 0 && (i & 1)) {
                cs[i] = cs[i - 1];
                sn[i] = sn[i - 1];
                continue;
            }
            const int pair = p.mode == 0 ? (d0 + i) / 2 : d0 < half ? d0 + i : d0 + i - half;
            const double a = pos * p.turn[pair];
            const float f = (float) (a - floor(a));
            cs[i] = __builtin_amdgcn_cosf(f);
            sn[i] = __builtin_amdgcn_sinf(f);
        }
    }
    const int partner = !turns ? lane : d0 < half ? lane + half / 8 : lane - half / 8;
    const int64_t slot = (p.past ? p.past[b] : 0) + (int64_t) t;
    const bool slot_ok = slot >= 0 && slot < p.k_rows;

    for (int hb = h0; hb < h1; hb += HPW) {
        const int hh = hb + lane / LPH;
        const int h = min(hh, h1 - 1);  // lanes past the end repeat the last head
        const bool is_q = p.q && h < p.heads;
        const int hk = is_q ? h : h - (p.q ? p.heads : 0);
        const uint16_t * src = p.x + row * p.ldx + (is_q ? p.q_col : p.k_col) + (int64_t) hk * DH + d0;
        const loose_bf16x8 a = *(const loose_bf16x8 *) src;
        const loose_bf16x8 g = *(const loose_bf16x8 *) ((is_q ? p.wq : p.wk) + d0);
        float v[8], ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = bf16_to_f32((uint16_t) (a.v[i >> 1] >> (16 * (i & 1))));
            ss = fmaf(v[i], v[i], ss);
        }
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o);
        const float r = rsqrtf(ss * (1.0f / DH) + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * bf16_to_f32((uint16_t) (g.v[i >> 1] >> (16 * (i & 1))));
        float o[8];
        if (p.mode == 0) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                o[i] = turns ? v[i] * cs[i] - v[i + 1] * sn[i] : v[i];
                o[i + 1] = turns ? v[i] * sn[i] + v[i + 1] * cs[i] : v[i + 1];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = __shfl(v[i], partner);
                o[i] = !turns ? v[i] : d0 < half ? v[i] * cs[i] - u * sn[i] : u * sn[i] + v[i] * cs[i];
            }
        }
        if (hh >= h1 || (!is_q && !slot_ok)) continue;
        loose_bf16x8 out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out.v[i] = pack_bf16x2(o[2 * i], o[2 * i + 1]);
        uint16_t * dst = is_q ? p.q + ((b * p.heads + hk) * p.tokens + t) * DH + d0
                              : p.k + ((b * p.kv_heads + hk) * p.k_rows + slot) * DH + d0;
        *(loose_bf16x8 *) dst = out;
    }
}

template <int DH>
static hipError_t run(const HeadNormArgs & a, HeadNormParams & p, hipStream_t s) {
    constexpr int HPW = 64 / (DH / 8);
    const int64_t total = (a.q ? a.heads : 0) + (a.k ? a.kv_heads : 0);
    p.qk_wgs = 0;
    p.chunks = 1;
    p.pass_heads = HPW;
    if (total > 0) {
        // One pass of a wave per HPW heads until the waves would outnumber the
        // GPU's slots, then more heads to a wave.
        const int64_t waves = p.rows * ((total + HPW - 1) / HPW);
        const int64_t passes = std::min<int64_t>(std::max<int64_t>(waves / 8192, 1), 16);
        p.pass_heads = (int32_t) std::min<int64_t>(passes * HPW, (total + HPW - 1) / HPW * HPW);
        p.chunks = (int32_t) ((total + p.pass_heads - 1) / p.pass_heads);
        const int64_t per = kHnThreads / 64;
        p.qk_wgs = (p.rows * p.chunks + per - 1) / per;
    }
    p.v_tiles = (p.tokens + kHnTile - 1) / kHnTile;
    const int64_t wgs = p.qk_wgs + (a.vt ? a.batch * a.kv_heads * p.v_tiles : 0);
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
