// Attention of a tree of drafted tokens over a resident cache.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,
//   j over the cache slots [0, past) and the slots past + a of token i itself
//   and its ancestors a (parents[]).
//
// K is [slot][dh] and V is held transposed, [dh][slot].  The cache bytes bound
// it: every slot is read once, straight into matrix operands, by one pass that
// carries each row's running maximum and sum.  S^T = K Q^T puts a query in a
// lane's column and, with the slots of two 16-row tiles interleaved, eight
// consecutive slots in its registers: exactly the operand of O^T = V^T P^T, so
// the probabilities never leave the lane.  The rows are the drafted tokens of
// every query head that shares a key head.  The slots are split over the waves
// of a workgroup and over workgroups, whose f32 results a second launch joins.
#include "../internal.h"
#include "device.h"

#include <algorithm>

namespace wamx {

struct TreeParams {
    const uint16_t * q;
    const uint16_t * k;
    const uint16_t * vt;
    const int32_t * parents;
    const int32_t * past;
    uint16_t * out;
    float * po;          // [row][split][dh], or null: one split
    float * pml;         // [row][split][2]
    int64_t capacity, vt_ld;
    int32_t heads, kv_heads, tq, splits;
    float scale;         // times log2 e
};

constexpr int kTreeWaves = 4, kTreeMax = 256, kTreeWords = kTreeMax / 32;

// The path of every token as a bit set, by doubling: after round r a token
// holds the 2^r nearest of its ancestors, and its jump leads past them.  A
// parent outside [-1, tq) marks a slot without a token.
struct TreePaths {
    uint32_t bits[2][kTreeMax][kTreeWords];
    int16_t jump[2][kTreeMax];
};
__device__ __forceinline__ const uint32_t (*tree_paths(TreePaths & s, const int32_t * parents, int tq))[kTreeWords] {
    const int words = (tq + 31) / 32;
    for (int i = threadIdx.x; i < tq; i += blockDim.x) {
        const int pr = parents[i];
        s.jump[0][i] = (int16_t) (pr >= 0 && pr < tq ? pr : -1);
        const bool token = pr >= -1 && pr < tq;
        for (int w = 0; w < words; ++w) s.bits[0][i][w] = token && w == i / 32 ? 1u << (i & 31) : 0u;
    }
    __syncthreads();
    int cur = 0;
    for (int span = 1; span < tq; span *= 2, cur ^= 1) {
        for (int i = threadIdx.x; i < tq; i += blockDim.x) {
            const int j = s.jump[cur][i];
            s.jump[cur ^ 1][i] = j >= 0 ? s.jump[cur][j] : (int16_t) -1;
            for (int w = 0; w < words; ++w) s.bits[cur ^ 1][i][w] = s.bits[cur][i][w] | (j >= 0 ? s.bits[cur][j][w] : 0u);
        }
        __syncthreads();
    }
    return s.bits[cur];
}

__device__ __forceinline__ bool not_finite_bf16(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }

// NR tiles of 16 rows, slots in tiles of 32 HF.
template <int DH, int NR, int HF>
__global__ __launch_bounds__(kTreeWaves * 64) void tree_attn_part(TreeParams p) {
    constexpr int KC = DH / 32, DT = DH / 16, TILE = 32 * HF;
    __shared__ TreePaths paths;
    __shared__ __align__(16) f32x4_t red[kTreeWaves][DT * 64];
    __shared__ float rm[kTreeWaves][NR][16], rl[kTreeWaves][NR][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c16 = lane & 15, g = lane >> 4;
    const int split = blockIdx.x;
    const int64_t bz = blockIdx.z;
    const int b = (int) (bz / p.kv_heads), hk = (int) (bz - (int64_t) b * p.kv_heads);
    const int group = p.heads / p.kv_heads, rows = group * p.tq, row0 = blockIdx.y * 16 * NR;

    // A length that does not fit leaves its sequence without keys.
    const int64_t past = p.past ? p.past[b] : 0;
    const int64_t n = past >= 0 && past + p.tq <= p.capacity ? past + p.tq : 0;
    const int64_t tiles = (n + TILE - 1) / TILE;
    const int64_t t0 = tiles * split / p.splits, t1 = tiles * (split + 1) / p.splits;
    const int32_t * parents = p.parents + (int64_t) b * p.tq;
    const uint32_t (*path)[kTreeWords] = paths.bits[0];
    if (t1 * TILE > past) path = tree_paths(paths, parents, p.tq);

    const uint16_t * kb = p.k + bz * p.capacity * DH;
    const uint16_t * vb = p.vt + bz * DH * p.vt_ld;

    // This lane's query of each row tile.
    int tok[NR];
    bool token[NR];
    bf16x8_t qf[NR][KC];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int row = min(row0 + i * 16 + c16, rows - 1);
        tok[i] = row % p.tq;
        const int pr = parents[tok[i]];
        token[i] = pr >= -1 && pr < p.tq;
        const uint16_t * qr = p.q + (((int64_t) b * p.heads + hk * group + row / p.tq) * p.tq + tok[i]) * DH;
#pragma unroll
        for (int c = 0; c < KC; ++c) qf[i][c] = *(const bf16x8_t *) (qr + c * 32 + g * 8);
    }
    float m[NR], l[NR];
    f32x4_t o[NR][DT];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[i][d] = (f32x4_t){0, 0, 0, 0};
    }

    for (int64_t kt = t0 + wave; kt < t1; kt += kTreeWaves) {
        const int64_t base = kt * TILE;
        f32x4_t s[NR][2 * HF];
#pragma unroll
        for (int u = 0; u < 2 * HF; ++u) {
            // Row a of tile u is slot 8 (a / 4) + 4 (u % 2) + a % 4 of its half.
            const int64_t slot = min(base + (u >> 1) * 32 + 8 * (c16 >> 2) + 4 * (u & 1) + (c16 & 3), n - 1);
            bf16x8_t kf[KC];
#pragma unroll
            for (int c = 0; c < KC; ++c) kf[c] = *(const bf16x8_t *) (kb + slot * DH + c * 32 + g * 8);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                s[i][u] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < KC; ++c)
                    s[i][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[c], qf[i][c], s[i][u], 0, 0, 0);
            }
        }
        const bool edge = base + TILE > past;  // drafted slots, or the end, in this tile
        bf16x8_t pf[NR][HF];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2 * HF; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = s[i][u][r] * p.scale;
                    if (edge) {
                        const int64_t slot = base + (u >> 1) * 32 + 8 * g + 4 * (u & 1) + r;
                        bool seen = slot < past;
                        if (slot >= past && slot < n) {
                            const int a = (int) (slot - past);
                            seen = path[tok[i]][a >> 5] >> (a & 31) & 1;
                        }
                        v = seen ? v : -INFINITY;
                    }
                    s[i][u][r] = v;
                    top = fmaxf(top, v);
                }
            top = max_xor32(max_xor16(top));
            const float mn = fmaxf(m[i], top);
            const float base_m = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m[i] - base_m);
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2 * HF; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[i][u][r] = __builtin_amdgcn_exp2f(s[i][u][r] - base_m);
                    sum += s[i][u][r];
                }
            l[i] = l[i] * alpha + sum;
            if (__any(mn != m[i])) {
#pragma unroll
                for (int d = 0; d < DT; ++d) o[i][d] *= alpha;
            }
            m[i] = mn;
#pragma unroll
            for (int h = 0; h < HF; ++h) {
                union {
                    uint32_t d[4];
                    bf16x8_t v;
                } pk;
                pk.d[0] = pack_bf16x2(s[i][2 * h][0], s[i][2 * h][1]);
                pk.d[1] = pack_bf16x2(s[i][2 * h][2], s[i][2 * h][3]);
                pk.d[2] = pack_bf16x2(s[i][2 * h + 1][0], s[i][2 * h + 1][1]);
                pk.d[3] = pack_bf16x2(s[i][2 * h + 1][2], s[i][2 * h + 1][3]);
                pf[i][h] = pk.v;
            }
        }
        bool bad = false;
#pragma unroll
        for (int h = 0; h < HF; ++h) {
            const int64_t v0 = base + h * 32 + g * 8;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                union {
                    uint32_t w[4];
                    bf16x8_t v;
                } vf;
                vf.v = (bf16x8_t){};
                if (v0 < p.vt_ld) vf.v = *(const bf16x8_t *) (vb + (int64_t) (d * 16 + c16) * p.vt_ld + v0);
                if (edge) {
                    // Slots behind the last hold anything; a drafted slot's
                    // values must not reach the rows that do not see it, which
                    // for Inf and NaN takes the path below.
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t e = vf.w[j >> 1] >> (16 * (j & 1));
                        const bool drafted = v0 + j >= past;
                        const bool odd = drafted && v0 + j < n && not_finite_bf16(e);
                        bad |= odd;
                        if (odd || v0 + j >= n) vf.w[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    }
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf.v, pf[i][h], o[i][d], 0, 0, 0);
            }
        }
        if (edge && __any(bad)) {
            // Inf or NaN among the drafted values: added element by element to
            // the rows whose path holds the slot.
            float * pl = (float *) red[wave];  // [TILE][16], this wave's own
#pragma unroll
            for (int i = 0; i < NR; ++i) {
#pragma unroll
                for (int u = 0; u < 2 * HF; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) pl[((u >> 1) * 32 + 8 * g + 4 * (u & 1) + r) * 16 + c16] = s[i][u][r];
                __builtin_amdgcn_wave_barrier();
                for (int64_t slot = max(base, past); slot < min(base + TILE, n); ++slot) {
                    const int a = (int) (slot - past);
                    if (!(path[tok[i]][a >> 5] >> (a & 31) & 1)) continue;
                    const float pr = pl[(int) (slot - base) * 16 + c16];
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t e = vb[(int64_t) (d * 16 + 4 * g + r) * p.vt_ld + slot];
                            if (not_finite_bf16(e)) o[i][d][r] += pr * bf16_to_f32((uint16_t) e);
                        }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    }

    // The waves' results, joined in wave order.
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        l[i] = sum_xor32(sum_xor16(l[i]));
        if (g == 0) {
            rm[wave][i][c16] = m[i];
            rl[wave][i][c16] = l[i];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) top = fmaxf(top, rm[w][i][c16]);
        const float base_m = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(m[i] - base_m);
#pragma unroll
        for (int d = 0; d < DT; ++d) red[wave][d * 64 + lane] = o[i][d] * f;
        __syncthreads();
        for (int e = threadIdx.x; e < DT * 64; e += kTreeWaves * 64) {
            const int q = e & 15, d = (e >> 6) * 16 + ((e >> 4) & 3) * 4;
            const int row = row0 + i * 16 + q;
            float big = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kTreeWaves; ++w) big = fmaxf(big, rm[w][i][q]);
            const float bm = big == -INFINITY ? 0.0f : big;
            f32x4_t v = red[0][e];
            sum = rl[0][i][q] * __builtin_amdgcn_exp2f(rm[0][i][q] - bm);
#pragma unroll
            for (int w = 1; w < kTreeWaves; ++w) {
                v += red[w][e];
                sum += rl[w][i][q] * __builtin_amdgcn_exp2f(rm[w][i][q] - bm);
            }
            if (row >= rows) continue;
            const int t = row % p.tq;
            const int pr = parents[t];
            const bool has = pr >= -1 && pr < p.tq;
            if (p.po) {
                const int64_t at = (bz * rows + row) * p.splits + split;
                *(f32x4_t *) (p.po + at * DH + d) = v;
                if (d == 0) {
                    p.pml[2 * at] = has ? big : -INFINITY;
                    p.pml[2 * at + 1] = has ? sum : 0.0f;
                }
            } else {
                const float inv = 1.0f / sum;
                const bool none = !has || (sum == 0.0f && big == -INFINITY);
                uint32_t w[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) w[r] = none ? 0u : pack_bf16x2(v[2 * r] * inv, v[2 * r + 1] * inv);
                uint16_t * y = p.out + (((int64_t) b * p.tq + t) * p.heads + hk * group + row / p.tq) * DH + d;
                *(uint32_t *) y = w[0];
                *(uint32_t *) (y + 2) = w[1];
            }
        }
        __syncthreads();
    }
}

// out = sum_s po_s 2^(m_s - m) / sum_s l_s 2^(m_s - m), splits in order: a wave
// per row, DH / 64 values a lane.
template <int DH>
__global__ __launch_bounds__(256) void tree_attn_join(TreeParams p, int64_t total) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= total) return;
    const int group = p.heads / p.kv_heads, rows = group * p.tq;
    const int64_t bz = at / rows;
    const int row = (int) (at - bz * rows);
    const int64_t b = bz / p.kv_heads;
    const int hk = (int) (bz - b * p.kv_heads);
    const float * ml = p.pml + at * p.splits * 2;
    float m = -INFINITY;
    for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, ml[2 * s]);
    m = wave_max(m);
    constexpr int V = DH / 64;
    float acc[V] = {}, sum = 0.0f;
    const float * po = p.po + at * p.splits * DH + lane * V;
    if (m != -INFINITY) {
        for (int s = 0; s < p.splits; ++s) {
            const float f = __builtin_amdgcn_exp2f(ml[2 * s] - m);
            sum += ml[2 * s + 1] * f;
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] += po[(int64_t) s * DH + v] * f;
        }
    }
    uint16_t * y = p.out + ((b * p.tq + row % p.tq) * p.heads + hk * group + row / p.tq) * DH + lane * V;
    const float inv = m == -INFINITY ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = m == -INFINITY ? 0 : f32_to_bf16(acc[v] * inv);
}

template <int DH, int NR, int HF>
static hipError_t run(TreeParams & p, const TreeArgs & a, hipStream_t s) {
    const int64_t bz = a.batch * a.kv_heads, rows = a.heads / a.kv_heads * a.tq, rt = (rows + 16 * NR - 1) / (16 * NR);
    if (bz > 65535 || rt > 65535) return hipErrorInvalidValue;
    // Splits: two workgroups per CU when the cache is long enough for each to
    // have eight tiles, as far as the workspace holds their results.
    const int64_t tiles = (a.capacity + 32 * HF - 1) / (32 * HF);
    int64_t splits = std::min<int64_t>(512 / std::max<int64_t>(bz * rt, 1), tiles / 8);
    const size_t per = (size_t) (bz * rows) * (DH + 2) * 4;
    if (!a.ws) splits = 1;
    else splits = std::min<int64_t>(splits, (int64_t) (a.ws_bytes / std::max<size_t>(per, 1)));
    if (splits < 2) splits = 1;
    p.splits = (int32_t) splits;
    if (splits > 1) {
        p.po = (float *) a.ws;
        p.pml = p.po + bz * rows * splits * DH;
    }
    hipLaunchKernelGGL((tree_attn_part<DH, NR, HF>), dim3((unsigned) splits, (unsigned) rt, (unsigned) bz),
                       dim3(kTreeWaves * 64), 0, s, p);
    if (splits > 1)
        hipLaunchKernelGGL(tree_attn_join<DH>, dim3((unsigned) ((bz * rows + 3) / 4)), dim3(256), 0, s, p, bz * rows);
    return hipGetLastError();
}

hipError_t launch_tree_attn(const TreeArgs & a, hipStream_t s) {
    if (a.tq <= 0 || a.batch <= 0) return hipSuccess;
    if (a.tq > kTreeMax || a.heads <= 0 || a.kv_heads <= 0 || a.heads % a.kv_heads != 0 || a.vt_ld % 8 != 0 ||
        a.vt_ld < a.capacity || a.capacity <= 0)
        return hipErrorInvalidValue;
    TreeParams p{};
    p.q = (const uint16_t *) a.q;
    p.k = (const uint16_t *) a.k;
    p.vt = (const uint16_t *) a.vt;
    p.parents = a.parents;
    p.past = a.past;
    p.out = (uint16_t *) a.out;
    p.capacity = a.capacity;
    p.vt_ld = a.vt_ld;
    p.heads = (int32_t) a.heads;
    p.kv_heads = (int32_t) a.kv_heads;
    p.tq = (int32_t) a.tq;
    p.scale = a.scale * 1.4426950408889634f;
    const int64_t rows = a.heads / a.kv_heads * a.tq;
    switch (a.head_dim) {
        case 64:
            return rows <= 16 ? run<64, 1, 2>(p, a, s) : rows <= 32 ? run<64, 2, 2>(p, a, s) : run<64, 4, 2>(p, a, s);
        case 128:
            return rows <= 16 ? run<128, 1, 2>(p, a, s) : rows <= 32 ? run<128, 2, 2>(p, a, s) : run<128, 4, 1>(p, a, s);
        case 256: return rows <= 16 ? run<256, 1, 1>(p, a, s) : run<256, 2, 1>(p, a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace wamx
