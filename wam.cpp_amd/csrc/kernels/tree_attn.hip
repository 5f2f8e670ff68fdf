// Attention of a tree of drafted tokens over a resident cache.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,
//   j over the cache slots [0, past) and the slots past + a of token i itself
//   and its ancestors a (parents[]).
//
// K is [slot][dh] and V is held transposed, [dh][slot].  The cache's bytes bound
// a few rows, the softmax's arithmetic and the products many; one pass over the
// slots carries each row's running maximum and sum.  S^T = K Q^T puts a query
// into a lane's column, the layout in which its probabilities are the operand
// of O^T = V^T P^T.  The rows are the drafted tokens of every query head that
// shares a key head, so the slots are read once for all of them.  The slots are
// split over workgroups, whose f32 results a second launch joins.
#include "../internal.h"
#include "device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace wamx {

struct TreeParams {
    const uint16_t * q;
    const uint16_t * k;
    const uint16_t * vt;
    const int32_t * parents;
    const int32_t * past;
    uint16_t * out;
    float * po;          // [unit][key head][row][dh], or null: nothing split
    float * pml;         // [unit][key head][row][2]
    int64_t capacity, vt_ld;
    int32_t heads, kv_heads, tq, batch;
    int32_t even;        // units / batch for every sequence
    int32_t units;       // parts of all sequences' slots, for each key head
    float scale;         // times log2 e, positive
    uint32_t q_and, q_xor;  // on pairs of Q's bits: the scale's sign, or 0
};

constexpr int kTreeWaves = 4, kTreeMax = 256, kTreeWords = kTreeMax / 32;

// The path of every token as a bit set, by doubling: after round r a token
// holds the 2^r nearest of its ancestors, and its jump leads past them.  A
// parent outside [-1, tq) marks a slot without a token.  `work` is LDS that the
// workgroup uses for something else afterwards (a barrier ends this).
struct TreeWork {
    uint32_t bits[kTreeMax][kTreeWords];
    int16_t jump[2][kTreeMax];
};
typedef uint32_t TreePaths[kTreeMax][kTreeWords];
__device__ __forceinline__ void tree_paths(TreePaths & path, void * work, int parent, int tq) {
    TreeWork & w = *(TreeWork *) work;
    const int words = (tq + 31) / 32;
    int rounds = 0;
    while ((1 << rounds) < tq) ++rounds;
    // The last round writes `path`.
    uint32_t (*from)[kTreeWords] = rounds & 1 ? w.bits : path;
    uint32_t (*to)[kTreeWords] = rounds & 1 ? path : w.bits;
    const int i = threadIdx.x;
    if (i < tq) {
        w.jump[0][i] = (int16_t) (parent >= 0 && parent < tq ? parent : -1);
        const bool token = parent >= -1 && parent < tq;
        for (int k = 0; k < words; ++k) from[i][k] = token && k == i / 32 ? 1u << (i & 31) : 0u;
    }
    __syncthreads();
    for (int r = 0; r < rounds; ++r) {
        if (i < tq) {
            const int j = w.jump[r & 1][i];
            w.jump[(r & 1) ^ 1][i] = j >= 0 ? w.jump[r & 1][j] : (int16_t) -1;
            for (int k = 0; k < words; ++k) to[i][k] = from[i][k] | (j >= 0 ? from[j][k] : 0u);
        }
        __syncthreads();
        uint32_t (*t)[kTreeWords] = from;
        from = to;
        to = t;
    }
}

// The same for at most 64 tokens, lane i's in a register of every wave.
__device__ __forceinline__ uint64_t tree_path(int parent, int tq) {
    const int lane = threadIdx.x & 63;
    int jump = parent >= 0 && parent < tq ? parent : -1;
    const bool token = lane < tq && parent >= -1 && parent < tq;
    uint32_t lo = token && lane < 32 ? 1u << lane : 0u, hi = token && lane >= 32 ? 1u << (lane - 32) : 0u;
    for (int reach = 1; reach < tq; reach *= 2) {
        const int from = max(jump, 0), next = __shfl(jump, from);
        const uint32_t l = (uint32_t) __shfl((int) lo, from), h = (uint32_t) __shfl((int) hi, from);
        if (jump >= 0) {
            lo |= l;
            hi |= h;
            jump = next;
        }
    }
    return (uint64_t) hi << 32 | lo;
}
// Four bits of it from drafted slot `off` on (negative: still in the cache).
__device__ __forceinline__ uint32_t tree_seen4(uint64_t path, int64_t off) {
    if (off >= 64) return 0u;
    if (off >= 0) return (uint32_t) (path >> off);
    return off <= -4 ? 15u : (uint32_t) path << -off | ((1u << -off) - 1);
}

__device__ __forceinline__ bool not_finite_bf16(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }

// The offset that a row's exponents are taken from: its first maximum, raised
// only when a tile's passes it by more than 2^8, so that the sums are seldom
// rescaled (16 rows of a wave see some new maximum in half of all tiles).  A
// weight is then at most 2^8, as exact in bf16 as one below 1.  A tile whose
// scores are all NaN leaves it (the sum is NaN then), so it is never NaN itself.
__device__ __forceinline__ float tree_offset(float m, float top) { return top > m + 8.0f ? top : m; }

// Eight values of Q with the scale's sign.
__device__ __forceinline__ bf16x8_t tree_q(const TreeParams & p, const uint16_t * q) {
    union {
        bf16x8_t v;
        uint32_t w[4];
    } u;
    u.v = *(const bf16x8_t *) q;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.w[i] = (u.w[i] & p.q_and) ^ p.q_xor;
    return u.v;
}

// 2^(scale q.k - m) of one row and slot, element by element: the weight of an
// Inf or NaN value, which reaches its row whatever the weight's last bits.
__device__ float tree_weight(const TreeParams & p, int64_t b, int64_t head, int64_t tok,
                                                       const uint16_t * k, int dh, float m) {
    const uint16_t * q = p.q + ((b * p.heads + head) * p.tq + tok) * dh;
    float s = 0.0f;
    for (int i = 0; i < dh; ++i)
        s = fmaf(bf16_to_f32((uint16_t) ((q[i] & p.q_and) ^ p.q_xor)), bf16_to_f32(k[i]), s);
    return __builtin_amdgcn_exp2f(s * p.scale - m);
}

// Which of 32 slots a token sees, the first being drafted slot `off` (negative:
// still in the cache, where every slot is seen).
__device__ __forceinline__ uint32_t tree_seen(const uint32_t * path, int64_t off, int tq) {
    if (off <= -32) return 0xffffffffu;
    const int o = off < tq ? (int) off : kTreeMax, words = (tq + 31) / 32, w = o >> 5, sh = o & 31;
    const uint32_t lo = w < 0 ? 0xffffffffu : w < words ? path[w] : 0u, hi = w + 1 < words ? path[w + 1] : 0u;
    return sh ? lo >> sh | hi << (32 - sh) : lo;
}

// Eight values of V^T from `slot` on in a tile that reaches past `past`: slots
// behind the last hold anything and become zero, and so do Inf and NaN of a
// drafted slot, which must not reach the rows that do not see it (true: there
// is one, added to the rows that do by itself).
__device__ __forceinline__ bool tree_mask_values(uint32_t * w, int64_t slot, int64_t past, int64_t n) {
    const int held = (int) max((int64_t) 0, min((int64_t) 8, n - slot));
    bool any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[j] &= held > 2 * j + 1 ? 0xffffffffu : held == 2 * j + 1 ? 0x0000ffffu : 0u;
        any |= not_finite_bf16(w[j]) || not_finite_bf16(w[j] >> 16);
    }
    if (!any || slot + 8 <= past) return false;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (slot + j >= past && not_finite_bf16(w[j >> 1] >> (16 * (j & 1)))) {
            bad = true;
            w[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
        }
    return bad;
}

// The units of the slots: sequence b gets 1 + (units - batch) tiles_b / tiles of
// them (its share by length, but kTreeLeast tiles a unit at least), one after another;
// units / batch each where the sequences are more than a wave's lanes (or the
// product would pass 32 bits).  Unit u's sequence, the first of that sequence's
// units and their number; no sequence (-1) past the last unit.
constexpr int kTreeTile = 64, kTreeLeast = 2;
struct TreeUnit {
    int b, first, count, slots;
};
__device__ __forceinline__ int64_t tree_slots(const TreeParams & p, int b) {
    // A length that does not fit leaves its sequence without slots.
    const int64_t past = p.past ? p.past[b] : 0;
    return past >= 0 && past + p.tq <= p.capacity ? past + p.tq : 0;
}
__device__ __forceinline__ TreeUnit tree_unit(const TreeParams & p, int u, int b_known = -1) {
    if (p.even) {
        const int each = (int) ((uint32_t) p.units / (uint32_t) p.batch);
        const int b = b_known >= 0 ? b_known : (int) ((uint32_t) u / (uint32_t) each);
        return {b < p.batch ? b : -1, b * each, each, b < p.batch ? (int) tree_slots(p, b) : 0};
    }
    const int lane = threadIdx.x & 63;
    const int slots = lane < p.batch ? (int) tree_slots(p, lane) : 0;
    const uint32_t tiles = ((uint32_t) slots + kTreeTile - 1) / kTreeTile;
    uint32_t sum = tiles;
    for (int o = 1; o < p.batch; o <<= 1) sum += (uint32_t) __shfl_xor((int) sum, o);
    // Past the batch's power of two the lanes hold nothing, and take nothing.
    int mine = 0;
    if (lane < p.batch) {
        mine = 1 + (sum ? (int) ((uint32_t) (p.units - p.batch) * tiles / sum) : 0);
        mine = min(mine, max(1, (int) (tiles / kTreeLeast)));
    }
    int end = mine;  // inclusive prefix
    for (int o = 1; o < p.batch; o <<= 1) {
        const int v = __shfl_up(end, o);
        if (lane >= o) end += v;
    }
    int b = b_known;
    if (b < 0) {
        const unsigned long long past_u = __ballot(lane < p.batch && end > u);
        if (!past_u) return {-1, 0, 0, 0};
        b = __ffsll(past_u) - 1;
    }
    const int count = __shfl(mine, b);
    return {b, __shfl(end, b) - count, count, __shfl(slots, b)};
}
// The tiles [t0, t1) of part i out of `count`.
__device__ __forceinline__ void tree_range(int64_t n, int i, int count, int64_t & t0, int64_t & t1) {
    const uint32_t tiles = (uint32_t) ((n + kTreeTile - 1) / kTreeTile);
    const uint32_t q = tiles / (uint32_t) count, r = tiles - q * (uint32_t) count;
    t0 = q * (uint32_t) i + min((uint32_t) i, r);
    t1 = t0 + q + ((uint32_t) i < r);
}

// All rows, up to NR tiles of 16, for a workgroup; slots in tiles of 64: wave w takes slots
// 16w .. of a tile for the scores of all rows, and DH / 4 of the result's
// dimensions for all rows and slots, so every K and V element is loaded once,
// by one wave, into the registers that feed its matrix operand.  The rows (Q)
// and the probabilities lie in LDS.  K of the next tile is requested when this
// tile's scores are done and V when its product is.  The slots' bytes bound it:
// one token of 2 x 16 heads of 64 (4 key heads) over 100000 slots 36 to 39 us
// with the join, 4.6 to 4.9 TB/s.
//
// The probabilities are rounded to bf16, the only operand type that V's matrix
// instruction takes beside it, here and in tree_attn_many; their sum is of the
// unrounded ones, in f32, as are maxima and results.  Each is off by at most 2^-8
// of itself, independently, so a result by at most 2^-8 sum p |v| / sum p and
// typically by 1.5e-3 of itself, as much as the rounding of the result to bf16
// alone (against 64 bits: 2.3e-3 together, 1.7e-3 with exact probabilities).  A
// second operand with the rounded-off parts would double the products of V.
template <int DH, int NR>
__global__ __launch_bounds__(kTreeWaves * 64, 2) void tree_attn_rows(TreeParams p) {
    constexpr int KC = DH / 32, DT = DH / 64, TILE = 64, R = NR * 16, QCH = DH / 8;
    __shared__ __align__(16) uint16_t qs[R * DH];
    __shared__ __align__(16) uint16_t ps[R * TILE];
    __shared__ float sm[kTreeWaves][R];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const int group = p.heads / p.kv_heads, rows = group * p.tq;
    const int hk = (int) (blockIdx.x / (uint32_t) p.units), u = (int) blockIdx.x - hk * p.units;
    if (hk >= p.kv_heads) return;
    const TreeUnit unit = tree_unit(p, u);
    if (unit.b < 0) return;
    const int b = unit.b;
    const int64_t n = unit.slots, past = n ? n - p.tq : 0;
    int64_t t0, t1;
    tree_range(n, u - unit.first, unit.count, t0, t1);
    const int64_t bz = (int64_t) b * p.kv_heads + hk;
    const int32_t * parents = p.parents + (int64_t) b * p.tq;
    const int parent = lane < p.tq ? parents[lane] : -1;

    const uint16_t * kb = p.k + bz * p.capacity * DH + g * 8;
    const uint16_t * vb = p.vt + (bz * DH + wave * (DH / 4) + c16) * p.vt_ld;
    bf16x8_t kf[KC], vf[2][DT];
    auto load_k = [&](int64_t kt) {
        const int64_t slot = min(kt * TILE + wave * 16 + c16, n - 1);
#pragma unroll
        for (int c = 0; c < KC; ++c) kf[c] = *(const bf16x8_t *) (kb + slot * DH + c * 32);
    };
    auto load_v = [&](int64_t kt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t v0 = min(kt * TILE + h * 32 + g * 8, p.vt_ld - 8);
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[h][d] = *(const bf16x8_t *) (vb + (int64_t) d * 16 * p.vt_ld + v0);
        }
    };
    if (t0 < t1) {
        load_k(t0);
        load_v(t0);
    }

    // Q into LDS: 16-byte chunk c of row r at c ^ (r's swizzle), so that the 16
    // rows of an operand read lie in different banks.
    auto qswz = [](int r) { return DH == 64 ? (r >> 1) & 7 : r & 15; };
    for (int e = threadIdx.x; e < R * QCH; e += kTreeWaves * 64) {
        const int r = e / QCH, c = e % QCH, row = min(r, rows - 1);
        const uint16_t * qr = p.q + (((int64_t) b * p.heads + hk * group + row / p.tq) * p.tq + row % p.tq) * DH;
        *(bf16x8_t *) (qs + r * DH + (c ^ qswz(r)) * 8) = tree_q(p, qr + c * 8);
    }
    int tok[NR];
    bool token[NR];  // a place that holds a token
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        tok[i] = min(i * 16 + c16, rows - 1) % p.tq;
        const int pr = parents[tok[i]];
        token[i] = pr >= -1 && pr < p.tq;
    }
    uint64_t path[NR] = {};
    if (t0 < t1 && t1 * TILE > past) {
        const uint64_t mine = tree_path(parent, p.tq);
#pragma unroll
        for (int i = 0; i < NR; ++i)
            path[i] = (uint64_t) (uint32_t) __shfl((int) (mine >> 32), tok[i]) << 32 | (uint32_t) __shfl((int) mine, tok[i]);
    }
    __syncthreads();

    float m[NR], l[NR];
    f32x4_t o[NR][DT];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[i][d] = (f32x4_t){0, 0, 0, 0};
    }
    bool bad = false;
    for (int64_t kt = t0; kt < t1; ++kt) {
        const int64_t base = kt * TILE;
        const bool edge = base + TILE > past;
        f32x4_t s[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) s[i] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int r = i * 16 + c16;
                const bf16x8_t q = *(const bf16x8_t *) (qs + r * DH + ((c * 4 + g) ^ qswz(r)) * 8);
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[c], q, s[i], 0, 0, 0);
            }
        if (kt + 1 < t1) load_k(kt + 1);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (edge) {
                const uint32_t seen = tree_seen4(path[i], base + wave * 16 + 4 * g - past);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][r] = seen >> r & 1 ? s[i][r] : -INFINITY;
            }
            float top = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
            top = max_xor32(max_xor16(top)) * p.scale;
            if (g == 0) sm[wave][i * 16 + c16] = top;
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = i * 16 + c16;
            const float mn = tree_offset(m[i], fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r])));
            const float bm = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m[i] - bm);
            float pr[4], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pr[e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], p.scale, -bm));
                sum += pr[e];
            }
            l[i] = l[i] * alpha + sum;
            if (__any(mn != m[i])) {
#pragma unroll
                for (int d = 0; d < DT; ++d) o[i][d] *= alpha;
            }
            m[i] = mn;
            uint2 w;
            w.x = pack_bf16x2(pr[0], pr[1]);
            w.y = pack_bf16x2(pr[2], pr[3]);
            *(uint2 *) (ps + r * TILE + ((2 * wave + (g >> 1)) ^ ((r >> 1) & 7)) * 8 + (g & 1) * 4) = w;
        }
        lds_barrier();
        if (edge) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    union {
                        bf16x8_t v;
                        uint32_t w[4];
                    } u;
                    u.v = vf[h][d];
                    bad |= tree_mask_values(u.w, base + h * 32 + g * 8, past, n);
                    vf[h][d] = u.v;
                }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int r = i * 16 + c16;
                const bf16x8_t pf = *(const bf16x8_t *) (ps + r * TILE + ((4 * h + g) ^ ((r >> 1) & 7)) * 8);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[h][d], pf, o[i][d], 0, 0, 0);
            }
        if (kt + 1 < t1) load_v(kt + 1);
    }
    if (__any(bad)) {
        // Inf or NaN among the drafted values: added element by element to the
        // rows whose path holds the slot.
        for (int64_t slot = max(t0 * TILE, past); slot < min(t1 * TILE, n); ++slot) {
            const int a = (int) (slot - past);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                if (!(path[i] >> a & 1)) continue;
                const int row = min(i * 16 + c16, rows - 1);
                const float pr =
                    tree_weight(p, b, hk * group + row / p.tq, tok[i], kb - g * 8 + slot * DH, DH, m[i]);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t v = vb[(int64_t) (d * 16 + 4 * g + e - c16) * p.vt_ld + slot];
                        if (not_finite_bf16(v)) o[i][d][e] += pr * bf16_to_f32(v);
                    }
            }
        }
    }

    // The rows' sums over the lanes and waves that hold their parts.
    lds_barrier();
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const float t = sum_xor32(sum_xor16(l[i]));
        if (g == 0) sm[wave][i * 16 + c16] = t;
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int row = i * 16 + c16;
        const float sum = (sm[0][row] + sm[1][row]) + (sm[2][row] + sm[3][row]);
        if (row >= rows) continue;
        // Scores that are all -Inf leave 0 / 0, which is NaN.
        const bool none = !token[i] || n == 0;
        const int d0 = wave * (DH / 4) + 4 * g;
        if (p.po) {
            const int64_t at = ((int64_t) u * p.kv_heads + hk) * rows + row;
#pragma unroll
            for (int d = 0; d < DT; ++d) *(f32x4_t *) (p.po + at * DH + d0 + d * 16) = o[i][d];
            if (wave == 0 && g == 0) {
                p.pml[2 * at] = m[i];
                p.pml[2 * at + 1] = sum;
            }
        } else {
            const float inv = none ? 0.0f : 1.0f / sum;
            uint16_t * y = p.out + (((int64_t) b * p.tq + tok[i]) * p.heads + hk * group + row / p.tq) * DH + d0;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                *(uint32_t *) (y + d * 16) = none ? 0u : pack_bf16x2(o[i][d][0] * inv, o[i][d][1] * inv);
                *(uint32_t *) (y + d * 16 + 2) = none ? 0u : pack_bf16x2(o[i][d][2] * inv, o[i][d][3] * inv);
            }
        }
    }
}

// Many rows: W waves of NR tiles of 16 rows each, every wave over all slots of
// a tile, so a row's maximum, sum and probabilities stay in its wave.  S^T =
// K Q^T puts a query in a lane's column, and with the slots of two 16-row tiles
// interleaved (row a of tile u is slot 8 (a / 4) + 4 (u % 2) + a % 4 of its
// half) eight consecutive slots in its registers: the operand of O^T = V^T P^T
// as it stands.  K and V^T tiles of 64 slots go through registers into one of
// two LDS buffers while the other is used; one barrier a tile.  A tile of 128
// dimensions takes 5 k cycles, of which MFMA fill 34%, other vector instructions
// 32% and LDS 21%: 64 tokens of 4 x 32 heads (8 key heads) over 16000 slots 87 us
// with the join, 0.63 PFLOP/s (102 call after call, where the clock sinks).  Two row tiles a wave in eight waves; four in four
// waves of 512 registers 106 us, two in four 99.  What is not to be seen of V is
// taken out once, on its way to LDS (100 tokens of 2 x 8 heads of 256 over 4000
// slots 34 us, by every wave that reads it 43).
template <int DH, int NR, int W>
__global__ __launch_bounds__(W * 64, 1) void tree_attn_many(TreeParams p) {
    constexpr int KC = DH / 32, DT = DH / 16, TILE = 64, R = W * NR * 16, QCH = DH / 8;
    constexpr int KN = TILE * QCH / (W * 64), VN = DH * 8 / (W * 64);  // 16-byte pieces of a thread
    __shared__ __align__(16) uint16_t kt_lds[2][TILE * DH];
    __shared__ __align__(16) uint16_t vt_lds[2][DH * TILE];
    __shared__ TreePaths path;
    __shared__ int bad;  // Inf or NaN among the drafted values
    static_assert(sizeof(TreeWork) <= sizeof vt_lds, "the paths' scratch lies in the value tiles");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const int group = p.heads / p.kv_heads, rows = group * p.tq;
    // Row tiles of one unit are eight workgroups apart: the same XCD, whose L2
    // then holds the slots they share.
    const int rt = (rows + R - 1) / R;
    const uint32_t id = blockIdx.x, at8 = id / (uint32_t) (8 * rt) * 8 + id % 8;
    const int row0 = (int) (id / 8 % (uint32_t) rt) * R + wave * NR * 16;
    const int hk = (int) (at8 / (uint32_t) p.units), u = (int) at8 - hk * p.units;
    if (hk >= p.kv_heads) return;
    const TreeUnit unit = tree_unit(p, u);
    if (unit.b < 0) return;
    const int b = unit.b;
    const int64_t n = unit.slots, past = n ? n - p.tq : 0;
    int64_t t0, t1;
    tree_range(n, u - unit.first, unit.count, t0, t1);
    const int64_t bz = (int64_t) b * p.kv_heads + hk;
    const int32_t * parents = p.parents + (int64_t) b * p.tq;
    const int parent = (int) threadIdx.x < p.tq ? parents[threadIdx.x] : -1;
    const uint16_t * kb = p.k + bz * p.capacity * DH;
    const uint16_t * vb = p.vt + bz * DH * p.vt_ld;

    // 16 rows of an operand read fall into different banks: chunk c of K slot
    // k at c ^ kswz(k) (the 16 slots of a tile differ in bits 0, 1, 3 and 4),
    // of V^T row d at c ^ (d / 2) % 8.
    auto kswz = [](int k) {
        return DH == 64 ? ((k >> 1) & 1) | ((k >> 3) & 3) << 1 : (k & 3) | ((k >> 3) & 3) << 2;
    };
    // K of the next tile is requested before this tile's scores and deposited
    // after them, V then, behind the softmax and the products.
    static_assert(KN == VN, "one set of registers for both");
    bf16x8_t sr[KN];
    auto request_k = [&](int64_t kt) {
#pragma unroll
        for (int j = 0; j < KN; ++j) {
            const int e = threadIdx.x + j * W * 64;
            sr[j] = *(const bf16x8_t *) (kb + min(kt * TILE + e / QCH, n - 1) * DH + e % QCH * 8);
        }
    };
    auto request_v = [&](int64_t kt, bf16x8_t * sr) {
#pragma unroll
        for (int j = 0; j < VN; ++j) {
            const int e = threadIdx.x + j * W * 64;
            sr[j] = *(const bf16x8_t *) (vb + (int64_t) (e >> 3) * p.vt_ld + min(kt * TILE + (e & 7) * 8, p.vt_ld - 8));
        }
    };
    auto deposit_k = [&](int buf) {
#pragma unroll
        for (int j = 0; j < KN; ++j) {
            const int e = threadIdx.x + j * W * 64, k = e / QCH;
            *(bf16x8_t *) (kt_lds[buf] + k * DH + ((e % QCH) ^ kswz(k)) * 8) = sr[j];
        }
    };
    // A tile that reaches past the cache is looked over on its way.
    auto deposit_v = [&](int64_t kt, int buf, const bf16x8_t * sr) {
        const bool edge = (kt + 1) * TILE > past;
#pragma unroll
        for (int j = 0; j < VN; ++j) {
            const int e = threadIdx.x + j * W * 64, d = e >> 3;
            union {
                bf16x8_t v;
                uint32_t w[4];
            } u;
            u.v = sr[j];
            if (edge && tree_mask_values(u.w, kt * TILE + (e & 7) * 8, past, n)) bad = 1;
            *(bf16x8_t *) (vt_lds[buf] + d * TILE + ((e & 7) ^ ((d >> 1) & 7)) * 8) = u.v;
        }
    };
    bf16x8_t first_v[VN];
    if (t0 < t1) {
        request_k(t0);
        request_v(t0, first_v);
    }
    if (threadIdx.x == 0) bad = 0;
    int tok[NR];
    bf16x8_t qf[NR][KC];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int row = min(row0 + i * 16 + c16, rows - 1);
        tok[i] = row % p.tq;
        const uint16_t * qr = p.q + (((int64_t) b * p.heads + hk * group + row / p.tq) * p.tq + tok[i]) * DH;
#pragma unroll
        for (int c = 0; c < KC; ++c) qf[i][c] = tree_q(p, qr + c * 32 + g * 8);
    }
    if (t0 < t1 && t1 * TILE > past) {
        if (p.tq > 64) {
            tree_paths(path, vt_lds, parent, p.tq);
        } else if (wave == 0) {
            const uint64_t mine = tree_path(parent, p.tq);
            path[lane][0] = (uint32_t) mine;
            path[lane][1] = (uint32_t) (mine >> 32);
        }
    }
    __syncthreads();
    if (t0 < t1) {
        deposit_k(0);
        deposit_v(t0, 0, first_v);
    }
    __syncthreads();

    float m[NR], l[NR];
    f32x4_t o[NR][DT];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[i][d] = (f32x4_t){0, 0, 0, 0};
    }
    // EDGE: a tile that reaches past the cache, where every slot is looked at.
    auto tile = [&](int64_t kt, auto edge_tag) __attribute__((always_inline)) {
        constexpr bool edge = decltype(edge_tag)::value;
        const int buf = (int) (kt - t0) & 1;
        const int64_t base = kt * TILE;
        if (kt + 1 < t1) request_k(kt + 1);
        f32x4_t s[NR][4];
        if (row0 < rows) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = (u >> 1) * 32 + 8 * (c16 >> 2) + 4 * (u & 1) + (c16 & 3);
#pragma unroll
                for (int i = 0; i < NR; ++i) s[i][u] = (f32x4_t){0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const bf16x8_t kf = *(const bf16x8_t *) (kt_lds[buf] + k * DH + ((c * 4 + g) ^ kswz(k)) * 8);
#pragma unroll
                    for (int i = 0; i < NR; ++i)
                        s[i][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[i][c], s[i][u], 0, 0, 0);
                }
            }
        }
        if (kt + 1 < t1) {
            deposit_k(buf ^ 1);
            request_v(kt + 1, sr);
        }
        if (row0 < rows) {
            bf16x8_t pf[NR][2];
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                if (edge) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t seen = tree_seen(path[tok[i]], base + h * 32 + 8 * g - past, p.tq);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            s[i][2 * h + e / 4][e % 4] = seen >> e & 1 ? s[i][2 * h + e / 4][e % 4] : -INFINITY;
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][u][r]);
                top = max_xor32(max_xor16(top)) * p.scale;
                const float mn = tree_offset(m[i], top);
                const float bm = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[i] - bm);
                float sum = 0.0f;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[i][u][r] = __builtin_amdgcn_exp2f(fmaf(s[i][u][r], p.scale, -bm));
                        sum += s[i][u][r];
                    }
                l[i] = l[i] * alpha + sum;
                if (__any(mn != m[i])) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[i][d] *= alpha;
                }
                m[i] = mn;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
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
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int dr = d * 16 + c16;
                    const bf16x8_t vf = *(const bf16x8_t *) (vt_lds[buf] + dr * TILE + ((4 * h + g) ^ ((dr >> 1) & 7)) * 8);
#pragma unroll
                    for (int i = 0; i < NR; ++i)
                        o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[i][h], o[i][d], 0, 0, 0);
                }
        }
        if (kt + 1 < t1) deposit_v(kt + 1, buf ^ 1, sr);
        lds_barrier();
    };
    const int64_t inner = max(t0, min(t1, past / TILE));
    for (int64_t kt = t0; kt < inner; ++kt) tile(kt, std::false_type{});
    for (int64_t kt = inner; kt < t1; ++kt) tile(kt, std::true_type{});
    if (bad) {
        // Inf or NaN among the drafted values: added element by element to the
        // rows whose path holds the slot.
        for (int64_t slot = max(t0 * TILE, past); slot < min(t1 * TILE, n); ++slot) {
            const int a = (int) (slot - past);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                if (!(path[tok[i]][a >> 5] >> (a & 31) & 1)) continue;
                const int row = min(row0 + i * 16 + c16, rows - 1);
                const float pr = tree_weight(p, b, hk * group + row / p.tq, tok[i], kb + slot * DH, DH, m[i]);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t v = vb[(int64_t) (d * 16 + 4 * g + e) * p.vt_ld + slot];
                        if (not_finite_bf16(v)) o[i][d][e] += pr * bf16_to_f32(v);
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int row = row0 + i * 16 + c16;
        const float sum = sum_xor32(sum_xor16(l[i]));
        if (row >= rows) continue;
        const int pr = parents[tok[i]];
        const bool none = !(pr >= -1 && pr < p.tq) || n == 0;
        if (p.po) {
            const int64_t at = ((int64_t) u * p.kv_heads + hk) * rows + row;
#pragma unroll
            for (int d = 0; d < DT; ++d) *(f32x4_t *) (p.po + at * DH + d * 16 + 4 * g) = o[i][d];
            if (g == 0) {
                p.pml[2 * at] = m[i];
                p.pml[2 * at + 1] = sum;
            }
        } else {
            const float inv = none ? 0.0f : 1.0f / sum;
            uint16_t * y = p.out + (((int64_t) b * p.tq + tok[i]) * p.heads + hk * group + row / p.tq) * DH + 4 * g;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                *(uint32_t *) (y + d * 16) = none ? 0u : pack_bf16x2(o[i][d][0] * inv, o[i][d][1] * inv);
                *(uint32_t *) (y + d * 16 + 2) = none ? 0u : pack_bf16x2(o[i][d][2] * inv, o[i][d][3] * inv);
            }
        }
    }
}

// out = sum_s po_s 2^(m_s - m) / sum_s l_s 2^(m_s - m) over a row's units, DH / 4
// threads with four values each.  BY_ROWS: 1024 / DH rows of one (sequence, key
// head) to a workgroup, each thread over all units;
// else one row, its units shared out among as many groups of threads, whose
// results are added in order.
template <int DH, bool BY_ROWS>
__global__ __launch_bounds__(256) void tree_attn_join(TreeParams p, int row_parts) {
    constexpr int PC = DH / 4, GR = 256 / PC, AT_ONCE = 8;
    __shared__ __align__(16) f32x4_t acc[GR][PC];
    __shared__ float parts[GR][2];
    const int piece = threadIdx.x % PC, gr = threadIdx.x / PC;
    const int group = p.heads / p.kv_heads, rows = group * p.tq;
    const uint32_t bz = blockIdx.x / (uint32_t) row_parts;
    const int first = (int) (blockIdx.x - bz * (uint32_t) row_parts) * (BY_ROWS ? GR : 1);
    const int row = min(first + (BY_ROWS ? gr : 0), rows - 1);
    const int64_t b = bz / (uint32_t) p.kv_heads;
    const int hk = (int) (bz - (uint32_t) b * (uint32_t) p.kv_heads);
    const TreeUnit unit = tree_unit(p, 0, (int) b);
    const int parent = p.parents[b * p.tq + row % p.tq];
    const int64_t step = (int64_t) p.kv_heads * rows, at = unit.first * step + hk * rows + row;
    float m = -INFINITY, sum = 0.0f;
    f32x4_t v = {0, 0, 0, 0};
    constexpr int BY = BY_ROWS ? 1 : GR;
    for (int s0 = BY_ROWS ? 0 : gr; s0 < unit.count; s0 += AT_ONCE * BY) {
        float ms[AT_ONCE], ls[AT_ONCE];
        f32x4_t o[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int64_t j = at + min(s0 + k * BY, unit.count - 1) * step;
            const float2 ml = *(const float2 *) (p.pml + 2 * j);
            ms[k] = s0 + k * BY < unit.count ? ml.x : -INFINITY;
            ls[k] = ml.y;
            o[k] = *(const f32x4_t *) (p.po + j * DH + piece * 4);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) top = fmaxf(top, ms[k]);
        const float bm = top == -INFINITY ? 0.0f : top, old = __builtin_amdgcn_exp2f(m - bm);
        sum *= old;
        v *= old;
        m = top;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            // A unit without a finite score has weight zero: 0 times its results,
            // which hold NaN where 0 met an Inf or NaN value.
            if (s0 + k * BY >= unit.count) continue;
            const float f = __builtin_amdgcn_exp2f(ms[k] - bm);
            sum += ls[k] * f;
            v += o[k] * f;
        }
    }
    if constexpr (!BY_ROWS) {
        acc[gr][piece] = v;
        if (piece == 0) {
            parts[gr][0] = m;
            parts[gr][1] = sum;
        }
        __syncthreads();
        if (gr) return;
        float top = m;
#pragma unroll
        for (int k = 1; k < GR; ++k) top = fmaxf(top, parts[k][0]);
        const float bm = top == -INFINITY ? 0.0f : top;
        const float old = __builtin_amdgcn_exp2f(m - bm);
        v *= old;
        sum *= old;
#pragma unroll
        for (int k = 1; k < GR; ++k) {
            const float f = __builtin_amdgcn_exp2f(parts[k][0] - bm);
            v += acc[k][piece] * f;
            sum += parts[k][1] * f;
        }
        m = top;
    } else if (first + gr >= rows) {
        return;
    }
    const bool none = !(parent >= -1 && parent < p.tq) || unit.slots == 0;
    const float inv = none ? 0.0f : 1.0f / sum;
    uint16_t * y = p.out + ((b * p.tq + row % p.tq) * p.heads + hk * group + row / p.tq) * DH + piece * 4;
    *(uint32_t *) y = none ? 0u : pack_bf16x2(v[0] * inv, v[1] * inv);
    *(uint32_t *) (y + 2) = none ? 0u : pack_bf16x2(v[2] * inv, v[3] * inv);
}

// Units: `wgs` workgroups in all where each has kTreeLeast tiles or more (two:
// 64 tokens of 4 x 8 heads over 1000 slots 26 us, four tiles 30, one 32; a
// draft of 8 over 128 slots not split 7.5 us, split 9.7), as far as the
// workspace holds their results.
static void plan(TreeParams & p, const TreeArgs & a, int64_t row_tiles, int64_t wgs) {
    const int64_t rows = a.heads / a.kv_heads * a.tq, tiles = (a.capacity + kTreeTile - 1) / kTreeTile;
    int64_t units = std::min<int64_t>(wgs / (a.kv_heads * row_tiles), a.batch * std::max<int64_t>(tiles / kTreeLeast, 1));
    const size_t per = (size_t) (a.kv_heads * rows) * (size_t) (a.head_dim + 2) * 4;
    units = std::min<int64_t>(units, (int64_t) (a.ws_bytes / per));
    p.even = a.batch > 64 || (uint64_t) units * (uint64_t) tiles * (uint64_t) a.batch > 0xffffffffull;
    if (p.even) units = units / a.batch * a.batch;
    p.units = (int32_t) std::max<int64_t>(units, a.batch);
    if (p.units > a.batch) {
        p.po = (float *) a.ws;
        p.pml = p.po + (int64_t) p.units * a.kv_heads * rows * a.head_dim;
    }
}

template <int DH>
static hipError_t launch(void (*kernel)(TreeParams), int R, int threads, int64_t target, TreeParams & p,
                         const TreeArgs & a, hipStream_t s) {
    const int64_t rows = a.heads / a.kv_heads * a.tq, rt = (rows + R - 1) / R;
    plan(p, a, rt, target);
    const int64_t wgs = ((int64_t) p.units * a.kv_heads + 7) / 8 * 8 * rt, joins = a.batch * a.kv_heads * rows;
    if (wgs > 0x7fffffff || joins > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kernel, dim3((unsigned) wgs), dim3((unsigned) threads), 0, s, p);
    if (p.po) {
        // Many rows fill the GPU by workgroups of rows (64 tokens of 4 x 32 heads
        // 85 us in all, a workgroup per row 101; 4 tokens of 16 x 32 heads 21,
        // 25), few by workgroups of one (33 tokens of 3 x 8: 34 us, by rows 35).
        if (joins > 1024) {
            const int parts = (int) ((rows + 1024 / DH - 1) / (1024 / DH));
            hipLaunchKernelGGL((tree_attn_join<DH, true>), dim3((unsigned) (a.batch * a.kv_heads * parts)), dim3(256), 0, s,
                               p, parts);
        } else {
            hipLaunchKernelGGL((tree_attn_join<DH, false>), dim3((unsigned) joins), dim3(256), 0, s, p, (int) rows);
        }
    }
    return hipGetLastError();
}

// Workgroups that keep enough of the slots requested, 256, 512 and 768 of them
// measured: narrow heads request little each (us, one token of 4 x 4 heads of 64
// over 100000 slots: 111, 66, 64; of 2 x 16 / 4 heads: 58, 38, 36), wider ones do
// with 512 (8 tokens of 4 x 8 heads of 128 over 8000: 32, 28, 29; 8 tokens of 16 /
// 8 heads of 256 over 20000: 41, 41, 42).  33 to 48 rows of 256 have results so
// large, 48 KB a unit, that twice the units cost more in the join than they
// bring (40 tokens of 8 heads over 16000: 39, 41, 53; 2 x 12 tokens of 16 / 4
// heads over 12000: 33, 37, 44; 3 x 33 of 8 over 5000: 36, 38, 49).
template <int DH, int NR>
static hipError_t run_rows(TreeParams & p, const TreeArgs & a, hipStream_t s) {
    constexpr int kWorkgroups = DH == 64 ? 768 : DH == 256 && NR > 2 ? 256 : 512;
    return launch<DH>(tree_attn_rows<DH, NR>, NR * 16, kTreeWaves * 64, kWorkgroups, p, a, s);
}
template <int DH, int NR, int W>
static hipError_t run_many(TreeParams & p, const TreeArgs & a, hipStream_t s) {
    return launch<DH>(tree_attn_many<DH, NR, W>, W * NR * 16, W * 64, 256, p, a, s);
}

hipError_t launch_tree_attn(const TreeArgs & a, hipStream_t s) {
    if (a.tq <= 0 || a.batch <= 0) return hipSuccess;
    // Wide reads of q, k and V^T, and result stores of two values.
    if (((uintptr_t) a.q | (uintptr_t) a.k | (uintptr_t) a.vt) % 16 != 0 || (uintptr_t) a.out % 4 != 0)
        return hipErrorInvalidValue;
    if (a.tq > kTreeMax || a.heads <= 0 || a.kv_heads <= 0 || a.heads % a.kv_heads != 0 ||
        a.batch > 0x7fffffff / a.kv_heads || a.vt_ld % 8 != 0 || a.vt_ld < a.capacity || a.capacity <= 0 || a.capacity > 0x7fffffff)
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
    p.batch = (int32_t) a.batch;
    // The kernels take a positive scale: a negative one turns Q's signs, zero
    // makes Q zero.
    p.scale = a.scale == 0.0f ? 1.0f : std::fabs(a.scale) * 1.4426950408889634f;
    p.q_and = a.scale == 0.0f ? 0u : 0xffffffffu;
    p.q_xor = a.scale < 0.0f ? 0x80008000u : 0u;
    const int64_t rows = a.heads / a.kv_heads * a.tq;
    switch (a.head_dim) {
        case 64:
            if (rows <= 16) return run_rows<64, 1>(p, a, s);
            if (rows <= 32) return run_rows<64, 2>(p, a, s);
            if (rows <= 48) return run_rows<64, 3>(p, a, s);
            return rows <= 64 ? run_rows<64, 4>(p, a, s) : run_many<64, 2, 8>(p, a, s);
        case 128:
            if (rows <= 16) return run_rows<128, 1>(p, a, s);
            if (rows <= 32) return run_rows<128, 2>(p, a, s);
            if (rows <= 48) return run_rows<128, 3>(p, a, s);
            return rows <= 64 ? run_rows<128, 4>(p, a, s) : run_many<128, 2, 8>(p, a, s);
        case 256:
            if (rows <= 16) return run_rows<256, 1>(p, a, s);
            if (rows <= 32) return run_rows<256, 2>(p, a, s);
            return rows <= 48 ? run_rows<256, 3>(p, a, s) : run_many<256, 1, 8>(p, a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace wamx
