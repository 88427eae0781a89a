// Group normalisation with an activation over channels-last tensors, forward and backward.
//
// A workgroup owns a TILE: some pixel rows of one sample, over a SLAB of channels that holds whole groups.  Its
// elements are read once into registers as 16-byte chunks of 8 channels (thread = one chunk column, every
// rows_per_pass-th row) and everything the tile needs is computed from there: the mean first, then the sum of
// (x - mean)^2, so no digits are lost to E[x^2] - mean^2.
//   one tile per (sample, slab): the workgroup normalises its registers and writes y; x is read once.
//   more than one: the tiles write (mean, M2) per group, a second kernel merges them (Chan's formula) and applies.
// The backward pass is built the same way over per-channel sums of g and g * xhat, which also give dgamma / dbeta.
// Bound by memory.  bf16: 256 x 32 x 32 x 128 with skip forward 46.6 us call to call over rotating buffers (201 MB, 4.3 TB/s; 35
// where the 256 MB cache still holds them); 256 x 64 x 64 x 64 forward 75-78 us (3.5 TB/s; 128 registers a thread, two
// workgroups a CU, which costs 48 to 68 bytes of scratch memory a lane) and backward 143-146 (2.8 TB/s: x and dy of one
// workgroup fill a CU's registers, so its loads, sums and stores take turns; workgroups that walk over samples and load ahead
// were slower, 232 against 217 us for both).
// In the tiled form every workgroup merges the partial sums of its whole sample, work that grows with the square of the
// tiles: one picture of 64 channels, forward / backward, takes 57 / 64 us at 512 x 512, 144 / 235 at 1024 x 1024 (704 tiles
// at 600 x 600), 902 / 1895 at 2048 x 2048, where the tensors need 206 / 310.
#include "rowops.h"

namespace {

struct GnArgs {
    const void *x, *res, *dy;
    void *y, *dx, *dres;
    float* stats;                    // [2][B][G]
    const float *gamma, *beta;
    float* part;                     // forward: [B][G][tiles][2]; backward: [B][tiles][2][C]
    int B, HW, C, G, act, tiles, rows_tile, nslab, nv, rpp, ent;
    int x_ld, res_ld, y_ld, dx_ld, dres_ld;
    float eps;
    int seg;                         // lanes that sum one group (a power of two)
    FastDiv cg, nvd, tiled, slabd;   // divisions by C / G, nv, tiles, nslab
};

constexpr int GN_MAX_GROUPS = 64;    // groups of a slab (slabs wider than 64 channels hold at most 8)

// What a thread knows about its place: chunk column, first row, channels.
struct Place {
    int b, tile, c0, chunk, ty, r0, r1, nv, nch, ngr, g0;
    bool live;
};
__device__ __forceinline__ Place gn_place(const GnArgs& a, uint32_t blk) {
    Place p;
    uint32_t slab;
    if (a.tiles == 1) {
        // Workgroups go round-robin over the 8 dies: the slabs of one sample are given to one die, one after the other,
        // because a slab may be narrower than the 128-byte lines they share.
        const uint32_t q = blk >> 3, whole = (uint32_t)(a.B & ~7) * a.nslab;
        p.tile = 0;
        if (blk < whole) {
            const uint32_t grp = fdiv(q, a.slabd);
            slab = q - grp * a.nslab;
            p.b = grp * 8 + (blk & 7);
        } else {
            const uint32_t rest = blk - whole, bb = fdiv(rest, a.slabd);
            slab = rest - bb * a.nslab;
            p.b = (a.B & ~7) + bb;
        }
    } else {
        const uint32_t bs = fdiv(blk, a.tiled);
        p.tile = blk - bs * a.tiles;
        p.b = fdiv(bs, a.slabd);
        slab = bs - p.b * a.nslab;
    }
    p.c0 = slab * a.nv * 8;
    p.nch = min(a.nv * 8, a.C - p.c0);
    p.nv = p.nch >> 3;
    p.ty = fdiv(threadIdx.x, a.nvd);
    p.chunk = threadIdx.x - p.ty * a.nv;
    p.live = p.ty < a.rpp && p.chunk < p.nv;
    p.r0 = p.tile * a.rows_tile;
    p.r1 = min(a.HW, p.r0 + a.rows_tile);
    p.g0 = fdiv(p.c0, a.cg);
    p.ngr = fdiv(p.nch, a.cg);
    return p;
}

// Partial column sums: N values per channel of the slab into sm[n][ent][nv * 8], one entry per wave where a wave's lanes
// share chunk columns evenly (a power of two up to 32 of them), otherwise one per row lane.  Up to 8 chunk columns the
// lanes split the eight channels among themselves while they add (4 + 2 + 1 shuffles, then one for each remaining
// halving) instead of carrying all eight through every step.
template <int N>
__device__ __forceinline__ void column_parts(const GnArgs& a, const Place& p, float (&v)[N][8], float* sm) {
    const int width = a.nv * 8, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool fold = (a.nv & (a.nv - 1)) == 0 && a.nv <= 32;
    if (fold && a.nv <= 8) {
        const bool h32 = lane & 32, h16 = lane & 16, h8 = lane & 8;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[n][j] = (h32 ? v[n][j + 4] : v[n][j]) + __shfl_xor(h32 ? v[n][j] : v[n][j + 4], 32, 64);
#pragma unroll
            for (int j = 0; j < 2; ++j) v[n][j] = (h16 ? v[n][j + 2] : v[n][j]) + __shfl_xor(h16 ? v[n][j] : v[n][j + 2], 16, 64);
            v[n][0] = (h8 ? v[n][1] : v[n][0]) + __shfl_xor(h8 ? v[n][0] : v[n][1], 8, 64);
        }
        for (int o = a.nv; o < 8; o <<= 1)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n][0] += __shfl_xor(v[n][0], o, 64);
        lds_barrier();               // the last readers of sm are done
        if ((lane & 7) < a.nv)
#pragma unroll
            for (int n = 0; n < N; ++n) sm[(n * a.ent + wave) * width + (lane & 7) * 8 + (h32 ? 4 : 0) + (h16 ? 2 : 0) + (h8 ? 1 : 0)] = v[n][0];
    } else {
        int e = p.ty;
        bool writes = p.ty < a.rpp;
        if (fold) {
            for (int o = a.nv; o < 64; o <<= 1)
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[n][j] += __shfl_xor(v[n][j], o, 64);
            e = wave;
            writes = lane < a.nv;
        }
        lds_barrier();
        if (writes)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *(f32x4*)&sm[(n * a.ent + e) * width + p.chunk * 8 + j] = f32x4{v[n][j], v[n][j + 1], v[n][j + 2], v[n][j + 3]};
    }
    lds_barrier();
}
// adds the entries: afterwards sm[n][0][c] holds the sum of channel c
template <int N>
__device__ __forceinline__ void column_totals(const GnArgs& a, float* sm) {
    const int width = a.nv * 8;
    for (int t = threadIdx.x; t < N * width; t += blockDim.x) {
        const int n = t >= width ? 1 : 0, c = t - n * width;
        float* q = sm + (size_t)n * a.ent * width + c;
        float s = 0.f;
#pragma unroll 8
        for (int i = 0; i < a.ent; ++i) s += q[i * width];
        q[0] = s;                    // only this thread touches column c
    }
    lds_barrier();
}

// sums[n][g] = sum over the channels of group g and the first `ent` entries of w[c] * sm[n][entry][c] (w = 1 where null),
// through f: a.seg lanes per group
template <int N, typename F>
__device__ __forceinline__ void group_sums(const GnArgs& a, const Place& p, const float* sm, const float* w, int ent, float (*sums)[GN_MAX_GROUPS], F f) {
    const int cg = a.cg.d, width = a.nv * 8, lane = threadIdx.x & 63, seg = a.seg, per = 64 / seg;
    const int n_items = ent * cg;
    for (int base = (threadIdx.x >> 6) * per; base < p.ngr; base += (blockDim.x >> 6) * per) {
        const int g = base + lane / seg;
        float s[N];
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] = 0.f;
        if (g < p.ngr)
            for (int i = lane & (seg - 1); i < n_items; i += seg) {
                const int e = fdiv(i, a.cg), c = g * cg + i - e * cg;
                const float k = w ? w[p.c0 + c] : 1.f;
#pragma unroll
                for (int n = 0; n < N; ++n) s[n] += k * sm[(n * a.ent + e) * width + c];
            }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            for (int o = seg >> 1; o > 0; o >>= 1) s[n] += __shfl_xor(s[n], o, 64);
            if (g < p.ngr && (lane & (seg - 1)) == 0) sums[n][g] = f(s[n]);
        }
    }
    lds_barrier();
}

// per-channel constants of a thread's chunk
__device__ __forceinline__ void chunk_groups(const GnArgs& a, const Place& p, int (&gi)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) gi[j] = p.live ? fdiv(p.chunk * 8 + j, a.cg) : 0;
}

// pre = x (gamma rstd) + (beta - mean gamma rstd) (+ res) in both passes, one fma: LeakyReLU takes the same sign twice.
// Folding the mean into the constant costs an error of u |mean| gamma rstd, what the rounding of the mean itself costs.
template <typename T, int ACT>
__device__ __forceinline__ void apply_row(float (&v)[8], const float (&sc)[8], const float (&sh)[8], const float* q) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = fmaf(v[j], sc[j], sh[j]);
        if (q) v[j] += q[j];
        v[j] = act_value<sizeof(T) == 4>(v[j], ACT);
    }
}

template <typename T, int ACT, int R, int MAXT, int WAVES>
__global__ void __launch_bounds__(MAXT, WAVES) gn_fwd_tile(const GnArgs a) {
    extern __shared__ float sm[];
    __shared__ float sums[2][GN_MAX_GROUPS];
    const Place p = gn_place(a, blockIdx.x);
    const size_t row0 = (size_t)p.b * a.HW + p.r0;
    const int rows = p.r1 - p.r0, c = p.c0 + (p.live ? p.chunk * 8 : 0);
    float ga[8], be[8];                              // (before the tile: what they wait for is short; part of them is spilled at 16 chunks)
    load8<float>(a.gamma + c, ga);
    load8<float>(a.beta + c, be);
    const T* xp = (const T*)a.x + row0 * a.x_ld + c;
    Raw8<T> xv[R];
#pragma unroll
    for (int i = 0; i < R; ++i) raw_load(xv[i], xp + (size_t)min(p.ty + i * a.rpp, rows - 1) * a.x_ld);
    int gi[8];
    chunk_groups(a, p, gi);
    const int mine = p.live ? rows : 0;              // rows this thread may count
    float acc[1][8], mean[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[0][j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (p.ty + i * a.rpp < mine) {
            float v[8];
            pin(xv[i]);
            raw_f32(xv[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[0][j] += v[j];
        }
    }
    column_parts<1>(a, p, acc, sm);
    const float inv_n = 1.f / ((float)rows * (float)a.cg.d);
    group_sums<1>(a, p, sm, nullptr, a.ent, sums, [&](float s) { return s * inv_n; });
#pragma unroll
    for (int j = 0; j < 8; ++j) { mean[j] = sums[0][gi[j]]; acc[0][j] = 0.f; }
    pin(mean);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (p.ty + i * a.rpp < mine) {
            float v[8];
            pin(xv[i]);
            raw_f32(xv[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) { const float d = v[j] - mean[j]; acc[0][j] += d * d; }
        }
    }
    column_parts<1>(a, p, acc, sm);
    // M2 of a tile, or 1 / std of the whole group
    group_sums<1>(a, p, sm, nullptr, a.ent, sums + 1, [&](float s) { return a.tiles > 1 ? s : 1.f / sqrtf(s * inv_n + a.eps); });
    if (a.tiles > 1) {
        for (int g = threadIdx.x; g < p.ngr; g += blockDim.x) {
            float* o = a.part + (((size_t)p.b * a.G + p.g0 + g) * a.tiles + p.tile) * 2;
            o[0] = sums[0][g];
            o[1] = sums[1][g];
        }
        return;
    }
    if (a.stats)
        for (int g = threadIdx.x; g < p.ngr; g += blockDim.x) {
            const size_t o = (size_t)p.b * a.G + p.g0 + g;
            a.stats[o] = sums[0][g];
            a.stats[(size_t)a.B * a.G + o] = sums[1][g];
        }
    float sc[8], sh[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        sc[j] = ga[j] * sums[1][gi[j]];
        sh[j] = fmaf(-mean[j], sc[j], be[j]);
    }
    const T* rp = (const T*)a.res + row0 * a.res_ld + c;
    T* yp = (T*)a.y + row0 * a.y_ld + c;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = p.ty + i * a.rpp;
        if (r < mine) {
            float v[8], q[8];
            if (a.res) load8<T>(rp + (size_t)r * a.res_ld, q);
            pin(xv[i]);
            raw_f32(xv[i], v);
            if (a.res) apply_row<T, ACT>(v, sc, sh, q); else apply_row<T, ACT>(v, sc, sh, nullptr);
            store8<T>(yp + (size_t)r * a.y_ld, v);
        }
    }
}

// Second kernel of the tiled form: every workgroup merges its sample's (mean, M2) partials, then applies.
template <typename T, int ACT>
__global__ void __launch_bounds__(512) gn_fwd_apply(const GnArgs a) {
    __shared__ float mu[GN_MAX_GROUPS], rs[GN_MAX_GROUPS];
    const Place p = gn_place(a, blockIdx.x);
    const int lane = threadIdx.x & 63, cg = a.cg.d;
    for (int g = threadIdx.x >> 6; g < p.ngr; g += blockDim.x >> 6) {
        const float* q = a.part + ((size_t)p.b * a.G + p.g0 + g) * a.tiles * 2;
        float sm_ = 0.f, m2 = 0.f;
        for (int t = lane; t < a.tiles; t += 64) {
            const float n = (float)min(a.rows_tile, a.HW - t * a.rows_tile);
            sm_ += n * q[2 * t];
            m2 += q[2 * t + 1];
        }
        const float mean = wave_sum(sm_) / (float)a.HW;
        for (int t = lane; t < a.tiles; t += 64) {
            const float n = (float)min(a.rows_tile, a.HW - t * a.rows_tile) * (float)cg, d = q[2 * t] - mean;
            m2 += n * d * d;
        }
        const float var = wave_sum(m2) / ((float)a.HW * (float)cg);
        if (lane == 0) {
            mu[g] = mean;
            rs[g] = 1.f / sqrtf(var + a.eps);
            if (a.stats && p.tile == 0) {
                const size_t o = (size_t)p.b * a.G + p.g0 + g;
                a.stats[o] = mean;
                a.stats[(size_t)a.B * a.G + o] = rs[g];
            }
        }
    }
    __syncthreads();
    if (!p.live) return;
    int gi[8];
    chunk_groups(a, p, gi);
    const int c = p.c0 + p.chunk * 8;
    float sc[8], sh[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { sc[j] = a.gamma[c + j] * rs[gi[j]]; sh[j] = fmaf(-mu[gi[j]], sc[j], a.beta[c + j]); }
    const size_t row0 = (size_t)p.b * a.HW;
    constexpr int U = 4;                             // rows in flight per thread
    for (int r0 = p.r0 + p.ty; r0 < p.r1; r0 += U * a.rpp) {
        Raw8<T> xr[U], rr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = min(r0 + u * a.rpp, p.r1 - 1);
            raw_load(xr[u], (const T*)a.x + (row0 + r) * a.x_ld + c);
            if (a.res) raw_load(rr[u], (const T*)a.res + (row0 + r) * a.res_ld + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * a.rpp;
            if (r < p.r1) {
                float v[8], q[8];
                raw_f32(xr[u], v);
                if (a.res) raw_f32(rr[u], q);
                if (a.res) apply_row<T, ACT>(v, sc, sh, q); else apply_row<T, ACT>(v, sc, sh, nullptr);
                store8<T>((T*)a.y + (row0 + r) * a.y_ld + c, v);
            }
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------------
// One row of a chunk: x and g = dy act'(pre)
template <typename T, int ACT, bool RES>
__device__ __forceinline__ void bwd_row(const Raw8<T>& xr, const Raw8<T>& dr, const Raw8<T>& rr, const float (&sc)[8], const float (&sh)[8],
                                        float (&x)[8], float (&g)[8]) {
    float q[8];
    raw_f32(xr, x);
    raw_f32(dr, g);
    if (RES) raw_f32(rr, q);
    if (ACT != CVG_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float u = fmaf(x[j], sc[j], sh[j]);
            if (RES) u += q[j];
            g[j] *= act_slope<sizeof(T) == 4>(u, ACT);
        }
    }
}

template <typename T, int ACT, int R, bool RES, int MAXT, int WAVES>
__global__ void __launch_bounds__(MAXT, WAVES) gn_bwd_tile(const GnArgs a) {
    extern __shared__ float sm[];
    __shared__ float sums[2][GN_MAX_GROUPS];
    const Place p = gn_place(a, blockIdx.x);
    const size_t row0 = (size_t)p.b * a.HW + p.r0;
    const int rows = p.r1 - p.r0, c = p.c0 + (p.live ? p.chunk * 8 : 0);
    int gi[8];
    chunk_groups(a, p, gi);
    const float* gmean = a.stats + (size_t)p.b * a.G + p.g0;
    const float* grstd = gmean + (size_t)a.B * a.G;
    float mean[8], sc[8], sh[8], acc[2][8];
    {
        float ga[8], be[8];
        load8<float>(a.gamma + c, ga);
        load8<float>(a.beta + c, be);
#pragma unroll
        for (int j = 0; j < 8; ++j) { mean[j] = gmean[gi[j]]; sc[j] = grstd[gi[j]]; }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sc[j] *= ga[j];
            sh[j] = fmaf(-mean[j], sc[j], be[j]);
            acc[0][j] = acc[1][j] = 0.f;
        }
    }
    Raw8<T> xv[R], dv[R], qv[RES ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const size_t r = row0 + min(p.ty + i * a.rpp, rows - 1);
        raw_load(xv[i], (const T*)a.x + r * a.x_ld + c);
        raw_load(dv[i], (const T*)a.dy + r * a.y_ld + c);
        if (RES) raw_load(qv[RES ? i : 0], (const T*)a.res + r * a.res_ld + c);
    }
    const int mine = p.live ? rows : 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (p.ty + i * a.rpp < mine) {
            float x[8], g[8];
            pin(xv[i]);
            pin(dv[i]);
            bwd_row<T, ACT, RES>(xv[i], dv[i], qv[RES ? i : 0], sc, sh, x, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) { acc[0][j] += g[j]; acc[1][j] += g[j] * (x[j] - mean[j]); }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[1][j] *= grstd[gi[j]];         // sum of g xhat
    column_parts<2>(a, p, acc, sm);
    column_totals<2>(a, sm);
    const int width = a.nv * 8;
    float* o = a.part + ((size_t)p.b * a.tiles + p.tile) * 2 * a.C + p.c0;
    for (int t = threadIdx.x; t < p.nch; t += blockDim.x) {
        o[t] = sm[t];
        o[a.C + t] = sm[(size_t)a.ent * width + t];
    }
    if (a.tiles > 1) return;
    const float inv_n = 1.f / ((float)a.HW * (float)a.cg.d);
    group_sums<2>(a, p, sm, a.gamma, 1, sums, [&](float s) { return s * inv_n; });
    // dx = rstd (gamma g - mean(gamma g) - xhat mean(gamma g xhat)) = sc g + (x cd + c0)
    float cd[8], c0[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float rstd = grstd[gi[j]];
        cd[j] = -rstd * rstd * sums[1][gi[j]];
        c0[j] = fmaf(-mean[j], cd[j], -rstd * sums[0][gi[j]]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = p.ty + i * a.rpp;
        if (r < mine) {
            float x[8], g[8];
            pin(xv[i]);
            pin(dv[i]);
            bwd_row<T, ACT, RES>(xv[i], dv[i], qv[RES ? i : 0], sc, sh, x, g);
            if (a.dres) store8<T>((T*)a.dres + (row0 + r) * a.dres_ld + c, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = fmaf(sc[j], g[j], fmaf(x[j], cd[j], c0[j]));
            store8<T>((T*)a.dx + (row0 + r) * a.dx_ld + c, g);
        }
    }
}

// dgamma / dbeta from the partial rows [P][2][C] (P = samples * tiles): 16 columns by blockDim / 16 row lanes per workgroup
struct ParamGrad {
    const float* part;
    float *dgamma, *dbeta;
    int P, C, blocks;
};
__device__ __forceinline__ void param_grad(const ParamGrad& a, int blk, float (*sm)[17]) {
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, lanes = blockDim.x >> 4, col = blk * 16 + cl;     // columns: dbeta, then dgamma
    float s = 0.f;
    if (col < 2 * a.C) {
#pragma unroll 8
        for (int i = rl; i < a.P; i += lanes) s += a.part[(size_t)i * 2 * a.C + col];
    }
    sm[rl][cl] = s;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    // one wave: 4 lanes per column, a quarter of the rows each
    const int c = threadIdx.x & 15, q = threadIdx.x >> 4, per = lanes >> 2, cc = blk * 16 + c;
    float t = 0.f;
    for (int i = 0; i < per; ++i) t += sm[q * per + i][c];
    t += __shfl_xor(t, 16, 64);
    t += __shfl_xor(t, 32, 64);
    if (q == 0 && cc < 2 * a.C) (cc < a.C ? a.dbeta : a.dgamma)[cc < a.C ? cc : cc - a.C] = t;
}
__global__ void __launch_bounds__(1024) gn_param_grad(const ParamGrad a) {
    __shared__ float sm[64][17];
    param_grad(a, blockIdx.x, sm);
}

// The first blocks take the parameters' gradients, which need the same partial sums: a launch less.
template <typename T, int ACT, bool RES>
__global__ void __launch_bounds__(512) gn_bwd_apply(const GnArgs a, const ParamGrad pg) {
    extern __shared__ float sm[];            // [2][slab channels]
    __shared__ float sums[2][GN_MAX_GROUPS];
    __shared__ float pgm[32][17];
    if ((int)blockIdx.x < pg.blocks) {
        param_grad(pg, blockIdx.x, pgm);
        return;
    }
    const Place p = gn_place(a, blockIdx.x - pg.blocks);
    const int width = a.nv * 8;
    const float* q = a.part + (size_t)p.b * a.tiles * 2 * a.C + p.c0;
    for (int t = threadIdx.x; t < 2 * width; t += blockDim.x) {
        const int n = t >= width ? 1 : 0, ch = t - n * width;
        float s = 0.f;
        if (ch < p.nch)
#pragma unroll 8
            for (int i = 0; i < a.tiles; ++i) s += q[((size_t)i * 2 + n) * a.C + ch];
        sm[t] = s;
    }
    __syncthreads();
    group_sums<2>(a, p, sm, a.gamma, 1, sums, [](float s) { return s; });   // (a.ent is 1 in this launch)
    if (!p.live) return;
    int gi[8];
    chunk_groups(a, p, gi);
    const int c = p.c0 + p.chunk * 8;
    const float inv_n = 1.f / ((float)a.HW * (float)a.cg.d);
    float sc[8], sh[8], cd[8], c0[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const size_t o = (size_t)p.b * a.G + p.g0 + gi[j];
        const float rstd = a.stats[(size_t)a.B * a.G + o], mean = a.stats[o];
        sc[j] = a.gamma[c + j] * rstd;
        sh[j] = fmaf(-mean, sc[j], a.beta[c + j]);
        cd[j] = -rstd * rstd * sums[1][gi[j]] * inv_n;
        c0[j] = fmaf(-mean, cd[j], -rstd * sums[0][gi[j]] * inv_n);
    }
    const size_t row0 = (size_t)p.b * a.HW;
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    for (int r0 = p.r0 + p.ty; r0 < p.r1; r0 += U * a.rpp) {
        Raw8<T> xr[U], dr[U], rr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t r = row0 + min(r0 + u * a.rpp, p.r1 - 1);
            raw_load(xr[u], (const T*)a.x + r * a.x_ld + c);
            raw_load(dr[u], (const T*)a.dy + r * a.y_ld + c);
            if (RES) raw_load(rr[u], (const T*)a.res + r * a.res_ld + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * a.rpp;
            if (r < p.r1) {
                float x[8], g[8];
                bwd_row<T, ACT, RES>(xr[u], dr[u], rr[u], sc, sh, x, g);
                if (a.dres) store8<T>((T*)a.dres + (row0 + r) * a.dres_ld + c, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = fmaf(sc[j], g[j], fmaf(x[j], cd[j], c0[j]));
                store8<T>((T*)a.dx + (row0 + r) * a.dx_ld + c, g);
            }
        }
    }
}

// ---- planning ----------------------------------------------------------------------------------------------
struct Plan {
    int nv, nslab, threads, R, tiles, rows_tile, rpp;
};
int gcd(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

int check(const cvg_gn_desc* d, const char* who) {
    CVG_CHECK(d, "%s: null descriptor", who);
    CVG_CHECK(d->dtype == CVG_F32 || d->dtype == CVG_BF16, "%s: dtype %d", who, d->dtype);
    CVG_CHECK(d->B >= 0 && d->HW >= 1 && d->C >= 8 && d->C <= 1 << 24 && d->G >= 1, "%s: B %d, HW %d, C %d, G %d", who, d->B, d->HW, d->C, d->G);
    CVG_CHECK(d->C % 8 == 0, "%s: C = %d is not a multiple of 8", who, d->C);
    CVG_CHECK(d->C % d->G == 0, "%s: %d groups do not divide %d channels", who, d->G, d->C);
    const int cg = d->C / d->G;
    CVG_CHECK((int64_t)cg / gcd(cg, 8) * 8 <= 4096, "%s: groups of %d channels are too wide", who, cg);
    CVG_CHECK((int64_t)d->B * d->HW <= 0x7fff0000, "%s: %lld pixel rows", who, (long long)d->B * d->HW);   // (row loops step past the end)
    CVG_CHECK(act_known(d->act), "%s: activation %d", who, d->act);
    CVG_CHECK(d->eps >= 0.f, "%s: eps %g", who, (double)d->eps);
    const int per16 = d->dtype == CVG_BF16 ? 8 : 4;
    const int lds[5] = {d->x_ld, d->res_ld, d->y_ld, d->dx_ld, d->dres_ld};
    for (int ld : lds) CVG_CHECK(ld == 0 || (ld >= d->C && ld % per16 == 0), "%s: pitch %d for %d channels", who, ld, d->C);
    return 0;
}

// One tile per (sample, slab) or several?  Registers hold rmax chunks per thread (512 threads of 16 bf16 chunks: 128 KB).
//   Large batches: the widest slab, up to 128 bytes of a pixel row, that still fits and leaves 256 workgroups.  Measured
//     forward on 256 x 32 x 32 x 128 bf16 with skip: 47 us at 64-byte slabs, 53 at 128 (too few workgroups), and on
//     256 x 64 x 64 x 64 (512 KB a sample, so 32-byte slabs) 76 us against 87 for the two kernels of the tiled form.
//   Few samples: a workgroup's own arithmetic counts, about 1.8 us per 1000 bf16 chunks (5 in f32), against some 5 us
//     for a second launch.  Forward / backward us of 64 channels in 32 groups, one workgroup per slab and in tiles:
//       bf16, 1 sample    1024 pixels 6.4 / 10.4 and 8.2 / 9.1   2025  9.4 / 14.7 and  8.3 /  8.4   4096 13.5 / 22.9 and  8.4 /  9.0
//             8 samples   2025        8.9 / 14.0 and 10.2 / 11.9 3025 12.0 / 18.5 and 14.1 / 18.1   4096 13.0 / 20.8 and 12.4 / 14.9
//       f32,  1 sample     784        7.0 / 10.3 and 8.7 / 9.7   1024  7.2 / 12.4 and  8.6 /  9.8   2025 11.4 / 18.0 and  8.8 /  9.0
//             8 samples   1024        8.4 / 12.5 and 10.3 / 12.4 1444 10.1 / 15.4 and 12.6 / 15.8   2025 11.6 / 17.9 and 11.9 / 13.3
//     One 64 x 64 x 64 picture is 16 tiles of 256 chunks in each of 8 slabs, the f32 crop 3 x 1961 x 72 (10.3 forward, 12.7
//     backward) 8 tiles in each of 27.
Plan plan(const cvg_gn_desc* d, bool backward, bool res) {
    Plan p;
    const int cg = d->C / d->G, unit = cg / gcd(cg, 8);             // chunks of 8 channels that hold whole groups
    const int all = d->C / 8;
    const bool bf = d->dtype == CVG_BF16;
    const int want = bf ? 8 : 4;                                    // 128 bytes of a pixel row
    const int rmax = (bf ? 16 : 8) / (backward && res ? 2 : 1);
    auto cap = [&](int nv) { return 512 / nv * rmax; };             // rows one workgroup holds
    int wide = unit;
    while (wide < want && wide + unit <= all) wide += unit;
    int nv = wide;
    while (nv > unit && (d->HW > cap(nv) || (int64_t)d->B * ceil_div(all, nv) < 256)) nv -= unit;
    const int64_t groups_of = (int64_t)d->B * ceil_div(all, nv);    // workgroups with one tile each
    bool single = d->HW <= cap(nv);
    if (groups_of < 256 && (int64_t)d->HW * nv > (bf ? 3000 : 1000)) single = false;
    p.threads = nv <= 256 ? 256 : 512;
    int rows = rmax;
    if (single) {
        while (p.threads < 512 && p.threads / nv * rmax < d->HW) p.threads *= 2;
    } else {
        const int64_t chunks = (int64_t)d->B * d->HW * all;
        if (chunks > (1 << 19)) nv = wide;                          // more than 8 MB: bandwidth, not latency
        p.threads = nv <= 256 ? 256 : 512;
        // about 512 workgroups, and no more tiles per sample than one wave merges at once
        rows = 1;
        while (rows < rmax && (chunks > (int64_t)rows * 512 * 256 || (int64_t)rows * (p.threads / nv) * 64 < d->HW)) rows *= 2;
        while (p.threads < 512 && chunks > (int64_t)rows * 1024 * 256) p.threads *= 2;
    }
    p.nv = nv;
    p.nslab = ceil_div(all, nv);
    p.rpp = p.threads / nv;
    const int need = min(rows, ceil_div(d->HW, p.rpp));
    p.R = 1;
    while (p.R < need) p.R *= 2;
    p.rows_tile = min(d->HW, p.R * p.rpp);
    p.tiles = ceil_div(d->HW, p.rows_tile);
    return p;
}

int entries(const Plan& p) {
    const bool fold = (p.nv & (p.nv - 1)) == 0 && p.nv <= 32;
    return fold ? p.threads / 64 : p.rpp;
}

void fill(GnArgs& a, const cvg_gn_desc* d, const Plan& p) {
    a.B = d->B; a.HW = d->HW; a.C = d->C; a.G = d->G; a.act = d->act; a.eps = d->eps;
    a.tiles = p.tiles; a.rows_tile = p.rows_tile; a.nslab = p.nslab; a.nv = p.nv; a.rpp = p.rpp; a.ent = entries(p);
    a.x_ld = d->x_ld ? d->x_ld : d->C; a.res_ld = d->res_ld ? d->res_ld : d->C; a.y_ld = d->y_ld ? d->y_ld : d->C;
    a.dx_ld = d->dx_ld ? d->dx_ld : d->C; a.dres_ld = d->dres_ld ? d->dres_ld : d->C;
    a.seg = 1;
    while (a.seg < 64 && a.seg < a.ent * (d->C / d->G)) a.seg *= 2;
    a.cg = make_fastdiv(d->C / d->G); a.nvd = make_fastdiv(p.nv); a.tiled = make_fastdiv(p.tiles); a.slabd = make_fastdiv(p.nslab);
}

bool launchable(const cvg_gn_desc* d, const Plan& p) {
    return ((int64_t)d->B * p.nslab * p.tiles + ceil_div(2 * d->C, 16)) * p.threads < (int64_t)1 << 32;
}
size_t ws_need(const cvg_gn_desc* d, const Plan& p, bool backward) {
    if (backward) return (size_t)d->B * p.tiles * 2 * d->C * 4;
    return p.tiles > 1 ? (size_t)d->B * d->G * p.tiles * 2 * 4 : 0;
}

// (the second number of a launch bound is waves per SIMD: 4 leave 128 registers, 2 leave 256)
template <typename T, int ACT>
void run_fwd(const GnArgs& a, const Plan& p, hipStream_t s) {
    const int blocks = a.B * p.nslab * p.tiles;
    const size_t lds = (size_t)a.ent * p.nv * 8 * 4;
    constexpr int RMAX = sizeof(T) == 2 ? 16 : 8;
    if (p.R == 1) gn_fwd_tile<T, ACT, 1, 512, 4><<<blocks, p.threads, lds, s>>>(a);
    else if (p.R <= RMAX / 4) gn_fwd_tile<T, ACT, RMAX / 4, 512, 4><<<blocks, p.threads, lds, s>>>(a);
    else if (p.R <= RMAX / 2) gn_fwd_tile<T, ACT, RMAX / 2, 512, 4><<<blocks, p.threads, lds, s>>>(a);
    else gn_fwd_tile<T, ACT, RMAX, 512, 4><<<blocks, p.threads, lds, s>>>(a);
    if (p.tiles > 1) gn_fwd_apply<T, ACT><<<blocks, p.threads, 0, s>>>(a);
}
template <typename T, int ACT, bool RES>
void run_bwd(GnArgs a, const Plan& p, ParamGrad pg, hipStream_t s) {
    const int blocks = a.B * p.nslab * p.tiles;
    const size_t lds = (size_t)a.ent * p.nv * 8 * 4 * 2;
    constexpr int RMAX = (sizeof(T) == 2 ? 16 : 8) / (RES ? 2 : 1);
    if (p.R == 1) gn_bwd_tile<T, ACT, 1, RES, 512, 4><<<blocks, p.threads, lds, s>>>(a);
    else if (p.R <= RMAX / 4) gn_bwd_tile<T, ACT, RMAX / 4, RES, 512, 2><<<blocks, p.threads, lds, s>>>(a);
    else if (p.R <= RMAX / 2) gn_bwd_tile<T, ACT, RMAX / 2, RES, 512, 2><<<blocks, p.threads, lds, s>>>(a);
    else gn_bwd_tile<T, ACT, RMAX, RES, 512, 2><<<blocks, p.threads, lds, s>>>(a);
    if (p.tiles > 1) {
        a.ent = 1;
        gn_bwd_apply<T, ACT, RES><<<blocks + pg.blocks, p.threads, (size_t)2 * p.nv * 8 * 4, s>>>(a, pg);
    } else {
        gn_param_grad<<<pg.blocks, 1024, 0, s>>>(pg);
    }
}
template <typename T, int ACT>
void run_bwd(const GnArgs& a, const Plan& p, const ParamGrad& pg, hipStream_t s) {
    if (a.res) run_bwd<T, ACT, true>(a, p, pg, s); else run_bwd<T, ACT, false>(a, p, pg, s);
}
#define GN_BY_ACT(run, T, ...) \
    switch (a.act) { \
        case CVG_ACT_LRELU: run<T, CVG_ACT_LRELU>(a, p, __VA_ARGS__); break; \
        case CVG_ACT_SILU: run<T, CVG_ACT_SILU>(a, p, __VA_ARGS__); break; \
        case CVG_ACT_GELU: run<T, CVG_ACT_GELU>(a, p, __VA_ARGS__); break; \
        default: run<T, CVG_ACT_NONE>(a, p, __VA_ARGS__); \
    }

}  // namespace

extern "C" {

size_t cvg_gn_act_workspace(const cvg_gn_desc* d, int32_t backward) {
    if (check(d, "gn_act_workspace") != 0) return 0;
    size_t n = ws_need(d, plan(d, false, false), false);
    for (int res = 0; res < 2 && backward; ++res) {
        const size_t b = ws_need(d, plan(d, true, res), true);
        n = b > n ? b : n;
    }
    return n;
}

int cvg_gn_act_fwd(const cvg_gn_desc* d, const void* x, const void* res, void* y, float* stats, const float* gamma,
                   const float* beta, void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "gn_act_fwd") != 0) return -1;
    CVG_CHECK(gamma && beta, "gn_act_fwd: null gamma / beta");
    if (d->B == 0) return 0;
    CVG_CHECK(x && y, "gn_act_fwd: null tensor");
    CVG_CHECK(aligned16(x) && aligned16(res) && aligned16(y), "gn_act_fwd: tensors have to start at 16-byte borders");
    const Plan p = plan(d, false, res != nullptr);
    CVG_CHECK(launchable(d, p), "gn_act_fwd: too many tiles");
    const size_t need = ws_need(d, p, false);
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 3) == 0), "gn_act_fwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    const int x_ld = d->x_ld ? d->x_ld : d->C, res_ld = d->res_ld ? d->res_ld : d->C, y_ld = d->y_ld ? d->y_ld : d->C;
    CVG_CHECK((y != x || y_ld == x_ld) && (y != res || y_ld == res_ld), "gn_act_fwd: in place with different pitches");
    CVG_CHECK(apart({y, stats}, {gamma, beta}) && apart({stats}, {x, res}), "gn_act_fwd: an output over another tensor");
    GnArgs a{};
    fill(a, d, p);
    a.x = x; a.res = res; a.y = y; a.stats = stats; a.gamma = gamma; a.beta = beta; a.part = (float*)ws;
    hipStream_t st = (hipStream_t)s;
    if (d->dtype == CVG_BF16) { GN_BY_ACT(run_fwd, bf16, st) } else { GN_BY_ACT(run_fwd, float, st) }
    CVG_LAUNCH_CHECK();
    return 0;
}

int cvg_gn_act_bwd(const cvg_gn_desc* d, const void* dy, const void* x, const void* res, void* dx, void* dres,
                   const float* stats, const float* gamma, const float* beta, float* dgamma, float* dbeta,
                   void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "gn_act_bwd") != 0) return -1;
    CVG_CHECK(gamma && beta && dgamma && dbeta, "gn_act_bwd: null gamma / beta / dgamma / dbeta");
    CVG_CHECK(d->B == 0 || (dy && x && dx && stats), "gn_act_bwd: null tensor");
    CVG_CHECK(aligned16(x) && aligned16(res) && aligned16(dy) && aligned16(dx) && aligned16(dres),
              "gn_act_bwd: tensors have to start at 16-byte borders");
    const Plan p = plan(d, true, res != nullptr);
    CVG_CHECK(launchable(d, p), "gn_act_bwd: too many tiles");
    const size_t need = ws_need(d, p, true);
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 3) == 0), "gn_act_bwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    const int dy_ld = d->y_ld ? d->y_ld : d->C, dx_ld = d->dx_ld ? d->dx_ld : d->C, dres_ld = d->dres_ld ? d->dres_ld : d->C;
    CVG_CHECK(!dy || ((dx != dy || dx_ld == dy_ld) && (dres != dy || dres_ld == dy_ld)), "gn_act_bwd: in place with different pitches");
    // (dgamma and dbeta are written while other workgroups still read gamma, beta and stats)
    CVG_CHECK(apart({dx, dres, dgamma, dbeta}, {x, res, stats, gamma, beta}) && apart({dgamma, dbeta}, {dy}),
              "gn_act_bwd: a gradient over another tensor");
    GnArgs a{};
    fill(a, d, p);
    a.x = x; a.res = res; a.dy = dy; a.dx = dx; a.dres = dres; a.stats = (float*)stats; a.gamma = gamma; a.beta = beta;
    a.part = (float*)ws;
    hipStream_t st = (hipStream_t)s;
    const ParamGrad pg{a.part, dgamma, dbeta, d->B * p.tiles, d->C, ceil_div(2 * d->C, 16)};
    if (d->B == 0) {
        gn_param_grad<<<pg.blocks, 1024, 0, st>>>(pg);          // (sums over nothing)
    } else if (d->dtype == CVG_BF16) {
        GN_BY_ACT(run_bwd, bf16, pg, st)
    } else {
        GN_BY_ACT(run_bwd, float, pg, st)
    }
    CVG_LAUNCH_CHECK();
    return 0;
}

}
