// Group normalisation with an activation over channels-last tensors, forward and backward.
//
// A workgroup owns a TILE: some pixel rows of one sample, over a SLAB of channels that holds whole groups.  Its
// elements are read once into registers as 16-byte chunks of 8 channels (thread = one chunk column, every
// rows_per_pass-th row) and everything the tile needs is computed from there: the mean first, then the sum of
// (x - mean)^2, so no digits are lost to E[x^2] - mean^2.
//   one tile per (sample, slab): the workgroup normalises its registers and writes y; x is read once.
//   more than one: the tiles write (mean, M2) per group, a second kernel merges them (Chan's formula) and applies.
// The backward pass is built the same way over per-channel sums of g and g * xhat, which also give dgamma / dbeta.
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
    FastDiv cg, nvd, tiled, slabd;   // divisions by C / G, nv, tiles, nslab
};

constexpr int GN_MAX_GROUPS = 64;    // groups of a slab (slabs wider than 64 channels hold at most 8)

// What a thread knows about its place: chunk column, first row, channels.
struct Place {
    int b, tile, c0, chunk, ty, r0, r1, nv, nch, ngr, g0;
    bool live;
};
__device__ __forceinline__ Place gn_place(const GnArgs& a) {
    Place p;
    uint32_t blk = blockIdx.x;
    const uint32_t bs = fdiv(blk, a.tiled);
    p.tile = blk - bs * a.tiles;
    p.b = fdiv(bs, a.slabd);
    const int slab = bs - p.b * a.nslab;
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

// Column sums over the workgroup: N values per channel of the slab, sm[n][ent][nv * 8]; afterwards sm[n][0][c] holds
// the sum of channel c.  Where the chunk count is a power of two up to 32 the lanes of a wave that hold the same chunk
// are added by shuffles first, which leaves one entry per wave, otherwise one per row lane.
template <int N>
__device__ __forceinline__ void column_sums(const GnArgs& a, const Place& p, float (&v)[N][8], float* sm) {
    const int width = a.nv * 8;
    const bool fold = (a.nv & (a.nv - 1)) == 0 && a.nv <= 32;
    int e = p.ty;
    bool writes = p.ty < a.rpp;
    if (fold) {
        for (int o = a.nv; o < 64; o <<= 1)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[n][j] += __shfl_xor(v[n][j], o, 64);
        e = threadIdx.x >> 6;
        writes = (int)(threadIdx.x & 63) < a.nv;
    }
    __syncthreads();                 // the last readers of sm are done
    if (writes)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < 8; j += 4)
                *(f32x4*)&sm[(n * a.ent + e) * width + p.chunk * 8 + j] = f32x4{v[n][j], v[n][j + 1], v[n][j + 2], v[n][j + 3]};
    __syncthreads();
    for (int t = threadIdx.x; t < N * width; t += blockDim.x) {
        const int n = t >= width ? 1 : 0, c = t - n * width;
        float* q = sm + (size_t)n * a.ent * width + c;
        float s = 0.f;
        for (int i = 0; i < a.ent; ++i) s += q[i * width];
        q[0] = s;                    // only this thread touches column c
    }
    __syncthreads();
}

// sums[n][g] = sum over the channels of group g of w[c] * sm[n][0][c] (w = 1 where null): a wave per group, lanes over channels
template <int N>
__device__ __forceinline__ void group_sums(const GnArgs& a, const Place& p, const float* sm, const float* w, float (*sums)[GN_MAX_GROUPS]) {
    const int cg = a.cg.d, width = a.nv * 8, lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < p.ngr; g += blockDim.x >> 6) {
        float s[N];
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] = 0.f;
        for (int c = g * cg + lane; c < (g + 1) * cg; c += 64) {
            const float k = w ? w[p.c0 + c] : 1.f;
#pragma unroll
            for (int n = 0; n < N; ++n) s[n] += k * sm[(size_t)n * a.ent * width + c];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float t = wave_sum(s[n]);
            if (lane == 0) sums[n][g] = t;
        }
    }
    __syncthreads();
}

// per-channel constants of a thread's chunk
__device__ __forceinline__ void chunk_groups(const GnArgs& a, const Place& p, int (&gi)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) gi[j] = p.live ? fdiv(p.chunk * 8 + j, a.cg) : 0;
}

template <typename T, int R>
__global__ void __launch_bounds__(1024) gn_fwd_tile(const GnArgs a) {
    extern __shared__ float sm[];
    __shared__ float sums[2][GN_MAX_GROUPS];
    constexpr bool EXACT = sizeof(T) == 4;
    const Place p = gn_place(a);
    const size_t row0 = (size_t)p.b * a.HW + p.r0;
    const int rows = p.r1 - p.r0, c = p.c0 + p.chunk * 8;
    const T* xp = (const T*)a.x + row0 * a.x_ld + c;
    Raw8<T> xv[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = p.ty + i * a.rpp;
        raw_zero(xv[i]);
        if (p.live && r < rows) raw_load(xv[i], xp + (size_t)r * a.x_ld);
    }
    int gi[8];
    chunk_groups(a, p, gi);
    float acc[1][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[0][j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float v[8];
        raw_f32(xv[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[0][j] += v[j];
    }
    column_sums<1>(a, p, acc, sm);
    group_sums<1>(a, p, sm, nullptr, sums);
    const float inv_n = 1.f / ((float)rows * (float)a.cg.d);
    float mean[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { mean[j] = sums[0][gi[j]] * inv_n; acc[0][j] = 0.f; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (p.ty + i * a.rpp < rows && p.live) {
            float v[8];
            raw_f32(xv[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) { const float d = v[j] - mean[j]; acc[0][j] += d * d; }
        }
    }
    column_sums<1>(a, p, acc, sm);
    group_sums<1>(a, p, sm, nullptr, sums + 1);
    if (a.tiles > 1) {
        for (int g = threadIdx.x; g < p.ngr; g += blockDim.x) {
            float* o = a.part + (((size_t)p.b * a.G + p.g0 + g) * a.tiles + p.tile) * 2;
            o[0] = sums[0][g] * inv_n;
            o[1] = sums[1][g];
        }
        return;
    }
    if (a.stats)
        for (int g = threadIdx.x; g < p.ngr; g += blockDim.x) {
            const size_t o = (size_t)p.b * a.G + p.g0 + g;
            a.stats[o] = sums[0][g] * inv_n;
            a.stats[(size_t)a.B * a.G + o] = 1.f / sqrtf(sums[1][g] * inv_n + a.eps);
        }
    if (!p.live) return;
    float sc[8], be[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        sc[j] = a.gamma[c + j] * (1.f / sqrtf(sums[1][gi[j]] * inv_n + a.eps));
        be[j] = a.beta[c + j];
    }
    const T* rp = (const T*)a.res + row0 * a.res_ld + c;
    T* yp = (T*)a.y + row0 * a.y_ld + c;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = p.ty + i * a.rpp;
        if (r < rows) {
            float v[8], q[8];
            raw_f32(xv[i], v);
            if (a.res) load8<T>(rp + (size_t)r * a.res_ld, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = (v[j] - mean[j]) * sc[j] + be[j];
                if (a.res) v[j] += q[j];
            }
            act_value8<EXACT>(v, a.act);
            store8<T>(yp + (size_t)r * a.y_ld, v);
        }
    }
}

// Second kernel of the tiled form: every workgroup merges its sample's (mean, M2) partials, then applies.
template <typename T>
__global__ void __launch_bounds__(512) gn_fwd_apply(const GnArgs a) {
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ float mu[GN_MAX_GROUPS], rs[GN_MAX_GROUPS];
    const Place p = gn_place(a);
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
    float mean[8], sc[8], be[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { mean[j] = mu[gi[j]]; sc[j] = a.gamma[c + j] * rs[gi[j]]; be[j] = a.beta[c + j]; }
    const size_t row0 = (size_t)p.b * a.HW;
    for (int r = p.r0 + p.ty; r < p.r1; r += a.rpp) {
        float v[8], q[8];
        load8<T>((const T*)a.x + (row0 + r) * a.x_ld + c, v);
        if (a.res) load8<T>((const T*)a.res + (row0 + r) * a.res_ld + c, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = (v[j] - mean[j]) * sc[j] + be[j];
            if (a.res) v[j] += q[j];
        }
        act_value8<EXACT>(v, a.act);
        store8<T>((T*)a.y + (row0 + r) * a.y_ld + c, v);
    }
}

// ---- backward ----------------------------------------------------------------------------------------------
// One row of a chunk: xhat and g = dy act'(pre)
template <typename T>
__device__ __forceinline__ void bwd_row(const Raw8<T>& xr, const Raw8<T>& dr, const Raw8<T>& rr, bool has_res, int act,
                                        const float (&mean)[8], const float (&rstd)[8], const float (&ga)[8], const float (&be)[8],
                                        float (&xh)[8], float (&g)[8]) {
    constexpr bool EXACT = sizeof(T) == 4;
    float q[8], u[8];
    raw_f32(xr, xh);
    raw_f32(dr, g);
    if (has_res) raw_f32(rr, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // the same expression as the forward pass, so that the sign LeakyReLU takes is the same
        const float d = xh[j] - mean[j];
        u[j] = d * (ga[j] * rstd[j]) + be[j];
        if (has_res) u[j] += q[j];
        xh[j] = d * rstd[j];
    }
    if (act != CVG_ACT_NONE) {
        act_slope8<EXACT>(u, act);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] *= u[j];
    }
}

template <typename T, int R, bool RES>
__global__ void __launch_bounds__(1024) gn_bwd_tile(const GnArgs a) {
    extern __shared__ float sm[];
    __shared__ float sums[2][GN_MAX_GROUPS];
    const Place p = gn_place(a);
    const size_t row0 = (size_t)p.b * a.HW + p.r0;
    const int rows = p.r1 - p.r0, c = p.c0 + p.chunk * 8;
    Raw8<T> xv[R], dv[R], qv[RES ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = p.ty + i * a.rpp;
        raw_zero(xv[i]);
        raw_zero(dv[i]);
        if (RES) raw_zero(qv[RES ? i : 0]);
        if (p.live && r < rows) {
            raw_load(xv[i], (const T*)a.x + (row0 + r) * a.x_ld + c);
            raw_load(dv[i], (const T*)a.dy + (row0 + r) * a.y_ld + c);
            if (RES) raw_load(qv[RES ? i : 0], (const T*)a.res + (row0 + r) * a.res_ld + c);
        }
    }
    int gi[8];
    chunk_groups(a, p, gi);
    float mean[8], rstd[8], ga[8], be[8], acc[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const size_t o = (size_t)p.b * a.G + p.g0 + gi[j];
        mean[j] = a.stats[o];
        rstd[j] = a.stats[(size_t)a.B * a.G + o];
        ga[j] = p.live ? a.gamma[c + j] : 0.f;
        be[j] = p.live ? a.beta[c + j] : 0.f;
        acc[0][j] = acc[1][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (p.live && p.ty + i * a.rpp < rows) {
            float xh[8], g[8];
            bwd_row<T>(xv[i], dv[i], qv[RES ? i : 0], RES, a.act, mean, rstd, ga, be, xh, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) { acc[0][j] += g[j]; acc[1][j] += g[j] * xh[j]; }
        }
    }
    column_sums<2>(a, p, acc, sm);
    const int width = a.nv * 8;
    float* o = a.part + ((size_t)p.b * a.tiles + p.tile) * 2 * a.C + p.c0;
    for (int t = threadIdx.x; t < p.nch; t += blockDim.x) {
        o[t] = sm[t];
        o[a.C + t] = sm[(size_t)a.ent * width + t];
    }
    if (a.tiles > 1) return;
    group_sums<2>(a, p, sm, a.gamma, sums);
    if (!p.live) return;
    const float inv_n = 1.f / ((float)a.HW * (float)a.cg.d);
    float A[8], Bq[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { A[j] = sums[0][gi[j]] * inv_n; Bq[j] = sums[1][gi[j]] * inv_n; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = p.ty + i * a.rpp;
        if (r < rows) {
            float xh[8], g[8];
            bwd_row<T>(xv[i], dv[i], qv[RES ? i : 0], RES, a.act, mean, rstd, ga, be, xh, g);
            if (a.dres) store8<T>((T*)a.dres + (row0 + r) * a.dres_ld + c, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = rstd[j] * (ga[j] * g[j] - A[j] - xh[j] * Bq[j]);
            store8<T>((T*)a.dx + (row0 + r) * a.dx_ld + c, g);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(512) gn_bwd_apply(const GnArgs a) {
    extern __shared__ float sm[];            // [2][slab channels]
    __shared__ float sums[2][GN_MAX_GROUPS];
    const Place p = gn_place(a);
    const int width = a.nv * 8;
    const float* q = a.part + (size_t)p.b * a.tiles * 2 * a.C + p.c0;
    for (int t = threadIdx.x; t < 2 * width; t += blockDim.x) {
        const int n = t >= width ? 1 : 0, ch = t - n * width;
        float s = 0.f;
        if (ch < p.nch)
            for (int i = 0; i < a.tiles; ++i) s += q[((size_t)i * 2 + n) * a.C + ch];
        sm[t] = s;
    }
    __syncthreads();
    group_sums<2>(a, p, sm, a.gamma, sums);  // (ent = 1 in this launch)
    if (!p.live) return;
    int gi[8];
    chunk_groups(a, p, gi);
    const int c = p.c0 + p.chunk * 8;
    const float inv_n = 1.f / ((float)a.HW * (float)a.cg.d);
    float mean[8], rstd[8], ga[8], be[8], A[8], Bq[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const size_t o = (size_t)p.b * a.G + p.g0 + gi[j];
        mean[j] = a.stats[o];
        rstd[j] = a.stats[(size_t)a.B * a.G + o];
        ga[j] = a.gamma[c + j];
        be[j] = a.beta[c + j];
        A[j] = sums[0][gi[j]] * inv_n;
        Bq[j] = sums[1][gi[j]] * inv_n;
    }
    const size_t row0 = (size_t)p.b * a.HW;
    const bool has_res = a.res != nullptr;
    for (int r = p.r0 + p.ty; r < p.r1; r += a.rpp) {
        Raw8<T> xr, dr, rr;
        raw_load(xr, (const T*)a.x + (row0 + r) * a.x_ld + c);
        raw_load(dr, (const T*)a.dy + (row0 + r) * a.y_ld + c);
        if (has_res) raw_load(rr, (const T*)a.res + (row0 + r) * a.res_ld + c); else raw_zero(rr);
        float xh[8], g[8];
        bwd_row<T>(xr, dr, rr, has_res, a.act, mean, rstd, ga, be, xh, g);
        if (a.dres) store8<T>((T*)a.dres + (row0 + r) * a.dres_ld + c, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = rstd[j] * (ga[j] * g[j] - A[j] - xh[j] * Bq[j]);
        store8<T>((T*)a.dx + (row0 + r) * a.dx_ld + c, g);
    }
}

// dgamma / dbeta from the partial rows [P][2][C] (P = samples * tiles): 32 channels by 8 row lanes per workgroup
__global__ void __launch_bounds__(256) gn_param_grad(const float* __restrict__ part, int P, int C, float* dgamma, float* dbeta) {
    __shared__ float sm[2][8][32];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
    float s0 = 0.f, s1 = 0.f;
    if (c < C)
        for (int i = rl; i < P; i += 8) {
            s0 += part[(size_t)i * 2 * C + c];
            s1 += part[((size_t)i * 2 + 1) * C + c];
        }
    sm[0][rl][cl] = s0;
    sm[1][rl][cl] = s1;
    __syncthreads();
    if (rl < 2 && c < C) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += sm[rl][i][cl];
        (rl ? dgamma : dbeta)[c] = s;
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
    CVG_CHECK(d->B >= 0 && d->HW >= 1 && d->C >= 8 && d->G >= 1, "%s: B %d, HW %d, C %d, G %d", who, d->B, d->HW, d->C, d->G);
    CVG_CHECK(d->C % 8 == 0, "%s: C = %d is not a multiple of 8", who, d->C);
    CVG_CHECK(d->C % d->G == 0, "%s: %d groups do not divide %d channels", who, d->G, d->C);
    const int cg = d->C / d->G;
    CVG_CHECK((int64_t)cg / gcd(cg, 8) * 8 <= 4096, "%s: groups of %d channels are too wide", who, cg);
    CVG_CHECK((int64_t)d->B * d->HW <= 0x7fffffff, "%s: %lld pixel rows", who, (long long)d->B * d->HW);
    CVG_CHECK(act_known(d->act), "%s: activation %d", who, d->act);
    CVG_CHECK(d->eps >= 0.f, "%s: eps %g", who, (double)d->eps);
    const int per16 = d->dtype == CVG_BF16 ? 8 : 4;
    const int lds[5] = {d->x_ld, d->res_ld, d->y_ld, d->dx_ld, d->dres_ld};
    for (int ld : lds) CVG_CHECK(ld == 0 || (ld >= d->C && ld % per16 == 0), "%s: pitch %d for %d channels", who, ld, d->C);
    return 0;
}

Plan plan(const cvg_gn_desc* d, bool backward) {
    Plan p;
    const int cg = d->C / d->G, unit = cg / gcd(cg, 8);             // chunks of 8 channels that hold whole groups
    const int all = d->C / 8;
    // slabs of 128 bytes per pixel row, or whatever one unit needs
    const int want = d->dtype == CVG_BF16 ? 8 : 4;
    p.nv = unit;
    while (p.nv < want && p.nv + unit <= all) p.nv += unit;
    p.nslab = ceil_div(all, p.nv);
    const int rmax = (d->dtype == CVG_BF16 ? 8 : 4) / (backward ? 2 : 1);
    p.threads = 256;
    // (a chunk count that does not fold leaves one LDS row per row lane: 512 threads keep that within 32 KB)
    const int tmax = (p.nv & (p.nv - 1)) == 0 && p.nv <= 32 ? 1024 : 512;
    while (p.threads < tmax && (p.threads < p.nv || (int64_t)d->HW * p.nv > (int64_t)p.threads * rmax)) p.threads *= 2;
    p.rpp = p.threads / p.nv;
    int need = ceil_div(d->HW, p.rpp);
    if (need > rmax) {
        p.threads = p.nv <= 256 ? 256 : 512;
        p.rpp = p.threads / p.nv;
        need = rmax;
    }
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
    a.cg = make_fastdiv(d->C / d->G); a.nvd = make_fastdiv(p.nv); a.tiled = make_fastdiv(p.tiles); a.slabd = make_fastdiv(p.nslab);
}

size_t ws_need(const cvg_gn_desc* d, const Plan& p, bool backward) {
    if (backward) return (size_t)d->B * p.tiles * 2 * d->C * 4;
    return p.tiles > 1 ? (size_t)d->B * d->G * p.tiles * 2 * 4 : 0;
}

template <typename T>
void run_fwd(const GnArgs& a, const Plan& p, hipStream_t s) {
    const int64_t blocks = (int64_t)a.B * p.nslab * p.tiles;
    const size_t lds = (size_t)a.ent * p.nv * 8 * 4;
    switch (p.R) {
        case 1: gn_fwd_tile<T, 1><<<(int)blocks, p.threads, lds, s>>>(a); break;
        case 2: gn_fwd_tile<T, 2><<<(int)blocks, p.threads, lds, s>>>(a); break;
        case 4: gn_fwd_tile<T, 4><<<(int)blocks, p.threads, lds, s>>>(a); break;
        default: gn_fwd_tile<T, 8><<<(int)blocks, p.threads, lds, s>>>(a); break;
    }
}
template <typename T, bool RES>
void run_bwd(const GnArgs& a, const Plan& p, hipStream_t s) {
    const int64_t blocks = (int64_t)a.B * p.nslab * p.tiles;
    const size_t lds = (size_t)a.ent * p.nv * 8 * 4 * 2;
    switch (p.R) {
        case 1: gn_bwd_tile<T, 1, RES><<<(int)blocks, p.threads, lds, s>>>(a); break;
        case 2: gn_bwd_tile<T, 2, RES><<<(int)blocks, p.threads, lds, s>>>(a); break;
        default: gn_bwd_tile<T, 4, RES><<<(int)blocks, p.threads, lds, s>>>(a); break;
    }
}

}  // namespace

extern "C" {

size_t cvg_gn_act_workspace(const cvg_gn_desc* d, int32_t backward) {
    if (check(d, "gn_act_workspace") != 0) return 0;
    size_t n = ws_need(d, plan(d, false), false);
    if (backward) n = n > ws_need(d, plan(d, true), true) ? n : ws_need(d, plan(d, true), true);
    return n;
}

int cvg_gn_act_fwd(const cvg_gn_desc* d, const void* x, const void* res, void* y, float* stats, const float* gamma,
                   const float* beta, void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "gn_act_fwd") != 0) return -1;
    CVG_CHECK(gamma && beta, "gn_act_fwd: null gamma / beta");
    if (d->B == 0) return 0;
    CVG_CHECK(x && y, "gn_act_fwd: null tensor");
    CVG_CHECK(aligned16(x) && aligned16(res) && aligned16(y), "gn_act_fwd: tensors have to start at 16-byte borders");
    const Plan p = plan(d, false);
    CVG_CHECK((int64_t)d->B * p.nslab * p.tiles <= 0x7fffffff, "gn_act_fwd: too many tiles");
    const size_t need = ws_need(d, p, false);
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 3) == 0), "gn_act_fwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    GnArgs a{};
    fill(a, d, p);
    a.x = x; a.res = res; a.y = y; a.stats = stats; a.gamma = gamma; a.beta = beta; a.part = (float*)ws;
    hipStream_t st = (hipStream_t)s;
    if (d->dtype == CVG_BF16) run_fwd<bf16>(a, p, st); else run_fwd<float>(a, p, st);
    CVG_LAUNCH_CHECK();
    if (p.tiles > 1) {
        const int64_t blocks = (int64_t)d->B * p.nslab * p.tiles;
        if (d->dtype == CVG_BF16) gn_fwd_apply<bf16><<<(int)blocks, p.threads, 0, st>>>(a);
        else gn_fwd_apply<float><<<(int)blocks, p.threads, 0, st>>>(a);
        CVG_LAUNCH_CHECK();
    }
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
    const Plan p = plan(d, true);
    CVG_CHECK((int64_t)d->B * p.nslab * p.tiles <= 0x7fffffff, "gn_act_bwd: too many tiles");
    const size_t need = ws_need(d, p, true);
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 3) == 0), "gn_act_bwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    GnArgs a{};
    fill(a, d, p);
    a.x = x; a.res = res; a.dy = dy; a.dx = dx; a.dres = dres; a.stats = (float*)stats; a.gamma = gamma; a.beta = beta;
    a.part = (float*)ws;
    hipStream_t st = (hipStream_t)s;
    if (d->B > 0) {
        if (d->dtype == CVG_BF16) { if (res) run_bwd<bf16, true>(a, p, st); else run_bwd<bf16, false>(a, p, st); }
        else { if (res) run_bwd<float, true>(a, p, st); else run_bwd<float, false>(a, p, st); }
        CVG_LAUNCH_CHECK();
        if (p.tiles > 1) {
            const int64_t blocks = (int64_t)d->B * p.nslab * p.tiles;
                a.ent = 1;
            const size_t lds = (size_t)2 * p.nv * 8 * 4;
            if (d->dtype == CVG_BF16) gn_bwd_apply<bf16><<<(int)blocks, p.threads, lds, st>>>(a);
            else gn_bwd_apply<float><<<(int)blocks, p.threads, lds, st>>>(a);
            CVG_LAUNCH_CHECK();
        }
    }
    gn_param_grad<<<ceil_div(d->C, 32), 256, 0, st>>>((const float*)ws, d->B * p.tiles, d->C, dgamma, dbeta);
    CVG_LAUNCH_CHECK();
    return 0;
}

}
