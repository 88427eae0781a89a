// Linear layers with bias, activation and residual in the epilogue of the matrix product, forward and backward.
//
// One contraction serves the three products:  D[m][n] = sum_k A(m, k) B(n, k)
//   forward   A = x (k contiguous),  B = w (k contiguous)           M x N x K
//   dx        A = dz (k contiguous), B = w read along its rows       M x K x N
//   dw        A = dz, B = x, both read along their rows              N x K x M
#include "rowops.h"

namespace {

// What happens to an accumulator on its way out.
struct Epi {
    const float* bias;               // [n] or null
    const void* res;                 // T, or null
    void* pre;                       // T, or f32 where pre_f32, or null
    void* out;                       // T, or f32 where out_f32
    size_t res_ld, pre_ld, out_ld;
    int act, out_f32, pre_f32;
};

template <typename T>
__device__ __forceinline__ void emit(const Epi& e, int m, int n, float v) {
    constexpr bool EXACT = sizeof(T) == 4;
    if (e.bias) v += e.bias[n];
    if (e.pre) {
        if (e.pre_f32) ((float*)e.pre)[(size_t)m * e.pre_ld + n] = v;
        else ((T*)e.pre)[(size_t)m * e.pre_ld + n] = from_f32<T>(v);
    }
    v = act_value<EXACT>(v, e.act);
    if (e.res) v += to_f32(((const T*)e.res)[(size_t)m * e.res_ld + n]);
    if (e.out_f32) ((float*)e.out)[(size_t)m * e.out_ld + n] = v;
    else ((T*)e.out)[(size_t)m * e.out_ld + n] = from_f32<T>(v);
}

// 8 consecutive columns of one row through the epilogue.  `whole`: all of them exist and every tensor takes 16-byte
// accesses there.
template <typename T>
__device__ __forceinline__ void emit8(const Epi& e, int m, int n, int n_end, bool whole, float (&v)[8]) {
    constexpr bool EXACT = sizeof(T) == 4;
    if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < n_end) emit<T>(e, m, n + j, v[j]);
        return;
    }
    if (e.bias) {
        float b[8];
        load8<float>(e.bias + n, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += b[j];
    }
    if (e.pre) {
        if (e.pre_f32) store8<float>((float*)e.pre + (size_t)m * e.pre_ld + n, v);
        else store8<T>((T*)e.pre + (size_t)m * e.pre_ld + n, v);
    }
    act_value8<EXACT>(v, e.act);
    if (e.res) {
        float q[8];
        load8<T>((const T*)e.res + (size_t)m * e.res_ld + n, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += q[j];
    }
    if (e.out_f32) store8<float>((float*)e.out + (size_t)m * e.out_ld + n, v);
    else store8<T>((T*)e.out + (size_t)m * e.out_ld + n, v);
}

// D[m][n] = sum_k A(m, k) B(n, k) for one output tile, or one K range of it.
struct GemmArgs {
    const void *A, *B;
    size_t lda, ldb;                 // elements between consecutive m (n) where k is contiguous, between consecutive k otherwise
    int M, N, K;
    int ra, rb;                      // rows of A and B that may be addressed (the padded count where k is strided)
    int tiles_m, tiles_n, k_split;   // k_split: K range of one grid.y slice (a multiple of the K step)
    int vec;                         // every tensor of the epilogue takes 16-byte accesses at multiples of 8 columns
    float* slab;                     // [splits][M][N] partial sums instead of the epilogue, or null
    Epi e;
};

typedef __attribute__((address_space(3))) void* lds_dst;

// One operand of the tile kernel: ROWS rows of the output dimension, BK = 128 bytes of k per stage.
//   k contiguous (COL = false): LDS holds [ROWS][128 bytes]; the 16-byte chunk c of row r lies at c ^ (r & 7), so the 8 rows
//     that one pass of a 16-byte LDS read touches lie in 8 different chunk columns, i.e. in all banks.
//   k strided (COL = true): LDS holds [BK][ROWS]; bf16 fragments come out of ds_read_b64_tr_b16 (TrLoad), whose lanes read
//     8 k-rows of 64 bytes at once; 64-byte block b of k-row k lies at b ^ (k & 3 | (k >> 3 & 1) << 2) (as many bits as there
//     are blocks), which spreads those rows over the banks.  f32 reads single dwords, consecutive along the row.
// The swizzle is applied to the address a lane LOADS FROM: the direct-to-LDS load writes lane l at base + 16 l.
template <typename T, int ROWS, int NWAVES, bool COL>
struct Operand {
    static constexpr int ES = sizeof(T), BK = 128 / ES, BYTES = ROWS * 128;
    static constexpr int NL = BYTES / 1024 / NWAVES;              // 1 KB wave loads per wave and stage
    static_assert(BYTES % (1024 * NWAVES) == 0, "tile");
    static constexpr int RB = ROWS * ES;                          // bytes of a k-row (COL)
    static constexpr int NBLK = RB / 64, BMASK = (NBLK < 8 ? NBLK : 8) - 1;
    static_assert(!COL || RB <= 1024, "tile");
    int off[NL];                                                  // byte offset of this lane's source of each load from `base`
    const char* base;                                             // (uniform) start of the current stage
    int wave, tid;
    size_t step;

    __device__ __forceinline__ static int swz(int k) { return ((k & 3) | ((k >> 3 & 1) << 2)) & BMASK; }
    // first k, inside the stage, of load i of this lane
    __device__ __forceinline__ int k_of(int i) const {
        const int o = (i * NWAVES + wave) * 1024 + (tid & 63) * 16;
        if constexpr (!COL) return (((o >> 4) & 7) ^ ((o >> 7) & 7)) * (16 / ES);
        else return o / RB;
    }
    __device__ __forceinline__ void init(const void* p, size_t ld, int row0, int rows, int k0, int tid_) {
        tid = tid_;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        step = COL ? (size_t)BK * ld * ES : 128;
        base = (const char*)p + (COL ? ((size_t)k0 * ld + row0) * ES : ((size_t)row0 * ld + k0) * ES);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int o = (i * NWAVES + wave) * 1024 + (tid & 63) * 16;
            if constexpr (!COL) {
                const int r = min(o >> 7, rows - 1 - row0);       // rows beyond the matrix repeat its last one
                off[i] = (int)((size_t)r * ld * ES) + k_of(i) * ES;
            } else {
                const int k = o / RB, c = (o % RB) >> 4;
                const int cs = ES == 2 ? (((c >> 2) ^ swz(k)) << 2) | (c & 3) : c;
                int g = cs * (16 / ES);
                if (row0 + g >= rows) g = 0;                      // (rows is a multiple of the chunk)
                off[i] = (int)((size_t)k * ld * ES) + g * ES;
            }
        }
    }
    // FULL: the whole stage lies inside the k range; otherwise it is zero from k_left on
    template <bool FULL> __device__ __forceinline__ void issue(char* lds, int k_left) {
#ifdef __HIP_DEVICE_COMPILE__
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            char* to = lds + (i * NWAVES + wave) * 1024;
            if (FULL || k_of(i) < k_left)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_dst)to, 16, off[i], 0, 0, 0);
            else
                *(u32x4*)(to + (tid & 63) * 16) = u32x4{0, 0, 0, 0};
        }
#endif
        base += step;
    }
    // fragment of rows r0 .. r0 + 31, k-step s (16 values: slot (h, j) = k 8 h + j)
    __device__ __forceinline__ static typename Elem<T>::frag frag(const char* lds, int r0, int s, int lane) {
        const int l31 = lane & 31, h = lane >> 5;
        if constexpr (!COL) {
            const char* q = lds + (r0 + l31) * 128;
            if constexpr (ES == 2) {
                return *(const bf16x8*)(q + (((2 * s + h) ^ (l31 & 7)) << 4));
            } else {
                const f32x4 a = *(const f32x4*)(q + (((4 * s + 2 * h) ^ (l31 & 7)) << 4));
                const f32x4 b = *(const f32x4*)(q + (((4 * s + 2 * h + 1) ^ (l31 & 7)) << 4));
                return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            }
        } else {
            if constexpr (ES == 2) {
                typedef __attribute__((address_space(3))) bf16x4* lds4;
                const int i = lane & 15, qd = i >> 2, pp = i & 3, blk = (lane >> 4) & 1;
                const int f = (qd | (h << 2)) & BMASK;
                const char* q = lds + (16 * s + 8 * h + qd) * RB + ((((r0 >> 5) ^ f) << 6) | (blk * 32 + pp * 8));
                const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)q);
                const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(q + 4 * RB));
                return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            } else {
                f32x8 r;
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j] = *(const float*)(lds + (16 * s + 8 * h + j) * RB + (r0 + l31) * 4);
                return r;
            }
        }
    }
};

// Tile kernel: BM x BN per workgroup of WR x WC waves.  Two LDS stages of 128 bytes of k, filled by direct-to-LDS loads
// two stages ahead; fragments are read one 16-k step ahead of the MFMAs that use them, across the stage border too, so
// the one barrier of a stage sits between the last fragment reads of a stage and the MFMAs on them.
template <typename T, int BM, int BN, int WR, int WC, bool ACOL, bool BCOL>
__global__ void __launch_bounds__(WR * WC * 64) gemm_tile(GemmArgs a) {
    constexpr int NW = WR * WC, WM = BM / WR, WN = BN / WC, TI = WM / 32, TJ = WN / 32;
    typedef Operand<T, BM, NW, ACOL> OA;
    typedef Operand<T, BN, NW, BCOL> OB;
    typedef typename Elem<T>::frag frag;
    constexpr int BK = OA::BK, NS = BK / 16;
    constexpr int STAGE = OA::BYTES + OB::BYTES;
    constexpr int EP = WN * 4 + 16, EPI = NW * 32 * EP;            // epilogue: 32 rows of the wave's columns, f32
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE > EPI ? 2 * STAGE : EPI];
    // workgroups go round-robin over the 8 dies, each with its own L2: give every die a run of neighbouring tiles, walked
    // in strips of 4 tile rows
    const int nt = a.tiles_m * a.tiles_n;
    int id = blockIdx.x;
    {
        const int per = nt >> 3, rest = nt & 7, x = id & 7, q = id >> 3;
        id = x * per + min(x, rest) + q;
    }
    const int strip = id / (4 * a.tiles_n), in = id - strip * 4 * a.tiles_n;
    const int h_strip = min(4, a.tiles_m - strip * 4);
    const int m0 = (strip * 4 + in % h_strip) * BM, n0 = (in / h_strip) * BN;
    const int k0 = blockIdx.y * a.k_split, k_len = min(a.K - k0, a.k_split);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave / WC) * WM, wn = (wave % WC) * WN;

    OA oa;
    OB ob;
    oa.init(a.A, a.lda, m0, a.ra, k0, tid);
    ob.init(a.B, a.ldb, n0, a.rb, k0, tid);
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // f32: every 512 k the running sums are added to a second set, so that no sum of K products is one chain of K / 2
    // additions (at K = 8192 the error of y fell from 1.9e-6 to below the 8.6e-7 of a library product)
    constexpr bool FOLD = sizeof(T) == 4;
    f32x16 far[FOLD ? TI : 1][FOLD ? TJ : 1];
    if constexpr (FOLD) {
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) far[i][j] = acc[i][j];
    }
    const int stages = (k_len + BK - 1) / BK, full = k_len / BK;
    auto issue = [&](int st) {
        char* base = lds + (st & 1) * STAGE;
        if (st < full) {
            oa.template issue<true>(base, 0);
            ob.template issue<true>(base + OA::BYTES, 0);
        } else {
            oa.template issue<false>(base, k_len - st * BK);
            ob.template issue<false>(base + OA::BYTES, k_len - st * BK);
        }
    };
    frag fa[2][TI], fb[2][TJ];
    auto read = [&](int st, int s, int into) {
        const char* base = lds + (st & 1) * STAGE;
#pragma unroll
        for (int i = 0; i < TI; ++i) fa[into][i] = OA::frag(base, wm + i * 32, s, lane);
#pragma unroll
        for (int j = 0; j < TJ; ++j) fb[into][j] = OB::frag(base + OA::BYTES, wn + j * 32, s, lane);
    };
    auto multiply = [&](int from) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) mma32(acc[i][j], fa[from][i], fb[from][j]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto fold = [&](int st) {
        if constexpr (FOLD) {
            if ((st & 15) == 15) {
#pragma unroll
                for (int i = 0; i < TI; ++i)
#pragma unroll
                    for (int j = 0; j < TJ; ++j)
#pragma unroll
                        for (int e = 0; e < 16; ++e) { far[i][j][e] += acc[i][j][e]; acc[i][j][e] = 0.f; }
            }
        }
    };
    // the border between stage st and st + 1: this wave's reads of st have arrived and so has its part of st + 1; behind
    // the barrier that holds for every wave, so st + 1 may be read and st overwritten
    auto border = [&]() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
    };
    constexpr int L = OA::NL + OB::NL;
    issue(0);
    if (stages > 1) {
        issue(1);
        if (stages - 1 < full || stages > 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(L) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");       // (a partial stage may take fewer loads)
    } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read(0, 0, 0);
    int st = 0;
    for (; st + 2 < full; ++st) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (s < NS - 1) {
                read(st, s + 1, (s + 1) & 1);
            } else {
                border();
                read(st + 1, 0, (s + 1) & 1);
                char* base = lds + (st & 1) * STAGE;
                oa.template issue<true>(base, 0);
                ob.template issue<true>(base + OA::BYTES, 0);
            }
            multiply(s & 1);
        }
        fold(st);
    }
    for (; st < stages; ++st) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (s < NS - 1) {
                read(st, s + 1, (s + 1) & 1);
            } else if (st + 1 < stages) {
                border();
                read(st + 1, 0, (s + 1) & 1);
                if (st + 2 < stages) issue(st + 2);
            }
            multiply(s & 1);
        }
        fold(st);
    }
    if constexpr (FOLD) {
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] += far[i][j][e];
    }
    // epilogue: 32 x WN blocks through LDS, so that a lane ends up with 8 consecutive columns
    __syncthreads();
    char* ep = lds + wave * 32 * EP;
    constexpr int LPR = WN / 8, RPP = 64 / LPR;                    // lanes per row, rows per pass
    const int l31 = lane & 31, h = lane >> 5, cl = (lane % LPR) * 8, rl = lane / LPR;
    const int n = n0 + wn + cl;
    const bool whole = a.vec && n + 8 <= a.N;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                *(float*)(ep + ((e & 3) + 8 * (e >> 2) + 4 * h) * EP + (j * 32 + l31) * 4) = acc[i][j][e];
        // (the region is this wave's own: its LDS accesses complete in order)
#pragma unroll 1
        for (int r = 0; r < 32; r += RPP) {
            const int m = m0 + wm + i * 32 + r + rl;
            float v[8];
            load8<float>((const float*)(ep + (r + rl) * EP + cl * 4), v);
            if (m >= a.M || n >= a.N) continue;
            if (a.slab) {
                float* o = a.slab + ((size_t)blockIdx.y * a.M + m) * a.N + n;
                if (n + 8 <= a.N && (a.N & 3) == 0) store8<float>(o, v);
                else
                    for (int j = 0; j < 8; ++j)
                        if (n + j < a.N) o[j] = v[j];
            } else {
                emit8<T>(a.e, m, n, a.N, whole, v);
            }
        }
    }
}

// sums the slabs of a split contraction in order and applies the epilogue: 8 columns per thread
template <typename T>
__global__ void __launch_bounds__(256) slab_sum(const GemmArgs a, int splits) {
    const int n8 = (a.N + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.M * n8) return;
    const int m = (int)(i / n8), n = (int)(i % n8) * 8;
    const float* p = a.slab + (size_t)m * a.N + n;
    const size_t stride = (size_t)a.M * a.N;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n + 8 <= a.N && (a.N & 3) == 0) {
        for (int z = 0; z < splits; ++z) {
            float q[8];
            load8<float>(p + z * stride, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += q[j];
        }
    } else {
        for (int z = 0; z < splits; ++z)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < a.N) v[j] += p[z * stride + j];
    }
    emit8<T>(a.e, m, n, a.N, a.vec && n + 8 <= a.N, v);
}

// Rows that do not start on 16-byte borders (or are no whole number of 16 bytes long) are copied to padded rows first:
// [rows][width] at pitch ld -> [rows][round_up(width, 8)], zeros behind.  One read and one write of an operand that the
// product reads several times.
template <typename T>
__global__ void __launch_bounds__(256) pad_rows(const T* __restrict__ in, size_t ld, T* __restrict__ out, int rows, int width, int out_ld) {
    const int n8 = out_ld / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)rows * n8) return;
    const int r = (int)(i / n8), c = (int)(i % n8) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < width ? to_f32(in[(size_t)r * ld + c + j]) : 0.f;
    store8<T>(out + (size_t)r * out_ld + c, v);
}

// dz = dy act'(pre), rounded to T, into padded rows (zeros behind the N columns), and column sums of the unrounded values
// over blocks of `rows_blk` rows.  A thread owns 8 columns; 32 column chunks by 8 row lanes per workgroup.
template <typename T, typename P>
__global__ void __launch_bounds__(256) dz_colsum(const T* __restrict__ dy, size_t dy_ld, const P* __restrict__ pre, size_t pre_ld,
                                                 T* dz, int dz_ld, float* part, int M, int N, int act, int rows_blk, int vec) {
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ float sm[8][264];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = (blockIdx.x * 32 + cl) * 8;
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 0.f;
    if (c < N) {
        const bool whole = vec && c + 8 <= N;
        const int64_t r1 = min((int64_t)M, ((int64_t)blockIdx.y + 1) * rows_blk);
        for (int64_t r = (int64_t)blockIdx.y * rows_blk + rl; r < r1; r += 8) {
            float g[8], q[8];
            const T* gp = dy + (size_t)r * dy_ld + c;
            const P* qp = pre + (size_t)r * pre_ld + c;
            if (whole) {
                load8<T>(gp, g);
                if (act != CVG_ACT_NONE) load8<P>(qp, q);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    g[j] = c + j < N ? to_f32(gp[j]) : 0.f;
                    q[j] = act != CVG_ACT_NONE && c + j < N ? to_f32(qp[j]) : 0.f;
                }
            }
            if (act != CVG_ACT_NONE) {
                act_slope8<EXACT>(q, act);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = c + j < N ? g[j] * q[j] : 0.f;
            }
            if (dz) store8<T>(dz + (size_t)r * dz_ld + c, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += g[j];
        }
    }
    if (!part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sm[rl][cl * 8 + j] = s[j];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= N) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sm[i][threadIdx.x];
    part[(size_t)blockIdx.y * N + col] = t;
}
// [P][N] -> column sums: 32 columns by 8 row lanes
__global__ void __launch_bounds__(256) sum_rows(const float* __restrict__ part, int P, int N, float* out) {
    __shared__ float sm[8][32];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
    float s = 0.f;
    if (c < N)
        for (int i = rl; i < P; i += 8) s += part[(size_t)i * N + c];
    sm[rl][cl] = s;
    __syncthreads();
    if (rl || c >= N) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sm[i][cl];
    out[c] = s;
}

__global__ void __launch_bounds__(256) zero_rows(char* out, size_t pitch, int rows, int width, int es) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)rows * width) return;
    char* q = out + (size_t)(i / width) * pitch + (size_t)(i % width) * es;
    if (es == 4) *(float*)q = 0.f; else *(bf16*)q = (bf16)0.f;
}

// ---- host side ---------------------------------------------------------------------------------------------
size_t es_of(int dtype) { return dtype == CVG_BF16 ? 2 : 4; }
size_t ld_of(int ld, int width) { return (size_t)(ld ? ld : width); }
size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }
size_t max_sz(size_t a, size_t b) { return a > b ? a : b; }

// the tile kernel's lane offsets span 256 rows in 31 bits
constexpr int MAX_WIDTH = 2000000;
constexpr size_t MAX_PITCH = ((size_t)1 << 31) / 256 - 64;       // bytes

int check(const cvg_linear_desc* d, const char* who) {
    CVG_CHECK(d, "%s: null descriptor", who);
    CVG_CHECK(d->dtype == CVG_F32 || d->dtype == CVG_BF16, "%s: dtype %d", who, d->dtype);
    CVG_CHECK(d->dw_dtype == CVG_F32 || d->dw_dtype == d->dtype, "%s: dw_dtype %d", who, d->dw_dtype);
    CVG_CHECK(d->pre_dtype == CVG_F32 || d->pre_dtype == d->dtype, "%s: pre_dtype %d", who, d->pre_dtype);
    CVG_CHECK(d->M >= 0 && d->N >= 1 && d->K >= 1, "%s: M %d, N %d, K %d", who, d->M, d->N, d->K);
    CVG_CHECK(d->M <= 0x7fffff00 && d->N <= MAX_WIDTH && d->K <= MAX_WIDTH, "%s: M %d, N %d, K %d", who, d->M, d->N, d->K);
    CVG_CHECK(act_known(d->act), "%s: activation %d", who, d->act);
    const int ld[8] = {d->x_ld, d->w_ld, d->dx_ld, d->dw_ld, d->y_ld, d->res_ld, d->pre_ld, d->dy_ld};
    for (int i = 0; i < 8; ++i)
        CVG_CHECK(ld[i] == 0 || ld[i] >= (i < 4 ? d->K : d->N), "%s: pitch %d below the row length %d", who, ld[i], i < 4 ? d->K : d->N);
    const int64_t m = ceil_div(d->M, 64), n = ceil_div(d->N, 64), k = ceil_div(d->K, 64);
    CVG_CHECK(m * n <= 0x1000000 && m * k <= 0x1000000 && n * k <= 0x1000000, "%s: too many tiles", who);
    return 0;
}

// Tile and number of K ranges for one product.  The estimate is in MFMA cycles of one CU: a stage (128 bytes of k) of a
// BM x BN tile takes `mfma` cycles of its matrix units, never less than the load latency a two-stage pipeline leaves
// exposed; workgroups beyond one round queue up; K ranges add their f32 slabs (written and read once at ~2000 bytes per
// cycle chip-wide) and a launch.
struct Tile { int cfg, splits, k_split; };
struct TileShape { int bm, bn, occ; double mfma; };
Tile choose(int dtype, int64_t M, int64_t N, int64_t K) {
    static const TileShape bf[3] = {{256, 256, 1, 2048 / .8}, {128, 128, 2, 512 / .6}, {64, 64, 4, 128 / .4}};
    static const TileShape f3[3] = {{0, 0, 0, 0}, {128, 128, 2, 4096 / .85}, {64, 64, 3, 1024 / .7}};
    const TileShape* sh = dtype == CVG_BF16 ? bf : f3;
    const int bk = dtype == CVG_BF16 ? 64 : 32;
    const int64_t stages = (K + bk - 1) / bk;
    Tile best{2, 1, (int)round_up(K, bk)};
    double best_t = 1e300;
    for (int c = 0; c < 3; ++c) {
        if (!sh[c].bm) continue;
        const int64_t tiles = ((M + sh[c].bm - 1) / sh[c].bm) * ((N + sh[c].bn - 1) / sh[c].bn);
        for (int64_t sp = 1; sp <= 64; sp *= 2) {
            const int64_t per = (stages + sp - 1) / sp;
            if (sp > 1 && (per < 2 || tiles * sp > 2048)) break;
            const int64_t real = (stages + per - 1) / per;             // ranges that hold any k
            const int64_t wgs = tiles * real, per_cu = (wgs + 255) / 256;
            const int64_t rounds = (per_cu + sh[c].occ - 1) / sh[c].occ;
            const int64_t together = per_cu < sh[c].occ ? per_cu : sh[c].occ;
            double stage = sh[c].mfma * together;
            if (stage < 700) stage = 700;
            double t = rounds * (per * stage + 4000);
            if (real > 1) t += 6000 + (double)real * M * N * 8 / 2000;
            if (t < best_t) { best_t = t; best = Tile{c, (int)real, (int)(per * bk)}; }
        }
    }
    return best;
}
size_t slab_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
    if (M == 0 || N == 0 || K == 0) return 0;                    // (no rows: nothing is multiplied)
    const Tile t = choose(dtype, M, N, K);
    return t.splits > 1 ? (size_t)t.splits * M * N * 4 : 0;
}

template <typename T, int BM, int BN, int WR, int WC>
void launch_tile(GemmArgs& a, bool acol, bool bcol, int splits, hipStream_t s) {
    a.tiles_m = ceil_div(a.M, BM);
    a.tiles_n = ceil_div(a.N, BN);
    const dim3 grid(a.tiles_m * a.tiles_n, splits);
    if (!acol && !bcol) gemm_tile<T, BM, BN, WR, WC, false, false><<<grid, WR * WC * 64, 0, s>>>(a);
    else if (!acol) gemm_tile<T, BM, BN, WR, WC, false, true><<<grid, WR * WC * 64, 0, s>>>(a);
    else gemm_tile<T, BM, BN, WR, WC, true, true><<<grid, WR * WC * 64, 0, s>>>(a);
}

// An operand as the caller holds it: `rows` rows of `width` elements.
struct Rows { const void* p; size_t ld; int64_t rows, width; };
bool fits(const Rows& r, size_t es) { return aligned16(r.p) && r.ld * es % 16 == 0 && r.width * es % 16 == 0 && r.ld * es <= MAX_PITCH; }
size_t padded_bytes(int64_t rows, int64_t width, size_t es) { return round_up((size_t)rows * round_up(width, 8) * es, 256); }

template <typename T>
int pad(Rows& r, char*& ws, hipStream_t s) {
    if (fits(r, sizeof(T))) return 0;
    T* out = (T*)ws;
    ws += padded_bytes(r.rows, r.width, sizeof(T));
    const int ld = (int)round_up(r.width, 8);
    pad_rows<T><<<ceil_div(r.rows * (ld / 8), 256), 256, 0, s>>>((const T*)r.p, r.ld, out, (int)r.rows, (int)r.width, ld);
    CVG_LAUNCH_CHECK();
    r.p = out;
    r.ld = ld;
    r.width = ld;
    return 0;
}

// D = A B^T with A, B fit for the tile kernel; acol / bcol: the operand's rows run along k
template <typename T>
int gemm(const Rows& A, bool acol, const Rows& B, bool bcol, int64_t M, int64_t N, int64_t K, const Epi& e, char* slab, hipStream_t s) {
    GemmArgs a{};
    a.A = A.p; a.B = B.p; a.lda = A.ld; a.ldb = B.ld;
    a.M = (int)M; a.N = (int)N; a.K = (int)K; a.e = e;
    a.ra = (int)(acol ? A.width : A.rows);
    a.rb = (int)(bcol ? B.width : B.rows);
    const size_t oes = e.out_f32 ? 4 : sizeof(T), pes = e.pre_f32 ? 4 : sizeof(T);
    a.vec = aligned16(e.out) && e.out_ld * oes % 16 == 0 && (!e.pre || (aligned16(e.pre) && e.pre_ld * pes % 16 == 0)) &&
            (!e.res || (aligned16(e.res) && e.res_ld * sizeof(T) % 16 == 0)) && aligned16(e.bias);
    const Tile t = choose(Elem<T>::DT, M, N, K);
    a.k_split = t.k_split;
    a.slab = t.splits > 1 ? (float*)slab : nullptr;
    if (t.cfg == 0) {
        if constexpr (sizeof(T) == 2) launch_tile<T, 256, 256, 2, 4>(a, acol, bcol, t.splits, s);
    } else if (t.cfg == 1) {
        launch_tile<T, 128, 128, 2, 2>(a, acol, bcol, t.splits, s);
    } else {
        launch_tile<T, 64, 64, 2, 2>(a, acol, bcol, t.splits, s);
    }
    CVG_LAUNCH_CHECK();
    if (t.splits > 1) {
        slab_sum<T><<<ceil_div(M * ((N + 7) / 8), 256), 256, 0, s>>>(a, t.splits);
        CVG_LAUNCH_CHECK();
    }
    return 0;
}

// Workspaces: padded copies first, then slabs.  The sizes do not depend on pitches or alignment, so one workspace serves
// every call of the same shape.
size_t fwd_ws(const cvg_linear_desc* d) {
    const size_t es = es_of(d->dtype);
    return padded_bytes(d->M, d->K, es) + padded_bytes(d->N, d->K, es) + slab_bytes(d->dtype, d->M, d->N, d->K);
}
int dz_rows_blk(const cvg_linear_desc* d) {
    // about 2048 workgroups where there are rows enough, at least 8 rows each
    const int64_t cols = ceil_div(d->N, 256);
    int64_t blks = 2048 / cols > 0 ? 2048 / cols : 1;
    if (blks > 256) blks = 256;
    const int64_t rb = ceil_div(d->M, blks);
    return (int)(rb < 8 ? 8 : round_up(rb, 8));
}
size_t part_bytes(const cvg_linear_desc* d) { return round_up((size_t)ceil_div(d->M, dz_rows_blk(d)) * d->N * 4, 256); }
size_t bwd_ws(const cvg_linear_desc* d) {
    const size_t es = es_of(d->dtype);
    return padded_bytes(d->M, d->N, es) + part_bytes(d) + padded_bytes(d->N, d->K, es) + padded_bytes(d->M, d->K, es) +
           max_sz(slab_bytes(d->dtype, d->M, d->K, d->N), slab_bytes(d->dtype, d->N, d->K, d->M));
}

template <typename T>
int forward(const cvg_linear_desc* d, const void* x, const void* w, const float* bias, const void* res, void* y, void* pre, char* ws,
            hipStream_t s) {
    Rows X{x, ld_of(d->x_ld, d->K), d->M, d->K}, W{w, ld_of(d->w_ld, d->K), d->N, d->K};
    if (pad<T>(X, ws, s) != 0 || pad<T>(W, ws, s) != 0) return -1;
    Epi e{};
    e.bias = bias; e.res = res; e.pre = pre; e.out = y; e.act = d->act;
    e.out_f32 = 0; e.pre_f32 = sizeof(T) == 2 && d->pre_dtype == CVG_F32;
    e.res_ld = ld_of(d->res_ld, d->N); e.pre_ld = ld_of(d->pre_ld, d->N); e.out_ld = ld_of(d->y_ld, d->N);
    return gemm<T>(X, false, W, false, d->M, d->N, d->K, e, ws, s);
}

template <typename T, typename P>
int backward(const cvg_linear_desc* d, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw,
             float* dbias, char* ws, hipStream_t s) {
    Rows G{dy, ld_of(d->dy_ld, d->N), d->M, d->N};
    const bool act = d->act != CVG_ACT_NONE, products = (dx || dw) && d->M > 0;
    const bool copy = products && (act || !fits(G, sizeof(T)));
    if (d->M > 0 && (dbias || copy)) {
        const int rb = dz_rows_blk(d), blks = ceil_div(d->M, rb);
        const size_t pld = ld_of(d->pre_ld, d->N);
        T* dz = copy ? (T*)ws : nullptr;
        ws += copy ? padded_bytes(d->M, d->N, sizeof(T)) : 0;
        float* part = dbias ? (float*)ws : nullptr;
        ws += dbias ? part_bytes(d) : 0;
        const int vec = aligned16(dy) && G.ld * sizeof(T) % 16 == 0 && (!act || (aligned16(pre) && pld * sizeof(P) % 16 == 0));
        const int dz_ld = (int)round_up(d->N, 8);
        dz_colsum<T, P><<<dim3(ceil_div(d->N, 256), blks), 256, 0, s>>>((const T*)dy, G.ld, (const P*)pre, pld, dz, dz_ld, part, d->M,
                                                                      d->N, d->act, rb, vec);
        CVG_LAUNCH_CHECK();
        if (dbias) {
            sum_rows<<<ceil_div(d->N, 32), 256, 0, s>>>(part, blks, d->N, dbias);
            CVG_LAUNCH_CHECK();
        }
        if (copy) { G.p = dz; G.ld = dz_ld; G.width = dz_ld; }
    } else if (dbias) {
        sum_rows<<<ceil_div(d->N, 32), 256, 0, s>>>(nullptr, 0, d->N, dbias);
        CVG_LAUNCH_CHECK();
    }
    if (dx && d->M > 0) {
        Rows W{w, ld_of(d->w_ld, d->K), d->N, d->K};
        char* at = ws;
        if (pad<T>(W, at, s) != 0) return -1;
        Epi e{};
        e.out = dx; e.out_ld = ld_of(d->dx_ld, d->K);
        if (gemm<T>(G, false, W, true, d->M, d->K, d->N, e, at, s) != 0) return -1;
    }
    if (dw) {
        Epi e{};
        e.out = dw; e.out_ld = ld_of(d->dw_ld, d->K); e.out_f32 = sizeof(T) == 2 && d->dw_dtype == CVG_F32;
        if (d->M == 0) {
            // no rows: the sum is zero
            zero_rows<<<ceil_div((int64_t)d->N * d->K, 256), 256, 0, s>>>((char*)dw, e.out_ld * (d->dw_dtype == CVG_F32 ? 4 : 2), d->N, d->K,
                                                                          d->dw_dtype == CVG_F32 ? 4 : 2);
            CVG_LAUNCH_CHECK();
            return 0;
        }
        Rows X{x, ld_of(d->x_ld, d->K), d->M, d->K};
        char* at = ws;
        if (pad<T>(X, at, s) != 0) return -1;
        if (gemm<T>(G, true, X, true, d->N, d->K, d->M, e, at, s) != 0) return -1;
    }
    return 0;
}

}  // namespace

extern "C" {

size_t cvg_linear_act_workspace(const cvg_linear_desc* d, int32_t backward) {
    if (check(d, "linear_act_workspace") != 0) return 0;
    return backward ? max_sz(fwd_ws(d), bwd_ws(d)) : fwd_ws(d);
}

int cvg_linear_act_fwd(const cvg_linear_desc* d, const void* x, const void* w, const float* bias, const void* res,
                       void* y, void* pre, void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "linear_act_fwd") != 0) return -1;
    if (d->M == 0) return 0;
    CVG_CHECK(x && w && y, "linear_act_fwd: null tensor");
    const size_t es = es_of(d->dtype);
    const void* ps[4] = {x, w, y, res};
    for (const void* p : ps) CVG_CHECK((uintptr_t)p % es == 0, "linear_act_fwd: misaligned tensor");
    CVG_CHECK((uintptr_t)pre % es_of(d->pre_dtype) == 0 && (uintptr_t)bias % 4 == 0, "linear_act_fwd: misaligned tensor");
    const size_t need = fwd_ws(d);
    CVG_CHECK(ws && ws_bytes >= need && aligned16(ws), "linear_act_fwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    hipStream_t st = (hipStream_t)s;
    return d->dtype == CVG_BF16 ? forward<bf16>(d, x, w, bias, res, y, pre, (char*)ws, st)
                                : forward<float>(d, x, w, bias, res, y, pre, (char*)ws, st);
}

int cvg_linear_act_bwd(const cvg_linear_desc* d, const void* dy, const void* x, const void* w, const void* pre,
                       void* dx, void* dw, float* dbias, void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "linear_act_bwd") != 0) return -1;
    CVG_CHECK(d->M == 0 || dy, "linear_act_bwd: null dy");
    CVG_CHECK(d->M == 0 || !dx || w, "linear_act_bwd: dx needs w");
    CVG_CHECK(d->M == 0 || !dw || x, "linear_act_bwd: dw needs x");
    CVG_CHECK(d->M == 0 || d->act == CVG_ACT_NONE || pre, "linear_act_bwd: an activation needs pre");
    const size_t es = es_of(d->dtype);
    const void* ps[4] = {dy, x, w, dx};
    for (const void* p : ps) CVG_CHECK((uintptr_t)p % es == 0, "linear_act_bwd: misaligned tensor");
    CVG_CHECK((uintptr_t)pre % es_of(d->pre_dtype) == 0 && (uintptr_t)dbias % 4 == 0, "linear_act_bwd: misaligned tensor");
    CVG_CHECK((uintptr_t)dw % es_of(d->dw_dtype) == 0, "linear_act_bwd: misaligned dw");
    const size_t need = bwd_ws(d);
    CVG_CHECK(ws && ws_bytes >= need && aligned16(ws), "linear_act_bwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    hipStream_t st = (hipStream_t)s;
    char* w0 = (char*)ws;
    if (d->dtype == CVG_F32) return backward<float, float>(d, dy, x, w, pre, dx, dw, dbias, w0, st);
    if (d->pre_dtype == CVG_F32) return backward<bf16, float>(d, dy, x, w, pre, dx, dw, dbias, w0, st);
    return backward<bf16, bf16>(d, dy, x, w, pre, dx, dw, dbias, w0, st);
}

}
