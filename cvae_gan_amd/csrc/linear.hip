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
// accesses there.  Bias and residual are loaded by the caller (zeros where there are none), well before they are needed.
__device__ __forceinline__ void load_bias8(const Epi& e, int n, int n_end, bool whole, float (&b)[8]) {
    if (e.bias && whole) {
        load8<float>(e.bias + n, b);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = e.bias && n + j < n_end ? e.bias[n + j] : 0.f;
}
template <typename T>
__device__ __forceinline__ void load_res8(const Epi& e, int m, int n, int n_end, bool whole, float (&q)[8]) {
    const T* r = (const T*)e.res + (size_t)m * e.res_ld + n;
    if (whole) {
        load8<T>(r, q);
    } else if (n + 8 <= n_end) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = to_f32(r[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = n + j < n_end ? to_f32(r[j]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void emit8(const Epi& e, int m, int n, int n_end, bool whole, float (&v)[8], const float (&b)[8], const float (&q)[8]) {
    constexpr bool EXACT = sizeof(T) == 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
    if (e.pre) {
        if (whole) {
            if (e.pre_f32) store8<float>((float*)e.pre + (size_t)m * e.pre_ld + n, v);
            else store8<T>((T*)e.pre + (size_t)m * e.pre_ld + n, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < n_end) {
                    if (e.pre_f32) ((float*)e.pre)[(size_t)m * e.pre_ld + n + j] = v[j];
                    else ((T*)e.pre)[(size_t)m * e.pre_ld + n + j] = from_f32<T>(v[j]);
                }
        }
    }
    act_value8<EXACT>(v, e.act);
    if (e.res)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += q[j];
    if (whole) {
        if (e.out_f32) store8<float>((float*)e.out + (size_t)m * e.out_ld + n, v);
        else store8<T>((T*)e.out + (size_t)m * e.out_ld + n, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < n_end) {
                if (e.out_f32) ((float*)e.out)[(size_t)m * e.out_ld + n + j] = v[j];
                else ((T*)e.out)[(size_t)m * e.out_ld + n + j] = from_f32<T>(v[j]);
            }
    }
}

// D[m][n] = sum_k A(m, k) B(n, k) for one output tile, or one K range of it.
struct GemmArgs {
    const void *A, *B;
    size_t lda, ldb;                 // elements between consecutive m (n) where k is contiguous, between consecutive k otherwise
    int M, N, K;
    int ra, rb;                      // rows of A and B that may be addressed (the padded count where k is strided)
    int tiles_m, tiles_n, k_split;   // k_split: K range of one grid.y slice (a multiple of the K step)
    int fast;                        // `vec`, whole 8-column groups only, and pitches that Streams takes
    int vec;                         // every tensor of the epilogue takes 16-byte accesses at multiples of 8 columns
    float* slab;                     // [splits][M][N] partial sums instead of the epilogue, or null
    Epi e;
};

typedef __attribute__((address_space(3))) void* lds_dst;

// One operand of the tile kernel: ROWS rows of the output dimension, BK = 128 bytes of k per stage.
//   k contiguous (COL = false): LDS holds [ROWS][128 bytes]; the 16-byte chunk c of row r lies at c ^ (r >> 1 & 7).  A
//     16-byte LDS read is served 16 lanes at a time ({0-3, 12-15, 20-27}, {4-11, 16-19, 28-31} and the same of the upper
//     half) over 64 banks of 4 bytes: the 16 rows of a group are 8 even and 8 odd ones, two rows fill the banks once, and
//     r >> 1 takes all 8 values in each half.  (c ^ (r & 7) collides two by two: 45 % of the LDS cycles of a 256 x 256 tile.)
//   k strided (COL = true): LDS holds [BK][ROWS]; bf16 fragments come out of ds_read_b64_tr_b16 (TrLoad), whose lanes read
//     8 k-rows of 64 bytes at once; 64-byte block b of k-row k lies at b ^ (k & 3 | (k >> 3 & 1) << 2) (as many bits as there
//     are blocks), which spreads those rows over the banks.  f32 reads single dwords, 32 columns of k-rows k and k + 8 at
//     once: the upper one's 128-byte blocks are exchanged in pairs.
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
        if constexpr (!COL) return (((o >> 4) ^ (o >> 8)) & 7) * (16 / ES);
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
                const int cs = ES == 2 ? (((c >> 2) ^ swz(k)) << 2) | (c & 3) : c ^ (k & 8);
                int g = cs * (16 / ES);
                if (row0 + g >= rows) g = 0;                      // (rows is a multiple of the chunk)
                off[i] = (int)((size_t)k * ld * ES) + g * ES;
            }
        }
    }
    // load i of a stage.  FULL: the whole stage lies inside the k range; otherwise it is zero from k_left on
    template <bool FULL> __device__ __forceinline__ void load(char* lds, int i, int k_left) {
#ifdef __HIP_DEVICE_COMPILE__
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
        char* to = lds + (i * NWAVES + wave) * 1024;
        if (FULL || k_of(i) < k_left)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_dst)to, 16, off[i], 0, 0, 0);
        else
            *(u32x4*)(to + (tid & 63) * 16) = u32x4{0, 0, 0, 0};
#endif
        if (i == NL - 1) base += step;
    }
    // the same by way of registers: fetch has the load under way, put writes it to LDS
    template <bool FULL> __device__ __forceinline__ u32x4 fetch(int i, int k_left) {
        u32x4 v = {0, 0, 0, 0};
#ifdef __HIP_DEVICE_COMPILE__
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
        if (FULL || k_of(i) < k_left) v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off[i], 0, 0));
#endif
        if (i == NL - 1) base += step;
        return v;
    }
    __device__ __forceinline__ void put(char* lds, int i, u32x4 v) const {
        *(u32x4*)(lds + (i * NWAVES + wave) * 1024 + (tid & 63) * 16) = v;
    }
    // fragment of rows r0 .. r0 + 31, k-step s (16 values: slot (h, j) = k 8 h + j)
    __device__ __forceinline__ static typename Elem<T>::frag frag(const char* lds, int r0, int s, int lane) {
        const int l31 = lane & 31, h = lane >> 5;
        if constexpr (!COL) {
            const char* q = lds + (r0 + l31) * 128;
            const int f = (l31 >> 1) & 7;
            if constexpr (ES == 2) {
                return *(const bf16x8*)(q + (((2 * s + h) ^ f) << 4));
            } else {
                const f32x4 a = *(const f32x4*)(q + (((4 * s + 2 * h) ^ f) << 4));
                const f32x4 b = *(const f32x4*)(q + (((4 * s + 2 * h + 1) ^ f) << 4));
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
                for (int j = 0; j < 8; ++j) r[j] = *(const float*)(lds + (16 * s + 8 * h + j) * RB + ((r0 + l31) ^ (h << 5)) * 4);
                return r;
            }
        }
    }
};

// The tensors of the epilogue as buffers at the corner of a tile, addressed by row and by this lane's 8 columns.
__device__ __forceinline__ u32x4 buf_load(const char* p, int bytes, int off) {
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000), off, 0, 0));
#else
    return u32x4{0, 0, 0, 0};
#endif
}
__device__ __forceinline__ void buf_store(char* p, int bytes, int off, u32x4 v) {
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_buffer_store_b128(v, __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000), off, 0, 0);
#endif
}
struct Stream {
    char* p;
    int bytes, pitch, col;
    // `present`: the tensor exists; pitches are at most MAX_PITCH, so offsets inside 256 rows stay below 2^31
    __device__ __forceinline__ void init(const void* base, bool present, size_t ld, int es, size_t m0, int n0, int c) {
        p = (char*)base + (m0 * ld + n0) * es;
        bytes = present ? 0x7fffffff : 0;
        pitch = (int)(ld * es);
        col = c * es;
    }
    __device__ __forceinline__ int at(int row, bool ok) const { return ok ? row * pitch + col : -1; }
    __device__ __forceinline__ void store_f32(int row, bool ok, const float (&v)[8]) const {
        const int o = at(row, ok);
        buf_store(p, bytes, o, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
        buf_store(p, bytes, ok ? o + 16 : o, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
    }
    __device__ __forceinline__ void store_bf16(int row, bool ok, const float (&v)[8]) const {
        bf16x8 r;
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = (bf16)v[j];
        buf_store(p, bytes, at(row, ok), __builtin_bit_cast(u32x4, r));
    }
};
template <typename T> struct Streams {
    static constexpr bool B = sizeof(T) == 2;
    static constexpr int NV = B ? 1 : 2;                           // 16-byte pieces of 8 elements
    Stream res, pre32, out32, pre16, out16;
    int act;
    __device__ __forceinline__ Streams(const GemmArgs& a, int slice, int m0, int n0, int c) {
        const bool slab = a.slab != nullptr;
        res.init(a.e.res, !slab && a.e.res, a.e.res_ld, sizeof(T), m0, n0, c);
        pre32.init(a.e.pre, !slab && a.e.pre && (!B || a.e.pre_f32), a.e.pre_ld, 4, m0, n0, c);
        if (slab) out32.init(a.slab + (size_t)slice * a.M * a.N, true, a.N, 4, m0, n0, c);
        else out32.init(a.e.out, !B || a.e.out_f32, a.e.out_ld, 4, m0, n0, c);
        if constexpr (B) {
            pre16.init(a.e.pre, !slab && a.e.pre && !a.e.pre_f32, a.e.pre_ld, 2, m0, n0, c);
            out16.init(a.e.out, !slab && !a.e.out_f32, a.e.out_ld, 2, m0, n0, c);
        }
        act = slab ? CVG_ACT_NONE : a.e.act;
    }
    __device__ __forceinline__ void load(u32x4 (&q)[NV], int row, bool ok) const {
        const int o = res.at(row, ok);
        q[0] = buf_load(res.p, res.bytes, o);
        if constexpr (!B) q[1] = buf_load(res.p, res.bytes, ok ? o + 16 : o);
    }
    __device__ __forceinline__ void emit(float (&v)[8], const float (&bias)[8], const u32x4 (&q)[NV], int row, bool ok) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += bias[j];
        pre32.store_f32(row, ok, v);
        if constexpr (B) pre16.store_bf16(row, ok, v);
        act_value8<!B>(v, act);
        float r[8];
        raw_f32(__builtin_bit_cast(Raw8<T>, q), r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
        out32.store_f32(row, ok, v);
        if constexpr (B) out16.store_bf16(row, ok, v);
    }
};

// Tile kernel: BM x BN per workgroup of 2 x 2 waves, 128 bytes of k per LDS stage.  Fragments are read one 16-k step ahead
// of the MFMAs that use them, across the stage border too, so the one barrier of a stage sits between the last fragment
// reads of a stage and the MFMAs on them.
//   256 x 256 (bf16): a wave holds 128 x 128 sums, which needs the least LDS traffic per MFMA (8 fragments for 16 MFMAs; 64 x
//     128 sums of eight waves need 6 for 8, and then the LDS is busy as long as the matrix units).  Its operands come by way
//     of registers, a stage ahead of the LDS: fetching straight to LDS keeps the LDS busy for longer than writing 128 bytes
//     a cycle does (8192 x 4096 x 4096 dw: staging alone takes 140 us, fragment reads alone 91, both together 221; the
//     product with its 161 us of MFMAs 322).  dw 250 us (1100 TFLOP/s; 237 at best), dx 262, forward with f32 pre and residual 284.
//   128 x 128 and 64 x 64: two or three workgroups share a CU; direct-to-LDS loads (550 x 8192 x 528 17 us, 26 by registers).  Two LDS stages
//     of 32 KB or three of 16: 512 x 4096 x 4096 by small tiles takes 31.9 us with two, 26.9 with three, 27.3 with four,
//     550 x 8192 x 528 in f32 47.8, 48.7 and 51.5.
//   Where an operand's rows run along k, bf16 comes by way of registers at every tile: the compiler lets a transposing LDS
//     read wait for every load to LDS under way (2048 x 2048 x 2048: dx 51 us with, 26 without).
template <typename T, int BM, bool COL> constexpr bool by_registers() { return BM == 256 || (sizeof(T) == 2 && COL); }
template <typename T, int BM, bool COL> constexpr int ring() { return BM == 64 && !by_registers<T, BM, COL>() ? 3 : 2; }
template <typename T, int BM, int BN, bool COL> struct TileLds {
    static constexpr int STAGES = ring<T, BM, COL>() * (BM + BN) * 128, EPI = 4 * 32 * (BN / 2 * 4 + 16);
    static constexpr int BYTES = STAGES > EPI ? STAGES : EPI;
};
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
template <typename T, int BM, int BN, bool ACOL, bool BCOL>
__device__ __forceinline__ void tile_body(const GemmArgs& a, int id, int slice, char* lds) {
    constexpr int NW = 4, WM = BM / 2, WN = BN / 2, TI = WM / 32, TJ = WN / 32;
    typedef Operand<T, BM, NW, ACOL> OA;
    typedef Operand<T, BN, NW, BCOL> OB;
    typedef typename Elem<T>::frag frag;
    constexpr int BK = OA::BK, NS = BK / 16;
    constexpr int STAGE = OA::BYTES + OB::BYTES, D = ring<T, BM, ACOL || BCOL>();
    constexpr bool REGS = by_registers<T, BM, ACOL || BCOL>();
    constexpr int EP = WN * 4 + 16;                                // epilogue: 32 rows of the wave's columns, f32
    // workgroups go round-robin over the 8 dies, each with its own L2: give every die a run of neighbouring tiles, walked
    // in strips of 4 tile rows
    const int nt = a.tiles_m * a.tiles_n;
    {
        const int per = nt >> 3, rest = nt & 7, x = id & 7, q = id >> 3;
        id = x * per + min(x, rest) + q;
    }
    const int strip = id / (4 * a.tiles_n), in = id - strip * 4 * a.tiles_n;
    const int h_strip = min(4, a.tiles_m - strip * 4);
    const int m0 = (strip * 4 + in % h_strip) * BM, n0 = (in / h_strip) * BN;
    const int k0 = slice * a.k_split, k_len = min(a.K - k0, a.k_split);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * WM, wn = (wave & 1) * WN;

    // this lane's columns in the epilogue; their bias is on its way while the products are taken
    constexpr int LPR = WN / 8, RPP = 64 / LPR, PASSES = 32 / RPP;      // lanes per row, rows per pass
    const int cl = (lane % LPR) * 8, rl = lane / LPR, n = n0 + wn + cl;
    const bool whole = a.vec && n + 8 <= a.N;
    float bias[8];
    load_bias8(a.e, n, a.N, whole, bias);
    if (a.slab) {
#pragma unroll
        for (int j = 0; j < 8; ++j) bias[j] = 0.f;
    }

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
    constexpr int L = OA::NL + OB::NL, R = TI + TJ, MF = TI * TJ, H = MF > 1 ? MF / 2 : 1, HL = MF / 2;
    // loads lo .. hi - 1 of a stage's L, straight to LDS
    auto load = [&](auto whole_stage, int buf, int lo, int hi, int k_left) {
        constexpr bool F = decltype(whole_stage)::value;
        char* base = lds + buf * STAGE;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            if (i < lo || i >= hi) continue;
            if (i < OA::NL) oa.template load<F>(base, i, k_left);
            else ob.template load<F>(base + OA::BYTES, i - OA::NL, k_left);
        }
    };
    auto issue = [&](int st, int buf) {
        if (st < full) load(Yes{}, buf, 0, L, 0);
        else load(No{}, buf, 0, L, k_len - st * BK);
    };
    // fragments lo .. hi - 1 of the R of k-step s
    frag fa[2][TI], fb[2][TJ];
    auto read = [&](int buf, int s, int into, int lo, int hi) {
        const char* base = lds + buf * STAGE;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i < lo || i >= hi) continue;
            if (i < TI) fa[into][i] = OA::frag(base, wm + i * 32, s, lane);
            else fb[into][i - TI] = OB::frag(base + OA::BYTES, wn + (i - TI) * 32, s, lane);
        }
    };
    // One 16-k step: behind MFMA q on fragment set `from` comes between(q).  An instruction that finds its unit's queue
    // full holds up the wave's MFMAs too, so LDS reads (first half) and loads (second half) are dealt out evenly.  A single
    // MFMA is over before the reads it would hide have arrived: they go first.
    auto step = [&](int from, auto between) {
#pragma unroll
        for (int q = 0; q < MF; ++q) {
            if (MF == 1) between(q);
            __builtin_amdgcn_sched_barrier(0);
            mma32(acc[q / TJ][q % TJ], fa[from][q / TJ], fb[from][q % TJ]);
            __builtin_amdgcn_sched_barrier(0);
            if (MF > 1) between(q);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto deal_reads = [&](int q, int buf, int s, int into) {
        if (q < H) read(buf, s, into, q * R / H, (q + 1) * R / H);
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
    // The border between stage st and st + 1: this wave's reads of st have arrived and so has its part of st + 1; behind
    // the barrier that holds for every wave, so st + 1 may be read and st overwritten.
    constexpr int P = MF > 1 ? L / NS : L;                         // loads per step (short stages: all of them as early as can be)
    static_assert(L % NS == 0, "tile");
    int st = 0, buf = 0;
    if constexpr (REGS) {
        u32x4 hold[L];                                             // stage st + 1 (from step `NS - 1` of st on: st + 2)
        auto fetch = [&](auto whole_stage, int lo, int hi, int k_left) {
            constexpr bool F = decltype(whole_stage)::value;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (i < lo || i >= hi) continue;
                if (i < OA::NL) hold[i] = oa.template fetch<F>(i, k_left);
                else hold[i] = ob.template fetch<F>(i - OA::NL, k_left);
            }
        };
        auto fetch_any = [&](int of, int lo, int hi) {
            if (of < full) fetch(Yes{}, lo, hi, 0);
            else if (of < stages) fetch(No{}, lo, hi, k_len - of * BK);
        };
        auto put = [&](int to, int lo, int hi) {
            char* base = lds + to * STAGE;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (i < lo || i >= hi) continue;
                if (i < OA::NL) oa.put(base, i, hold[i]);
                else ob.put(base + OA::BYTES, i - OA::NL, hold[i]);
            }
        };
        auto border = [&]() {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" : : : "memory");
        };
        // (The long run has its own beginning: behind a branch it would be unknown how many loads are under way, and the
        // first write of every stage would wait for all of them, the youngest too.)
        auto begin = [&](auto long_run) {
            constexpr bool S = decltype(long_run)::value;
            if constexpr (S) fetch(Yes{}, 0, L, 0); else fetch_any(0, 0, L);
            put(0, 0, L);
            if constexpr (S) fetch(Yes{}, 0, L, 0); else fetch_any(1, 0, L);
            border();
            read(0, 0, 0, 0, R);
            if (S || 1 < stages) put(1, 0, P);
            if constexpr (S) fetch(Yes{}, 0, P, 0); else fetch_any(2, 0, P);
        };
        if (full > 3) {
          begin(Yes{});
          for (; st + 3 < full; ++st, buf ^= 1) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const bool last = s == NS - 1;
                if (last) border();
                step(s & 1, [&](int q) {
                    if (last) deal_reads(q, buf ^ 1, 0, 0);
                    else deal_reads(q, buf, s + 1, (s + 1) & 1);
                    const int n = last ? 0 : s + 1;
#pragma unroll
                    for (int i = 0; i < L; ++i)
                        if (q >= HL && i >= n * P + (q - HL) * P / (MF - HL) && i < n * P + (q - HL + 1) * P / (MF - HL)) {
                            put(last ? buf : buf ^ 1, i, i + 1);
                            fetch(Yes{}, i, i + 1, 0);
                        }
                });
            }
          }
        } else {
            begin(No{});
        }
        for (; st < stages; ++st, buf ^= 1) {
#pragma unroll
            for (int s = 0; s < NS - 1; ++s) {
                step(s & 1, [&](int q) { deal_reads(q, buf, s + 1, (s + 1) & 1); });
                if (st + 1 < stages) put(buf ^ 1, (s + 1) * P, (s + 2) * P);
                fetch_any(st + 2, (s + 1) * P, (s + 2) * P);
            }
            border();
            step((NS - 1) & 1, [&](int q) { if (st + 1 < stages) deal_reads(q, buf ^ 1, 0, 0); });
            if (st + 2 < stages) put(buf, 0, P);
            fetch_any(st + 3, 0, P);
        }
    } else {
        // While only whole stages are in flight the D - 2 stages behind st + 1 stay so; a partial one takes an unknown
        // number of loads.
        auto border = [&](auto steady) {
            if constexpr (decltype(steady)::value) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((D - 2) * L) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" : : : "memory");
        };
        // a stage's loads are spread over NS steps, the first P in the last step of the stage whose place they take
        for (int i = 0; i < D - 1 && i < stages; ++i) issue(i, i);
        if (full > D) load(Yes{}, D - 1, 0, P, 0);
        else if (D <= stages) issue(D - 1, D - 1);
        if (full >= D) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((D - 2) * L + P) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
        read(0, 0, 0, 0, R);
        int before = D - 1;
        for (; st + D < full; ++st) {
            const int after = buf + 1 == D ? 0 : buf + 1;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const bool last = s == NS - 1;
                if (last) border(Yes{});
                step(s & 1, [&](int q) {
                    if (last) deal_reads(q, after, 0, 0);
                    else deal_reads(q, buf, s + 1, (s + 1) & 1);
                    const int n = last ? 0 : s + 1;
                    if (q >= HL) load(Yes{}, last ? buf : before, n * P + (q - HL) * P / (MF - HL), n * P + (q - HL + 1) * P / (MF - HL), 0);
                });
            }
            fold(st);
            before = buf;
            buf = after;
        }
        if (st > 0) load(Yes{}, before, P, L, 0);
        for (; st < stages; ++st) {
            const int after = buf + 1 == D ? 0 : buf + 1;
#pragma unroll
            for (int s = 0; s < NS - 1; ++s) step(s & 1, [&](int q) { deal_reads(q, buf, s + 1, (s + 1) & 1); });
            if (st + 1 < stages) {
                border(No{});
                if (st + D < stages) issue(st + D, buf);
            }
            step((NS - 1) & 1, [&](int q) { if (st + 1 < stages) deal_reads(q, after, 0, 0); });
            fold(st);
            buf = after;
        }
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
    const int l31 = lane & 31, h = lane >> 5;
    constexpr int PG = PASSES < 4 ? PASSES : 4;                    // passes whose residual is loaded together
    auto to_lds = [&](int i) {                                     // (the region is this wave's own: its accesses complete in order)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                *(float*)(ep + ((e & 3) + 8 * (e >> 2) + 4 * h) * EP + (j * 32 + l31) * 4) = acc[i][j][e];
    };
    auto from_lds = [&](int pass, float (&v)[8]) { load8<float>((const float*)(ep + (pass * RPP + rl) * EP + cl * 4), v); };
    if (a.fast) {
        // No branch around a memory access: a tensor that is not there has a descriptor of no bytes, a row or column outside
        // the matrix an offset beyond every descriptor.  So the number of accesses between a residual's load and its use is
        // known, and waiting for it waits for no store.
        const Streams<T> io(a, slice, m0, n0, wn + cl);
        u32x4 next[PG][Streams<T>::NV], q[PG][Streams<T>::NV];
        const int row0 = wm + rl, rows = n < a.N ? a.M - m0 : 0;
#pragma unroll
        for (int r = 0; r < PG; ++r) io.load(next[r], row0 + r * RPP, row0 + r * RPP < rows);
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            to_lds(i);
#pragma unroll 1
            for (int r0 = 0; r0 < PASSES; r0 += PG) {
                const int row = row0 + i * 32 + r0 * RPP;
#pragma unroll
                for (int r = 0; r < PG; ++r) {
#pragma unroll
                    for (int k = 0; k < Streams<T>::NV; ++k) q[r][k] = next[r][k];
                    const int rn = row + (PG + r) * RPP;           // (PASSES RPP is 32: behind a block's last group the next block's first)
                    io.load(next[r], rn, rn < rows && rn < wm + WM);
                }
#pragma unroll
                for (int r = 0; r < PG; ++r) {
                    float v[8];
                    from_lds(r0 + r, v);
                    io.emit(v, bias, q[r], row + r * RPP, row + r * RPP < rows);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        to_lds(i);
#pragma unroll 1
        for (int r0 = 0; r0 < PASSES; r0 += PG) {
            const int mb = m0 + wm + i * 32 + r0 * RPP + rl;
            float q[PG][8];
            if (!a.slab && a.e.res && n < a.N) {
#pragma unroll
                for (int r = 0; r < PG; ++r) load_res8<T>(a.e, min(mb + r * RPP, a.M - 1), n, a.N, whole, q[r]);
            }
#pragma unroll
            for (int r = 0; r < PG; ++r) {
                const int m = mb + r * RPP;
                float v[8];
                from_lds(r0 + r, v);
                if (m >= a.M || n >= a.N) continue;
                if (a.slab) {
                    float* o = a.slab + ((size_t)slice * a.M + m) * a.N + n;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (n + j < a.N) o[j] = v[j];
                } else {
                    emit8<T>(a.e, m, n, a.N, whole, v, bias, q[r]);
                }
            }
        }
    }
}

template <typename T, int BM, int BN, bool ACOL, bool BCOL>
__global__ void __launch_bounds__(256) gemm_tile(const GemmArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[TileLds<T, BM, BN, ACOL || BCOL>::BYTES];
    tile_body<T, BM, BN, ACOL, BCOL>(a, blockIdx.x, blockIdx.y, lds);
}

// ---- few rows: M <= 16 ---------------------------------------------------------------------------------------
// The weights are all there is to read.  A workgroup takes 16 of their rows; its eight waves take turns along k, 64 values
// (a whole cache line of a bf16 row) at a time, straight from memory into 16 x 16 MFMA fragments: lane (r, q) holds k
// values 16 q .. 16 q + 15 of the unit, of weight row r and of x row r alike, so any order of k inside the unit is right as
// long as both operands share it.  Units come in two sets, one on its way while the other is multiplied; what lies behind
// K, and x rows beyond M, read as zeros.  The waves' sums meet in LDS in wave order; no second launch, no workspace.
// Bound by memory: one token through 4096 x 4096 bf16, 34 MB, takes 8.0 us (4.2 TB/s), through 16384 x 4096 28 (4.8 TB/s).
template <typename T> struct Unit;                                // 16 consecutive k of one row
template <> struct Unit<bf16> { u32x4 a[2]; };
template <> struct Unit<float> { u32x4 a[4]; };
// `at`: byte offset of the row from base, or -1 for a row of zeros
template <typename T, bool ALIGNED>
__device__ __forceinline__ void unit_load(Unit<T>& u, const char* base, int at, const T* row, int k, int K) {
    constexpr int PER = 16 / sizeof(T), NV = 16 / PER;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int kk = k + i * PER;
        if constexpr (ALIGNED) {                                  // (K is a multiple of 16 bytes)
            u.a[i] = buf_load(base, 0x7fffffff, at >= 0 && kk < K ? at + kk * (int)sizeof(T) : -1);
        } else {
            u.a[i] = u32x4{0, 0, 0, 0};
            if (at >= 0) {
                T t[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) t[j] = kk + j < K ? row[kk + j] : from_f32<T>(0.f);
                u.a[i] = __builtin_bit_cast(u32x4, *(T (*)[PER])t);
            }
        }
    }
}
__device__ __forceinline__ void unit_mma(f32x4& acc, const Unit<bf16>& w, const Unit<bf16>& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.a[i]), __builtin_bit_cast(bf16x8, x.a[i]), acc, 0, 0, 0);
}
__device__ __forceinline__ void unit_mma(f32x4& acc, const Unit<float>& w, const Unit<float>& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.a[i][j]), __uint_as_float(x.a[i][j]), acc, 0, 0, 0);
}
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(512) few_rows(const GemmArgs a) {
    constexpr int U = ALIGNED && sizeof(T) == 2 ? 4 : 2;          // units of a set
    __shared__ float red[8][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4, n0 = blockIdx.x * 16;
    const char* wb = (const char*)((const T*)a.B + (size_t)n0 * a.ldb);
    const int wr = min(r, a.N - 1 - n0);
    const T *w = (const T*)wb + wr * a.ldb, *x = (const T*)a.A + min(r, a.M - 1) * a.lda;
    // (pitches of the aligned form are at most MAX_PITCH)
    const int w_at = ALIGNED ? wr * (int)(a.ldb * sizeof(T)) : 0, x_at = r >= a.M ? -1 : ALIGNED ? r * (int)(a.lda * sizeof(T)) : 0;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    Unit<T> uw[2][U], ux[2][U];
    auto load = [&](int set, int k0) {
#pragma unroll
        for (int u = 0; u < U; ++u) unit_load<T, ALIGNED>(uw[set][u], wb, w_at, w, k0 + u * 512 + q * 16, a.K);
#pragma unroll
        for (int u = 0; u < U; ++u) unit_load<T, ALIGNED>(ux[set][u], (const char*)a.A, x_at, x, k0 + u * 512 + q * 16, a.K);
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int u = 0; u < U; ++u) unit_mma(acc, uw[set][u], ux[set][u]);
    };
    const int k_wave = __builtin_amdgcn_readfirstlane(wave) * 64;
    if (a.K <= 2 * U * 512) {                                     // all of it at once, and nothing that is not there
#pragma unroll
        for (int u = 0; u < 2 * U; ++u)
            if (k_wave + u * 512 < a.K) unit_load<T, ALIGNED>(uw[u / U][u % U], wb, w_at, w, k_wave + u * 512 + q * 16, a.K);
#pragma unroll
        for (int u = 0; u < 2 * U; ++u)
            if (k_wave + u * 512 < a.K) unit_load<T, ALIGNED>(ux[u / U][u % U], (const char*)a.A, x_at, x, k_wave + u * 512 + q * 16, a.K);
#pragma unroll
        for (int u = 0; u < 2 * U; ++u)
            if (k_wave + u * 512 < a.K) unit_mma(acc, uw[u / U][u % U], ux[u / U][u % U]);
    } else {
        int k0 = k_wave;
        load(0, k0);
        load(1, k0 + U * 512);
        for (; k0 + 2 * U * 512 < a.K; k0 += 2 * U * 512) {
            multiply(0);
            load(0, k0 + 2 * U * 512);
            multiply(1);
            load(1, k0 + 3 * U * 512);
        }
        multiply(0);
        multiply(1);
    }
    // lane (r, q): x row r, weight rows 4 q .. 4 q + 3
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][r][4 * q + i] = acc[i];
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int n = threadIdx.x & 15, m = threadIdx.x >> 4;
    if (m >= a.M || n0 + n >= a.N) return;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v += red[j][m][n];
    emit<T>(a.e, m, n0 + n, v);
}

// column sums of [P][N] partial rows: 32 columns by `blockDim / 32` row lanes
__device__ __forceinline__ void sum_rows_body(const float* __restrict__ part, int P, int N, float* out, int blk, float (*sm)[32]) {
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, lanes = blockDim.x >> 5, c = blk * 32 + cl;
    float s = 0.f;
    if (c < N) {
#pragma unroll 8
        for (int i = rl; i < P; i += lanes) s += part[(size_t)i * N + c];
    }
    sm[rl][cl] = s;
    __syncthreads();
    if (rl || c >= N) return;
    s = 0.f;
    for (int i = 0; i < lanes; ++i) s += sm[i][cl];
    out[c] = s;
}
struct SumArgs { const float* part; float* out; int P, N; };

// Both gradients of a layer in one launch: neither waits for the other, small ones do not fill the chip alone, and a
// launch costs as much as they do.  The first blocks finish the bias gradient; the product with the longer range of k goes
// ahead of the other, so that what starts last is over soonest.
template <typename T, int BM, int BN>
__global__ void __launch_bounds__(256) gemm_pair(const GemmArgs dx, const GemmArgs dw, int blocks_dx, int blocks_dw, int blocks_db, const SumArgs db) {
    __shared__ __attribute__((aligned(1024))) char lds[TileLds<T, BM, BN, true>::BYTES];
    int blk = blockIdx.x - blocks_db;
    if (blk < 0) {
        sum_rows_body(db.part, db.P, db.N, db.out, blockIdx.x, (float (*)[32])lds);
        return;
    }
    const bool dw_first = dw.k_split > dx.k_split, is_dw = dw_first ? blk < blocks_dw : blk >= blocks_dx;
    if (is_dw != dw_first) blk -= dw_first ? blocks_dw : blocks_dx;
    if (is_dw) {
        const int nt = dw.tiles_m * dw.tiles_n, slice = blk / nt;
        tile_body<T, BM, BN, true, true>(dw, blk - slice * nt, slice, lds);
    } else {
        const int nt = dx.tiles_m * dx.tiles_n, slice = blk / nt;
        tile_body<T, BM, BN, false, true>(dx, blk - slice * nt, slice, lds);
    }
}
__global__ void __launch_bounds__(256) sum_rows(const SumArgs a) {
    __shared__ float sm[8][32];
    sum_rows_body(a.part, a.P, a.N, a.out, blockIdx.x, sm);
}

// Sums the slabs of a split contraction and applies the epilogue.  A thread owns 8 columns of one row and one of zl runs
// of consecutive slabs (few outputs would leave most of the chip idle otherwise); the runs are added in order.
template <typename T>
__device__ __forceinline__ void slab_sum_body(const GemmArgs& a, int splits, int zl, int blk, float (*sm)[8]) {
    const int n8 = (a.N + 7) / 8, per_blk = 256 / zl, lo = threadIdx.x % per_blk, zi = threadIdx.x / per_blk;
    const int64_t i = (int64_t)blk * per_blk + lo;
    const bool live = i < (int64_t)a.M * n8;
    const int m = live ? (int)(i / n8) : 0, n = live ? (int)(i % n8) * 8 : 0;
    const float* p = a.slab + (size_t)m * a.N + n;
    const size_t stride = (size_t)a.M * a.N;
    const int run = (splits + zl - 1) / zl, z1 = min(splits, (zi + 1) * run);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
        if (n + 8 <= a.N && (a.N & 3) == 0) {
#pragma unroll 4
            for (int z = zi * run; z < z1; ++z) {
                float q[8];
                load8<float>(p + z * stride, q);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += q[j];
            }
        } else {
#pragma unroll 2
            for (int z = zi * run; z < z1; ++z)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (n + j < a.N) v[j] += p[z * stride + j];
        }
    }
    if (zl > 1) {
        store8<float>(sm[threadIdx.x], v);
        __syncthreads();
        if (zi) return;
        for (int q = 1; q < zl; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += sm[q * per_blk + lo][j];
    }
    if (!live) return;
    const bool whole = a.vec && n + 8 <= a.N;
    float b[8], q8[8];
    load_bias8(a.e, n, a.N, whole, b);
    if (a.e.res) load_res8<T>(a.e, m, n, a.N, whole, q8);
    emit8<T>(a.e, m, n, a.N, whole, v, b, q8);
}
struct SlabJob { GemmArgs a; int splits, zl, blocks; };
template <typename T>
__global__ void __launch_bounds__(256) slab_sum(const SlabJob one, const SlabJob two) {
    __shared__ __attribute__((aligned(16))) float sm[256][8];
    if ((int)blockIdx.x < one.blocks) slab_sum_body<T>(one.a, one.splits, one.zl, blockIdx.x, sm);
    else slab_sum_body<T>(two.a, two.splits, two.zl, blockIdx.x - one.blocks, sm);
}

// Rows that do not start on 16-byte borders (or are no whole number of 16 bytes long) are copied to padded rows first:
// [rows][width] at pitch ld -> [rows][round_up(width, 8)], zeros behind.  One read and one write of an operand that the
// product reads several times.
template <typename T>
__device__ __forceinline__ void pad_body(const void* in, size_t ld, void* out, int rows, int width, int out_ld, int blk) {
    const int n8 = out_ld / 8;
    const int64_t i = (int64_t)blk * 256 + threadIdx.x;
    if (i >= (int64_t)rows * n8) return;
    const int r = (int)(i / n8), c = (int)(i % n8) * 8;
    const T* q = (const T*)in + (size_t)r * ld + c;
    float v[8];
    if (c + 8 <= width) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f32(q[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < width ? to_f32(q[j]) : 0.f;
    }
    store8<T>((T*)out + (size_t)r * out_ld + c, v);
}
struct PadJob { const void* in; void* out; size_t ld; int rows, width, out_ld, blocks; };

// dz = dy act'(pre), rounded to T, into padded rows (zeros behind the N columns), and column sums of the unrounded values
// over blocks of `rows_blk` rows.  A thread owns 8 columns; 32 column chunks by 8 row lanes per workgroup.
// What the rounding took away (but for infinities and NaN, which the first part carries alone) makes a second operand where
// the caller wants a weight gradient of f32: the two parts together are off by at most 2^-16 instead of 2^-8.
struct DzJob {
    const void *dy, *pre;
    void* dz;                        // or null
    void* lo;                        // what dz lacks, laid out like it, or null
    float* part;                     // or null
    size_t dy_ld, pre_ld;
    int dz_ld, M, N, act, rows_blk, vec, col_blocks, blocks;
};
template <typename T, typename P>
__device__ __forceinline__ void dz_body(const DzJob& a, int blk, float (*sm)[264]) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int U = 4;             // rows in flight per thread
    const int by = blk / a.col_blocks, bx = blk - by * a.col_blocks;
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = (bx * 32 + cl) * 8;
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 0.f;
    if (c < a.N) {
        const bool whole = a.vec && c + 8 <= a.N;
        const int64_t r1 = min((int64_t)a.M, ((int64_t)by + 1) * a.rows_blk);
        for (int64_t r0 = (int64_t)by * a.rows_blk + rl; r0 < r1; r0 += 8 * U) {
            float g[U][8], q[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (8 * u >= a.rows_blk) break;           // (few rows a block: no loads for rows that are not there)
                const int64_t r = min(r0 + 8 * u, r1 - 1);
                const T* gp = (const T*)a.dy + (size_t)r * a.dy_ld + c;
                const P* qp = (const P*)a.pre + (size_t)r * a.pre_ld + c;
                if (whole) {
                    load8<T>(gp, g[u]);
                    if (a.act != CVG_ACT_NONE) load8<P>(qp, q[u]);
                } else if (c + 8 <= a.N) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        g[u][j] = to_f32(gp[j]);
                        if (a.act != CVG_ACT_NONE) q[u][j] = to_f32(qp[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        g[u][j] = c + j < a.N ? to_f32(gp[j]) : 0.f;
                        q[u][j] = a.act != CVG_ACT_NONE && c + j < a.N ? to_f32(qp[j]) : 0.f;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + 8 * u;
                if (r >= r1) break;
                if (a.act != CVG_ACT_NONE) {
                    act_slope8<EXACT>(q[u], a.act);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[u][j] = c + j < a.N ? g[u][j] * q[u][j] : 0.f;
                }
                if (a.dz) store8<T>((T*)a.dz + (size_t)r * a.dz_ld + c, g[u]);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] += g[u][j];
                if (a.lo) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float left = g[u][j] - to_f32(from_f32<T>(g[u][j]));
                        g[u][j] = fabsf(left) < INFINITY ? left : 0.f;
                    }
                    store8<T>((T*)a.lo + (size_t)r * a.dz_ld + c, g[u]);
                }
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sm[rl][cl * 8 + j] = s[j];
    __syncthreads();
    const int col = bx * 256 + threadIdx.x;
    if (col >= a.N) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sm[i][threadIdx.x];
    a.part[(size_t)by * a.N + col] = t;
}

// What has to happen before the products, in one launch: dz and the bias gradient's partial sums, padded copies.  Bound by
// memory: 8192 x 4096 from bf16 dy and f32 pre, 268 MB in 62 us (4.3 TB/s).
template <typename T, typename P>
__global__ void __launch_bounds__(256) prepare(const DzJob dz, const PadJob p0, const PadJob p1) {
    __shared__ float sm[8][264];
    int blk = blockIdx.x;
    if (blk < dz.blocks) { dz_body<T, P>(dz, blk, sm); return; }
    blk -= dz.blocks;
    if (blk < p0.blocks) pad_body<T>(p0.in, p0.ld, p0.out, p0.rows, p0.width, p0.out_ld, blk);
    else pad_body<T>(p1.in, p1.ld, p1.out, p1.rows, p1.width, p1.out_ld, blk - p0.blocks);
}

__global__ void __launch_bounds__(256) zero_rows(char* out, size_t pitch, int rows, int width, int es) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * width; i += (int64_t)gridDim.x * 256) {
        char* q = out + (size_t)(i / width) * pitch + (size_t)(i % width) * es;
        if (es == 4) *(float*)q = 0.f; else *(bf16*)q = (bf16)0.f;
    }
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
    CVG_CHECK(m * n < 0x400000 && m * k < 0x400000 && n * k < 0x400000, "%s: too many tiles", who);   // (a launch has fewer than 2^32 threads)
    return 0;
}

// Tile and number of K ranges for one product.  The estimate is in MFMA cycles of one CU: a stage (128 bytes of k) of a
// BM x BN tile takes `mfma` cycles of its matrix units, never less than the load latency a two-stage pipeline leaves
// exposed; workgroups beyond one round queue up; K ranges add their f32 slabs (written and read once at ~2000 bytes per
// cycle chip-wide) and a launch.  Forward bf16, us by 256 x 256 / 128 x 128 / 64 x 64 tiles:
//   4096 x 4096 x 4096  116 / 131 / 203    2048 x 2048 x 2048  46 / 28 / 29    8192 x 1024 x 1024  35 / 23 / 29
//   3000 x 3000 x 1000   39 /  41 /  46     512 x 4096 x 4096  45 / 35 / 27     550 x 8192 x  528  26 / 15 / 16
// (The estimate counts two workgroups of 64 x 64 tiles a CU, where three run since their LDS has three stages: counting
// three left the times of these sizes, of 1000 x 1000 x 2056, 256 x 8192 x 1024 and of f32 as they are.)
// f32, whose MFMAs take eight times as long and need no more bytes, always takes 64 x 64: 128 x 128 measured 1114 against
// 986 us at 4096 x 4096 x 4096, 217 against 148 at 3000 x 3000 x 1000.
struct Tile { int cfg, splits, k_split; double t; };
struct TileShape { int bm, bn, occ; double mfma; };
const TileShape TILES[2][3] = {{{0, 0, 0, 0}, {0, 0, 0, 0}, {64, 64, 2, 1024 / .7}},
                               {{256, 256, 1, 2048 / .8}, {128, 128, 2, 512 / .6}, {64, 64, 2, 128 / .4}}};
Tile choose_split(int dtype, int c, int64_t M, int64_t N, int64_t K) {
    const TileShape& sh = TILES[dtype == CVG_BF16][c];
    const int bk = dtype == CVG_BF16 ? 64 : 32;
    const int64_t stages = (K + bk - 1) / bk;
    Tile best{c, 1, (int)round_up(K, bk), 1e300};
    const int64_t tiles = ((M + sh.bm - 1) / sh.bm) * ((N + sh.bn - 1) / sh.bn);
    // The bf16 matrix instruction cuts off what lies below the last bits of a sum that has grown large beside its products, and
    // cuts downwards, by some 1e-3 of the sum's last bit each: of K terms in ranges of L, sqrt(K L) times 1 to 3e-12 of the norm.  2^28 rows
    // in 64 ranges put every element of dw too low, by 1e-4; at most 2^18 terms a range hold that to 2e-5 there and to 1e-6 at
    // 2^20 rows.  (f32 sums start again every 512 k.)
    const int64_t most = dtype == CVG_BF16 ? (1 << 18) / bk : stages, least = (stages + most - 1) / most;
    for (int64_t sp = least; sp == least || sp <= 64; sp *= 2) {
        const int64_t per = (stages + sp - 1) / sp;
        if (sp > least && (per < 2 || tiles * sp > 2048)) break;
        const int64_t real = (stages + per - 1) / per;                 // ranges that hold any k
        const int64_t wgs = tiles * real, per_cu = (wgs + 255) / 256;
        const int64_t rounds = (per_cu + sh.occ - 1) / sh.occ;
        const int64_t together = per_cu < sh.occ ? per_cu : sh.occ;
        double stage = sh.mfma * together;
        if (stage < 700) stage = 700;
        double t = rounds * (per * stage + 4000);
        if (real > 1) t += 6000 + (double)real * M * N * 8 / 2000;
        if (t < best.t) best = Tile{c, (int)real, (int)(per * bk), t};
    }
    return best;
}
Tile choose(int dtype, int64_t M, int64_t N, int64_t K) {
    Tile best{2, 1, 0, 1e301};
    for (int c = dtype == CVG_BF16 ? 0 : 2; c < 3; ++c) {
        const Tile t = choose_split(dtype, c, M, N, K);
        if (t.t < best.t) best = t;
    }
    return best;
}
// Both gradients with one tile shape in one launch, or (cfg 0) apart
struct PairPlan { bool together; Tile dx, dw; };
PairPlan choose_pair(const cvg_linear_desc* d) {
    PairPlan p{false, choose(d->dtype, d->M, d->K, d->N), choose(d->dtype, d->N, d->K, d->M)};
    if (p.dx.cfg == 0 || p.dw.cfg == 0) return p;
    p.together = true;
    if (p.dx.cfg != p.dw.cfg) {
        const Tile a = choose_split(d->dtype, p.dw.cfg, d->M, d->K, d->N), b = choose_split(d->dtype, p.dx.cfg, d->N, d->K, d->M);
        if (a.t + p.dw.t < b.t + p.dx.t) p.dx = a; else p.dw = b;
    }
    return p;
}
size_t slab_of(const Tile& t, int64_t M, int64_t N) { return t.splits > 1 ? round_up((size_t)t.splits * M * N * 4, 256) : 0; }

template <typename T, int BM, int BN>
void launch_tile(GemmArgs& a, bool acol, bool bcol, int splits, hipStream_t s) {
    const dim3 grid(a.tiles_m * a.tiles_n, splits);
    if (!acol && !bcol) gemm_tile<T, BM, BN, false, false><<<grid, 256, 0, s>>>(a);
    else if (!acol) gemm_tile<T, BM, BN, false, true><<<grid, 256, 0, s>>>(a);
    else gemm_tile<T, BM, BN, true, true><<<grid, 256, 0, s>>>(a);
}

// An operand as the caller holds it: `rows` rows of `width` elements.
struct Rows { const void* p; size_t ld; int64_t rows, width; };
bool fits(const Rows& r, size_t es) { return aligned16(r.p) && r.ld * es % 16 == 0 && r.width * es % 16 == 0 && r.ld * es <= MAX_PITCH; }
size_t padded_bytes(int64_t rows, int64_t width, size_t es) { return round_up((size_t)rows * round_up(width, 8) * es, 256); }

template <typename T>
PadJob pad_job(Rows& r, char*& ws) {
    PadJob j{};
    if (fits(r, sizeof(T))) return j;
    j.in = r.p; j.ld = r.ld; j.out = ws; j.rows = (int)r.rows; j.width = (int)r.width; j.out_ld = (int)round_up(r.width, 8);
    j.blocks = ceil_div(r.rows * (j.out_ld / 8), 256);
    ws += padded_bytes(r.rows, r.width, sizeof(T));
    r.p = j.out; r.ld = j.out_ld; r.width = j.out_ld;
    return j;
}

// D = A B^T with A, B fit for the tile kernel; acol / bcol: the operand's rows run along k
template <typename T>
GemmArgs gemm_args(const Rows& A, bool acol, const Rows& B, bool bcol, int64_t M, int64_t N, int64_t K, const Epi& e, const Tile& t, char*& ws) {
    GemmArgs a{};
    a.A = A.p; a.B = B.p; a.lda = A.ld; a.ldb = B.ld;
    a.M = (int)M; a.N = (int)N; a.K = (int)K; a.e = e;
    a.ra = (int)(acol ? A.width : A.rows);
    a.rb = (int)(bcol ? B.width : B.rows);
    const size_t oes = e.out_f32 ? 4 : sizeof(T), pes = e.pre_f32 ? 4 : sizeof(T);
    a.vec = aligned16(e.out) && e.out_ld * oes % 16 == 0 && (!e.pre || (aligned16(e.pre) && e.pre_ld * pes % 16 == 0)) &&
            (!e.res || (aligned16(e.res) && e.res_ld * sizeof(T) % 16 == 0)) && aligned16(e.bias);
    const TileShape& sh = TILES[sizeof(T) == 2][t.cfg];
    a.tiles_m = ceil_div(M, sh.bm);
    a.tiles_n = ceil_div(N, sh.bn);
    a.k_split = t.k_split;
    a.slab = t.splits > 1 ? (float*)ws : nullptr;
    a.fast = N % 8 == 0 && (a.slab ? (size_t)N * 4 <= MAX_PITCH
                                   : a.vec && e.out_ld * oes <= MAX_PITCH && (!e.pre || e.pre_ld * pes <= MAX_PITCH) &&
                                         (!e.res || e.res_ld * sizeof(T) <= MAX_PITCH));
    ws += slab_of(t, M, N);
    return a;
}
template <typename T>
SlabJob slab_job(const GemmArgs& a, const Tile& t) {
    SlabJob j{};
    if (t.splits <= 1) return j;
    j.a = a;
    j.splits = t.splits;
    const int64_t outs = (int64_t)a.M * ((a.N + 7) / 8);
    j.zl = 1;
    while (j.zl < 16 && outs * j.zl < 131072 && t.splits >= 4 * j.zl) j.zl *= 2;
    j.blocks = ceil_div(outs, 256 / j.zl);
    return j;
}
template <typename T>
int sum_slabs(const SlabJob& one, const SlabJob& two, hipStream_t s) {
    if (one.blocks + two.blocks == 0) return 0;
    slab_sum<T><<<one.blocks + two.blocks, 256, 0, s>>>(one, two);
    CVG_LAUNCH_CHECK();
    return 0;
}
template <typename T>
int product(GemmArgs& a, bool acol, bool bcol, const Tile& t, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (t.cfg == 0) launch_tile<T, 256, 256>(a, acol, bcol, t.splits, s);
        else if (t.cfg == 1) launch_tile<T, 128, 128>(a, acol, bcol, t.splits, s);
    }
    if (t.cfg == 2) launch_tile<T, 64, 64>(a, acol, bcol, t.splits, s);
    CVG_LAUNCH_CHECK();
    return 0;
}
template <typename T>
int multiply(GemmArgs& a, bool acol, bool bcol, const Tile& t, hipStream_t s) {
    if (product<T>(a, acol, bcol, t, s) != 0) return -1;
    return sum_slabs<T>(slab_job<T>(a, t), SlabJob{}, s);
}

// Few rows: every workgroup of few_rows reads all of x, from 17 rows on more than its weights (32 rows of 4096 x 4096 bf16:
// 15.8 us, 14.0 by tiles).  Long rows of few weights leave most CUs without one of its workgroups, and a product split
// along k is faster in spite of its second launch (16 rows, us by few_rows / by tiles, bf16):
//   1024 x 8192 16.2 / 10.1    2048 x 8192 18.0 / 13.5    1024 x 4096 9.2 / 9.0    1024 x 2048 5.7 / 8.8    2048 x 2048 6.0 / 8.7
// and f32: 1024 x 4096 16.6 / 12.9, 1024 x 2048 9.9 / 10.5.
bool takes_few_rows(const cvg_linear_desc* d) { return d->M <= 16 && (d->K * es_of(d->dtype) <= 8192 || d->N > 2048); }

// Workspaces: dz, partial column sums, padded copies, slabs.  The sizes do not depend on pitches or alignment, so one
// workspace serves every call of the same shape.
size_t fwd_ws(const cvg_linear_desc* d) {
    if (d->M == 0 || takes_few_rows(d)) return 0;
    const size_t es = es_of(d->dtype);
    return padded_bytes(d->M, d->K, es) + padded_bytes(d->N, d->K, es) + slab_of(choose(d->dtype, d->M, d->N, d->K), d->M, d->N);
}
int dz_rows_blk(const cvg_linear_desc* d) {
    // about 2048 workgroups where there are rows enough, at most 128 rows of partial sums, at least 8 rows each
    const int64_t cols = ceil_div(d->N, 256);
    int64_t blks = 2048 / cols > 0 ? 2048 / cols : 1;
    if (blks > 128) blks = 128;
    const int64_t rb = ceil_div(d->M, blks);
    return (int)(rb < 32 ? round_up(rb, 8) : round_up(rb, 32));
}
// An f32 weight gradient of bf16 data behind an activation is taken with both parts of dz (a rounded dz alone leaves it the
// accuracy of bf16): a second product over the same rows of x, whose partial sums are slabs of their own.  Both gradients of
// 8192 x 4096 x 4096 take 859 us and dw is off by 2.5e-6 of its norm; with dw in bf16 586 us and 2.35e-3.
bool two_parts(const cvg_linear_desc* d) { return d->dtype == CVG_BF16 && d->act != CVG_ACT_NONE && d->dw_dtype == CVG_F32; }
Tile with_parts(const Tile& t, int parts) { return Tile{t.cfg, t.splits * parts, t.k_split, t.t}; }
size_t part_bytes(const cvg_linear_desc* d) { return round_up((size_t)ceil_div(d->M, dz_rows_blk(d)) * d->N * 4, 256); }
size_t bwd_ws(const cvg_linear_desc* d) {
    if (d->M == 0) return 0;
    const size_t es = es_of(d->dtype);
    const PairPlan p = choose_pair(d);
    const int parts = two_parts(d) ? 2 : 1;
    return parts * padded_bytes(d->M, d->N, es) + part_bytes(d) + padded_bytes(d->N, d->K, es) + padded_bytes(d->M, d->K, es) +
           slab_of(p.dx, d->M, d->K) + slab_of(with_parts(p.dw, parts), d->N, d->K);
}

template <typename T>
int forward(const cvg_linear_desc* d, const void* x, const void* w, const float* bias, const void* res, void* y, void* pre, char* ws,
            hipStream_t s) {
    Rows X{x, ld_of(d->x_ld, d->K), d->M, d->K}, W{w, ld_of(d->w_ld, d->K), d->N, d->K};
    Epi e{};
    e.bias = bias; e.res = res; e.pre = pre; e.out = y; e.act = d->act;
    e.out_f32 = 0; e.pre_f32 = sizeof(T) == 2 && d->pre_dtype == CVG_F32;
    e.res_ld = ld_of(d->res_ld, d->N); e.pre_ld = ld_of(d->pre_ld, d->N); e.out_ld = ld_of(d->y_ld, d->N);
    if (takes_few_rows(d)) {
        GemmArgs a{};
        a.A = X.p; a.B = W.p; a.lda = X.ld; a.ldb = W.ld; a.M = d->M; a.N = d->N; a.K = d->K; a.e = e;
        const bool al = fits(X, sizeof(T)) && fits(W, sizeof(T));
        const int blocks = ceil_div(d->N, 16);
        if (al) few_rows<T, true><<<blocks, 512, 0, s>>>(a); else few_rows<T, false><<<blocks, 512, 0, s>>>(a);
        CVG_LAUNCH_CHECK();
        return 0;
    }
    const PadJob p0 = pad_job<T>(X, ws), p1 = pad_job<T>(W, ws);
    if (p0.blocks + p1.blocks) {
        prepare<T, T><<<p0.blocks + p1.blocks, 256, 0, s>>>(DzJob{}, p0, p1);
        CVG_LAUNCH_CHECK();
    }
    const Tile t = choose(Elem<T>::DT, d->M, d->N, d->K);
    GemmArgs a = gemm_args<T>(X, false, W, false, d->M, d->N, d->K, e, t, ws);
    return multiply<T>(a, false, false, t, s);
}

// M > 0
template <typename T, typename P>
int backward(const cvg_linear_desc* d, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw,
             float* dbias, char* ws, hipStream_t s) {
    Rows G{dy, ld_of(d->dy_ld, d->N), d->M, d->N};
    const bool act = d->act != CVG_ACT_NONE, products = dx || dw;
    const bool copy = products && (act || !fits(G, sizeof(T))), two = dw && two_parts(d);
    DzJob z{};
    SumArgs sum{};
    if (dbias || copy) {
        z.dy = dy; z.dy_ld = G.ld; z.pre = pre; z.pre_ld = ld_of(d->pre_ld, d->N);
        z.M = d->M; z.N = d->N; z.act = d->act; z.dz_ld = (int)round_up(d->N, 8);
        z.rows_blk = dz_rows_blk(d);
        z.col_blocks = ceil_div(d->N, 256);
        z.blocks = z.col_blocks * ceil_div(d->M, z.rows_blk);
        z.vec = aligned16(dy) && G.ld * sizeof(T) % 16 == 0 && (!act || (aligned16(pre) && z.pre_ld * sizeof(P) % 16 == 0));
        if (copy) {
            z.dz = ws;
            ws += padded_bytes(d->M, d->N, sizeof(T));
            G.p = z.dz; G.ld = z.dz_ld; G.width = z.dz_ld;
            if (two) {
                z.lo = ws;
                ws += padded_bytes(d->M, d->N, sizeof(T));
            }
        }
        if (dbias) {
            z.part = (float*)ws;
            ws += part_bytes(d);
            sum.part = z.part; sum.out = dbias; sum.N = d->N; sum.P = ceil_div(d->M, z.rows_blk);
        }
    }
    Rows W{w, ld_of(d->w_ld, d->K), d->N, d->K}, X{x, ld_of(d->x_ld, d->K), d->M, d->K};
    const PadJob p0 = dx ? pad_job<T>(W, ws) : PadJob{}, p1 = dw ? pad_job<T>(X, ws) : PadJob{};
    if (z.blocks + p0.blocks + p1.blocks) {
        prepare<T, P><<<z.blocks + p0.blocks + p1.blocks, 256, 0, s>>>(z, p0, p1);
        CVG_LAUNCH_CHECK();
    }
    const PairPlan plan = choose_pair(d);
    Epi ex{}, ew{};
    ex.out = dx; ex.out_ld = ld_of(d->dx_ld, d->K);
    ew.out = dw; ew.out_ld = ld_of(d->dw_ld, d->K); ew.out_f32 = sizeof(T) == 2 && d->dw_dtype == CVG_F32;
    GemmArgs ax = gemm_args<T>(G, false, W, true, d->M, d->K, d->N, ex, plan.dx, ws);
    const Tile dw_all = with_parts(plan.dw, two ? 2 : 1);
    GemmArgs aw = gemm_args<T>(G, true, X, true, d->N, d->K, d->M, ew, dw_all, ws);
    GemmArgs lo = aw;                                              // (two: the slabs behind those of the first part)
    lo.A = z.lo;
    if (two) lo.slab += (size_t)plan.dw.splits * d->N * d->K;
    const int sum_blocks = dbias ? ceil_div(d->N, 32) : 0;
    if (plan.together && products) {
        const int bx = dx ? ax.tiles_m * ax.tiles_n * plan.dx.splits : 0, bw = dw ? aw.tiles_m * aw.tiles_n * plan.dw.splits : 0;
        if constexpr (sizeof(T) == 2) {
            if (plan.dx.cfg == 1) gemm_pair<T, 128, 128><<<bx + bw + sum_blocks, 256, 0, s>>>(ax, aw, bx, bw, sum_blocks, sum);
        }
        if (plan.dx.cfg == 2) gemm_pair<T, 64, 64><<<bx + bw + sum_blocks, 256, 0, s>>>(ax, aw, bx, bw, sum_blocks, sum);
        CVG_LAUNCH_CHECK();
        if (two && product<T>(lo, true, true, plan.dw, s) != 0) return -1;
        return sum_slabs<T>(dx ? slab_job<T>(ax, plan.dx) : SlabJob{}, dw ? slab_job<T>(aw, dw_all) : SlabJob{}, s);
    }
    if (sum_blocks) {
        sum_rows<<<sum_blocks, 256, 0, s>>>(sum);
        CVG_LAUNCH_CHECK();
    }
    if (dx && multiply<T>(ax, false, true, plan.dx, s) != 0) return -1;
    if (two && product<T>(lo, true, true, plan.dw, s) != 0) return -1;
    if (dw && product<T>(aw, true, true, plan.dw, s) != 0) return -1;
    return dw ? sum_slabs<T>(slab_job<T>(aw, dw_all), SlabJob{}, s) : 0;
}

// no rows: the sums are zero
int backward_empty(const cvg_linear_desc* d, void* dw, float* dbias, hipStream_t s) {
    const int es = d->dw_dtype == CVG_F32 ? 4 : 2;
    const int64_t dw_blocks = ((int64_t)d->N * d->K + 255) / 256;
    if (dw) zero_rows<<<(int)(dw_blocks < 65536 ? dw_blocks : 65536), 256, 0, s>>>((char*)dw, ld_of(d->dw_ld, d->K) * es, d->N, d->K, es);
    if (dbias) zero_rows<<<ceil_div(d->N, 256), 256, 0, s>>>((char*)dbias, 0, 1, d->N, 4);
    CVG_LAUNCH_CHECK();
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
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && aligned16(ws)), "linear_act_fwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    CVG_CHECK(apart({y, pre}, {x, w, bias}) && apart({pre}, {res}), "linear_act_fwd: an output over another tensor");
    CVG_CHECK(y != res || ld_of(d->res_ld, d->N) == ld_of(d->y_ld, d->N), "linear_act_fwd: in place with different pitches");
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
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && aligned16(ws)), "linear_act_bwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    CVG_CHECK(apart({dx, dw, dbias}, {dy, x, w, pre}), "linear_act_bwd: a gradient over another tensor");
    hipStream_t st = (hipStream_t)s;
    if (d->M == 0) return backward_empty(d, dw, dbias, st);
    char* w0 = (char*)ws;
    if (d->dtype == CVG_F32) return backward<float, float>(d, dy, x, w, pre, dx, dw, dbias, w0, st);
    if (d->pre_dtype == CVG_F32) return backward<bf16, float>(d, dy, x, w, pre, dx, dw, dbias, w0, st);
    return backward<bf16, bf16>(d, dy, x, w, pre, dx, dw, dbias, w0, st);
}

}
