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
    void* pre;                       // T, or null
    void* out;                       // T, or f32 where out_f32
    size_t res_ld, pre_ld, out_ld;
    int act, out_f32;
};

template <typename T>
__device__ __forceinline__ void emit(const Epi& e, int m, int n, float v) {
    constexpr bool EXACT = sizeof(T) == 4;
    if (e.bias) v += e.bias[n];
    if (e.pre) ((T*)e.pre)[(size_t)m * e.pre_ld + n] = from_f32<T>(v);
    v = act_value<EXACT>(v, e.act);
    if (e.res) v += to_f32(((const T*)e.res)[(size_t)m * e.res_ld + n]);
    if (e.out_f32) ((float*)e.out)[(size_t)m * e.out_ld + n] = v;
    else ((T*)e.out)[(size_t)m * e.out_ld + n] = from_f32<T>(v);
}

struct GemmArgs {
    const void *A, *B;
    size_t am, ak, bn, bk;           // strides of A(m, k) and B(n, k) in elements
    int M, N, K;
    Epi e;
};

// 64 x 64 tile, four waves of one 32 x 32 accumulator each, any strides: operands go through LDS element by element.
template <typename T>
__global__ void __launch_bounds__(256) gemm_any(const GemmArgs a) {
    constexpr int BK = 32, PITCH = BK + 16 / (int)sizeof(T);
    __shared__ __attribute__((aligned(16))) T As[64][PITCH];
    __shared__ __attribute__((aligned(16))) T Bs[64][PITCH];
    const int tiles_n = (a.N + 63) / 64;
    const int m0 = (int)(blockIdx.x / tiles_n) * 64, n0 = (int)(blockIdx.x % tiles_n) * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    f32x16 acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    for (int k0 = 0; k0 < a.K; k0 += BK) {
        for (int i = threadIdx.x; i < 64 * BK; i += 256) {
            // consecutive threads along whichever direction is contiguous in memory
            const int ra = a.ak == 1 ? i / BK : i % 64, ka = a.ak == 1 ? i % BK : i / 64;
            const int rb = a.bk == 1 ? i / BK : i % 64, kb = a.bk == 1 ? i % BK : i / 64;
            T va = from_f32<T>(0.f), vb = va;
            if (m0 + ra < a.M && k0 + ka < a.K) va = ((const T*)a.A)[(size_t)(m0 + ra) * a.am + (size_t)(k0 + ka) * a.ak];
            if (n0 + rb < a.N && k0 + kb < a.K) vb = ((const T*)a.B)[(size_t)(n0 + rb) * a.bn + (size_t)(k0 + kb) * a.bk];
            As[ra][ka] = va;
            Bs[rb][kb] = vb;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < BK / 16; ++s) {
            typename Elem<T>::frag fa = *(const typename Elem<T>::frag*)&As[wm + l31][s * 16 + 8 * h];
            typename Elem<T>::frag fb = *(const typename Elem<T>::frag*)&Bs[wn + l31][s * 16 + 8 * h];
            mma32(acc, fa, fb);
        }
        __syncthreads();
    }
    const int n = n0 + wn + l31;
    if (n >= a.N) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int m = m0 + wm + (i & 3) + 8 * (i >> 2) + 4 * h;
        if (m < a.M) emit<T>(a.e, m, n, acc[i]);
    }
}

// dz = dy act'(pre) rounded to T (where dz is wanted) and column sums of the unrounded values over 64-row blocks
template <typename T>
__global__ void __launch_bounds__(256) dz_colsum(const T* __restrict__ dy, size_t dy_ld, const T* __restrict__ pre, size_t pre_ld,
                                                 T* dz, size_t dz_ld, float* part, int M, int N, int act) {
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ float sm[4][64];
    const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6, c = blockIdx.x * 64 + cl;
    float s = 0.f;
    if (c < N) {
        const int r1 = min(M, ((int)blockIdx.y + 1) * 64);
        for (int r = blockIdx.y * 64 + rl; r < r1; r += 4) {
            float g = to_f32(dy[(size_t)r * dy_ld + c]);
            if (act != CVG_ACT_NONE) {
                g *= act_slope<EXACT>(to_f32(pre[(size_t)r * pre_ld + c]), act);
                if (dz) dz[(size_t)r * dz_ld + c] = from_f32<T>(g);
            }
            s += g;
        }
    }
    sm[rl][cl] = s;
    __syncthreads();
    if (part && rl == 0 && c < N) part[(size_t)blockIdx.y * N + c] = sm[0][cl] + sm[1][cl] + sm[2][cl] + sm[3][cl];
}
__global__ void __launch_bounds__(256) sum_rows(const float* __restrict__ part, int P, int N, float* out) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float s = 0.f;
    for (int i = 0; i < P; ++i) s += part[(size_t)i * N + c];
    out[c] = s;
}

// ---- host side ---------------------------------------------------------------------------------------------
size_t es_of(int dtype) { return dtype == CVG_BF16 ? 2 : 4; }
size_t ld_of(int ld, int width) { return (size_t)(ld ? ld : width); }
size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

int check(const cvg_linear_desc* d, const char* who) {
    CVG_CHECK(d, "%s: null descriptor", who);
    CVG_CHECK(d->dtype == CVG_F32 || d->dtype == CVG_BF16, "%s: dtype %d", who, d->dtype);
    CVG_CHECK(d->dw_dtype == CVG_F32 || d->dw_dtype == d->dtype, "%s: dw_dtype %d", who, d->dw_dtype);
    CVG_CHECK(d->M >= 0 && d->N >= 1 && d->K >= 1, "%s: M %d, N %d, K %d", who, d->M, d->N, d->K);
    CVG_CHECK(d->M <= 0x7fffff00 && d->N <= 0x7fffff00 && d->K <= 0x7fffff00, "%s: M %d, N %d, K %d", who, d->M, d->N, d->K);
    CVG_CHECK(act_known(d->act), "%s: activation %d", who, d->act);
    const int ld[8] = {d->x_ld, d->w_ld, d->dx_ld, d->dw_ld, d->y_ld, d->res_ld, d->pre_ld, d->dy_ld};
    for (int i = 0; i < 8; ++i)
        CVG_CHECK(ld[i] == 0 || ld[i] >= (i < 4 ? d->K : d->N), "%s: pitch %d below the row length %d", who, ld[i], i < 4 ? d->K : d->N);
    CVG_CHECK((int64_t)ceil_div(d->M, 64) * ceil_div(d->N, 64) <= 0x7fffffff && (int64_t)ceil_div(d->M, 64) * ceil_div(d->K, 64) <= 0x7fffffff &&
              (int64_t)ceil_div(d->N, 64) * ceil_div(d->K, 64) <= 0x7fffffff, "%s: too many tiles", who);
    return 0;
}

template <typename T>
void gemm(const GemmArgs& a, hipStream_t s) {
    const int64_t blocks = (int64_t)ceil_div(a.M, 64) * ceil_div(a.N, 64);
    gemm_any<T><<<(int)blocks, 256, 0, s>>>(a);
}

struct BwdWs { size_t dz, part, total; };
BwdWs bwd_ws(const cvg_linear_desc* d) {
    BwdWs w{};
    w.part = d->act == CVG_ACT_NONE ? 0 : round_up((size_t)d->M * round_up(d->N, 8) * es_of(d->dtype), 256);
    w.total = w.part + (size_t)ceil_div(d->M, 64) * d->N * 4;
    return w;
}

template <typename T>
int backward(const cvg_linear_desc* d, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw,
             float* dbias, char* ws, hipStream_t s) {
    const BwdWs o = bwd_ws(d);
    const T* dz = (const T*)dy;
    size_t dz_ld = ld_of(d->dy_ld, d->N);
    const bool act = d->act != CVG_ACT_NONE;
    if (d->M > 0 && (dbias || (act && (dx || dw)))) {
        dim3 grid(ceil_div(d->N, 64), ceil_div(d->M, 64));
        T* dzw = act && (dx || dw) ? (T*)ws : nullptr;
        dz_colsum<T><<<grid, 256, 0, s>>>((const T*)dy, dz_ld, (const T*)pre, ld_of(d->pre_ld, d->N), dzw, round_up(d->N, 8),
                                          dbias ? (float*)(ws + o.part) : nullptr, d->M, d->N, d->act);
        CVG_LAUNCH_CHECK();
        if (dzw) { dz = dzw; dz_ld = round_up(d->N, 8); }
    }
    if (dbias) {
        sum_rows<<<ceil_div(d->N, 256), 256, 0, s>>>((const float*)(ws + o.part), ceil_div(d->M, 64), d->N, dbias);
        CVG_LAUNCH_CHECK();
    }
    if (dx && d->M > 0) {
        GemmArgs a{};
        a.A = dz; a.am = dz_ld; a.ak = 1;
        a.B = w; a.bn = 1; a.bk = ld_of(d->w_ld, d->K);
        a.M = d->M; a.N = d->K; a.K = d->N;
        a.e.out = dx; a.e.out_ld = ld_of(d->dx_ld, d->K);
        gemm<T>(a, s);
        CVG_LAUNCH_CHECK();
    }
    if (dw) {
        GemmArgs a{};
        a.A = dz; a.am = 1; a.ak = dz_ld;
        a.B = x; a.bn = 1; a.bk = ld_of(d->x_ld, d->K);
        a.M = d->N; a.N = d->K; a.K = d->M;
        a.e.out = dw; a.e.out_ld = ld_of(d->dw_ld, d->K); a.e.out_f32 = d->dw_dtype == CVG_F32;
        gemm<T>(a, s);
        CVG_LAUNCH_CHECK();
    }
    return 0;
}

}  // namespace

extern "C" {

size_t cvg_linear_act_workspace(const cvg_linear_desc* d, int32_t backward) {
    if (check(d, "linear_act_workspace") != 0) return 0;
    return backward ? bwd_ws(d).total : 0;
}

int cvg_linear_act_fwd(const cvg_linear_desc* d, const void* x, const void* w, const float* bias, const void* res,
                       void* y, void* pre, void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "linear_act_fwd") != 0) return -1;
    if (d->M == 0) return 0;
    CVG_CHECK(x && w && y, "linear_act_fwd: null tensor");
    const size_t es = es_of(d->dtype);
    const void* ps[5] = {x, w, y, res, pre};
    for (const void* p : ps) CVG_CHECK((uintptr_t)p % es == 0, "linear_act_fwd: misaligned tensor");
    (void)ws; (void)ws_bytes;
    GemmArgs a{};
    a.A = x; a.am = ld_of(d->x_ld, d->K); a.ak = 1;
    a.B = w; a.bn = ld_of(d->w_ld, d->K); a.bk = 1;
    a.M = d->M; a.N = d->N; a.K = d->K;
    a.e.bias = bias; a.e.res = res; a.e.pre = pre; a.e.out = y; a.e.act = d->act; a.e.out_f32 = 0;
    a.e.res_ld = ld_of(d->res_ld, d->N); a.e.pre_ld = ld_of(d->pre_ld, d->N); a.e.out_ld = ld_of(d->y_ld, d->N);
    if (d->dtype == CVG_BF16) gemm<bf16>(a, (hipStream_t)s); else gemm<float>(a, (hipStream_t)s);
    CVG_LAUNCH_CHECK();
    return 0;
}

int cvg_linear_act_bwd(const cvg_linear_desc* d, const void* dy, const void* x, const void* w, const void* pre,
                       void* dx, void* dw, float* dbias, void* ws, size_t ws_bytes, cvg_stream s) {
    if (check(d, "linear_act_bwd") != 0) return -1;
    CVG_CHECK(d->M == 0 || dy, "linear_act_bwd: null dy");
    CVG_CHECK(d->M == 0 || !dx || w, "linear_act_bwd: dx needs w");
    CVG_CHECK(d->M == 0 || !dw || x, "linear_act_bwd: dw needs x");
    CVG_CHECK(d->M == 0 || d->act == CVG_ACT_NONE || pre, "linear_act_bwd: an activation needs pre");
    const size_t es = es_of(d->dtype);
    const void* ps[5] = {dy, x, w, pre, dx};
    for (const void* p : ps) CVG_CHECK((uintptr_t)p % es == 0, "linear_act_bwd: misaligned tensor");
    CVG_CHECK((uintptr_t)dw % (d->dw_dtype == CVG_F32 ? 4 : 2) == 0, "linear_act_bwd: misaligned dw");
    const size_t need = bwd_ws(d).total;
    CVG_CHECK(need == 0 || (ws && ws_bytes >= need && aligned16(ws)), "linear_act_bwd: workspace of %zu bytes, need %zu", ws_bytes, need);
    hipStream_t st = (hipStream_t)s;
    return d->dtype == CVG_BF16 ? backward<bf16>(d, dy, x, w, pre, dx, dw, dbias, (char*)ws, st)
                                : backward<float>(d, dy, x, w, pre, dx, dw, dbias, (char*)ws, st);
}

}
