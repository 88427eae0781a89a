// Distillation from a teacher's top logits: loss and gradient of T^2 KL(p || q) in one pass over the student's rows.
//
//   p = softmax(t / T) over the row's `top` teacher entries, q = softmax(s / T) over the V classes,
//   row loss = w T^2 sum_j p_j (log p_j - s[i_j] / T + lse),  ds = scale w T (q - scatter(p)).
//
// TPR threads own a row (a wave, 256 threads or 1024) and hold it in registers, R vectors of 8 each: every vector goes
// into a running (maximum, sum of exponentials) as it arrives, so the sum is taken while the rest of the row is still on
// its way, and the gradient is computed from the same registers: the logits are read once, the gradient is written once.
// Rows that do not fit (131072 bf16 or 65536 f32 classes) are read twice, the second time mostly from the 256 MB cache.
// The k classes of the teacher are written after a barrier, over the q the row pass left there.
#include "rowops.h"

namespace {

constexpr int MAX_TOP = 1024;

struct DistillArgs {
    const void* logits;
    const float* top_val;
    const int32_t* top_idx;
    const float* row_weight;
    float *row_loss, *loss;
    void* dlogits;
    int R, V, top;
    size_t ld, dld, tld;
    float inv_t, temp, scale;
};

// sum over the TPR threads of a row (one wave, or the whole workgroup through LDS)
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* sh) {
    v = wave_sum(v);
    if (TPR == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) s += sh[i];
    return s;
}

#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Running (maximum, sum of 2^(k (v - maximum))).  The maximum starts at the lowest finite value, so that a row may begin
// with -inf; a NaN or +inf reaches the sum.
struct Running {
    float m, s;
    __device__ __forceinline__ void add(const float (&v)[8], float k) {
        float n = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) n = fmaxf(n, v[j]);
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) t += exp2_((v[j] - n) * k);
        s = s * exp2_((m - n) * k) + t;
        m = n;
    }
    __device__ __forceinline__ void join(float m2, float s2, float k) {
        const float n = fmaxf(m, m2);
        s = s * exp2_((m - n) * k) + s2 * exp2_((m2 - n) * k);
        m = n;
    }
};
template <int TPR> __device__ __forceinline__ void row_join(Running& r, float k, float* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) r.join(__shfl_xor(r.m, o, 64), __shfl_xor(r.s, o, 64), k);
    if (TPR == 64) return;
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = r.m; sh[16 + (threadIdx.x >> 6)] = r.s; }
    __syncthreads();
    r.m = sh[0];
    r.s = sh[16];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) r.join(sh[i], sh[16 + i], k);
}

// The row as vectors of 8 elements on 16-byte borders: vector i covers elements [8 i - sh, 8 i - sh + 8), where sh is
// how far behind a border the row starts; the first and the last vector may hang over the row and go element by element.
template <typename T> __device__ __forceinline__ void vec_load(const T* base, int sh, int V, int i, float (&v)[8]) {
    const int e0 = i * 8 - sh;
    if (e0 >= 0 && e0 + 8 <= V) {
        load8<T>(base + e0, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = e0 + j >= 0 && e0 + j < V ? to_f32(base[e0 + j]) : -INFINITY;
    }
}
template <typename T> __device__ __forceinline__ void vec_store(T* base, int sh, int V, int i, bool whole, const float (&v)[8]) {
    const int e0 = i * 8 - sh;
    if (whole && e0 >= 0 && e0 + 8 <= V) {
        store8<T>(base + e0, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e0 + j >= 0 && e0 + j < V) base[e0 + j] = from_f32<T>(v[j]);
    }
}

template <typename T> __device__ __forceinline__ bool vec_inside(int sh, int V, int i) { return i * 8 - sh >= 0 && i * 8 - sh + 8 <= V; }

// R = 0: the row is read from memory twice
template <typename T, int TPR, int R>
__global__ void __launch_bounds__(TPR == 64 ? 256 : TPR) distill_row(const DistillArgs a) {
    constexpr int ROWS = TPR == 64 ? 4 : 1;
    __shared__ float sh[32];
    extern __shared__ float dyn[];                        // [ROWS][top] p, then [ROWS][top] class indices
    const int sub = ROWS == 1 ? 0 : threadIdx.x >> 6, tid = ROWS == 1 ? threadIdx.x : threadIdx.x & 63, lane = threadIdx.x & 63;
    const int r = blockIdx.x * ROWS + sub;
    if (ROWS > 1 && r >= a.R) return;                     // (whole waves; the wave form has no barrier)
    float* tp = dyn + sub * a.top;
    int32_t* ti = (int32_t*)(dyn + ROWS * a.top) + sub * a.top;
    const T* row = (const T*)a.logits + (size_t)r * a.ld;
    T* out = a.dlogits ? (T*)a.dlogits + (size_t)r * a.dld : nullptr;
    const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
    const bool whole = out && ((((uintptr_t)out) ^ (uintptr_t)row) & 15) == 0;
    const int nvec = (off + a.V + 7) / 8;
    const float k = a.inv_t * LOG2E;

    Raw8<T> x[R > 0 ? R : 1];
    if constexpr (R > 0) {                                // everything is requested before anything is waited for
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int i = tid + u * TPR;
            if (i < nvec && vec_inside<T>(off, a.V, i)) raw_load(x[u], row + i * 8 - off);
            else {
                float v[8];
                vec_load<T>(row, off, a.V, i, v);
                raw_pack(x[u], v);
            }
        }
    }
    // The teacher: every wave takes the maximum and the sum over all entries, so no wave waits for another.
    const float w = a.row_weight ? a.row_weight[r] : 1.f;
    const float* val = a.top_val + (size_t)r * a.tld;
    const int32_t* idx = a.top_idx + (size_t)r * a.tld;
    auto entry = [&](int j, int& i) {
        i = idx[j];
        const float v = val[j] * a.inv_t;
        if (i < 0 || i >= a.V || v == -INFINITY) i = -1;
        return i < 0 ? -INFINITY : v;
    };
    float tmax = -INFINITY, ps = 0.f, v0 = -INFINITY;
    int i0 = -1;
    if (lane < a.top) v0 = tmax = entry(lane, i0);        // (the first 64 entries are read once)
    for (int j = lane + 64; j < a.top; j += 64) { int i; tmax = fmaxf(tmax, entry(j, i)); }
    tmax = wave_max(tmax);
    if (i0 >= 0) ps = expf(v0 - tmax);
    for (int j = lane + 64; j < a.top; j += 64) {
        int i;
        const float v = entry(j, i);
        if (i >= 0) ps += expf(v - tmax);
    }
    ps = wave_sum(ps);                                    // 0: no entry at all (the largest adds 1, a NaN stays)
    if (w == 0.f || ps == 0.f) {                          // (the same for every thread of the row)
        if (tid == 0) a.row_loss[r] = 0.f;
        if (out) {
            const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int i = tid; i < nvec; i += TPR) vec_store<T>(out, off, a.V, i, whole, z);
        }
        return;
    }

    Running run{-3.402823466e38f, 0.f};
    if constexpr (R > 0) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            if (tid + u * TPR < nvec) {
                float v[8];
                raw_f32(x[u], v);
                run.add(v, k);
            }
        }
    } else {
        for (int i = tid; i < nvec; i += TPR) {
            float v[8];
            vec_load<T>(row, off, a.V, i, v);
            run.add(v, k);
        }
    }
    row_join<TPR>(run, k, sh);
    const float m = run.m, logz = logf(run.s), inv_z = 1.f / run.s, logp0 = logf(ps);
    // loss terms; p, the class and q at the class are kept for the gradient (q before the row is overwritten: dlogits may
    // be logits)
    float l = 0.f, qj[MAX_TOP / TPR > 0 ? MAX_TOP / TPR : 1];
#pragma unroll
    for (int u = 0; u < (MAX_TOP + TPR - 1) / TPR; ++u) {
        const int j = tid + u * TPR;
        if (j >= a.top) break;
        int i = i0;
        const float v = TPR == 64 && u == 0 ? v0 : entry(j, i), lp = v - tmax - logp0, p = i < 0 ? 0.f : expf(v - tmax) / ps;
        const float z = i < 0 ? 0.f : (to_f32(row[i]) - m) * a.inv_t;
        if (i >= 0 && (p > 0.f || p != p)) l += p * (lp - (z - logz));
        qj[u] = i < 0 ? 0.f : expf(z) * inv_z;
        tp[j] = p;
        ti[j] = i;
    }
    l = row_sum<TPR>(l, sh);                              // (its barriers also publish tp and ti, and end the reads of the row)
    if (tid == 0) a.row_loss[r] = w * a.temp * a.temp * l;
    if (!out) return;
    const float c = a.scale * w * a.temp, cz = c * inv_z;
    if constexpr (R > 0) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int i = tid + u * TPR;
            if (i < nvec) {
                float v[8];
                raw_f32(x[u], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = cz * exp2_((v[j] - m) * k);
                vec_store<T>(out, off, a.V, i, whole, v);
            }
        }
    } else {
        for (int i = tid; i < nvec; i += TPR) {
            float v[8];
            vec_load<T>(row, off, a.V, i, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = cz * exp2_((v[j] - m) * k);
            vec_store<T>(out, off, a.V, i, whole, v);
        }
    }
    // the row's stores are acknowledged before the teacher's classes are written over them
    if (TPR == 64) __threadfence_block(); else __syncthreads();
#pragma unroll
    for (int u = 0; u < (MAX_TOP + TPR - 1) / TPR; ++u) {
        const int j = tid + u * TPR;
        if (j >= a.top) break;
        if (ti[j] < 0) continue;
        // an index that appears more than once: its first entry writes the sum
        float p = 0.f;
        bool first = true;
        for (int e = 0; e < a.top; ++e)
            if (ti[e] == ti[j]) { first &= e >= j; p += tp[e]; }
        if (first) out[ti[j]] = from_f32<T>(c * (qj[u] - p));
    }
}

template <typename T>
void launch(const DistillArgs& a, hipStream_t st) {
    // (rows that do not all start on a 16-byte border may need one vector more)
    const bool even = aligned16(a.logits) && a.ld * sizeof(T) % 16 == 0;
    const int nvec = (a.V + 7) / 8 + (even ? 0 : 1);
    const size_t lds = (size_t)a.top * 8;
    constexpr bool B = sizeof(T) == 2;
    // a wave per row while 8 vectors per lane hold it, 256 threads for mid-sized rows, otherwise a workgroup of 1024
    if (nvec <= 64) distill_row<T, 64, 1><<<ceil_div(a.R, 4), 256, lds * 4, st>>>(a);
    else if (nvec <= 256) distill_row<T, 64, 4><<<ceil_div(a.R, 4), 256, lds * 4, st>>>(a);
    else if (nvec <= 1024) distill_row<T, 256, 4><<<a.R, 256, lds, st>>>(a);
    else if (nvec <= 4096) distill_row<T, 1024, 4><<<a.R, 1024, lds, st>>>(a);
    else if (nvec <= 8192) distill_row<T, 1024, 8><<<a.R, 1024, lds, st>>>(a);
    else if (B && nvec <= 16384) distill_row<T, 1024, B ? 16 : 8><<<a.R, 1024, lds, st>>>(a);
    else distill_row<T, 1024, 0><<<a.R, 1024, lds, st>>>(a);
}

__global__ void __launch_bounds__(1024) distill_total(const float* __restrict__ rows, int R, float* loss) {
    __shared__ float sh[16];
    float s = 0.f;
    for (int i = threadIdx.x; i < R; i += 1024) s += rows[i];
    s = row_sum<1024>(s, sh);
    if (threadIdx.x == 0) *loss = s;
}

}  // namespace

extern "C" int cvg_distill_topk(const cvg_distill_desc* d, const void* logits, const float* top_val, const int32_t* top_idx,
                                const float* row_weight, float* loss, float* row_loss, void* dlogits, cvg_stream s) {
    CVG_CHECK(d, "distill_topk: null descriptor");
    CVG_CHECK(d->dtype == CVG_F32 || d->dtype == CVG_BF16, "distill_topk: dtype %d", d->dtype);
    CVG_CHECK(d->R >= 0 && d->V >= 1, "distill_topk: R %d, V %d", d->R, d->V);
    CVG_CHECK(d->V <= 0x7ffffff0, "distill_topk: V %d", d->V);
    CVG_CHECK(d->top >= 1 && d->top <= MAX_TOP, "distill_topk: %d teacher entries (1..%d)", d->top, MAX_TOP);
    CVG_CHECK(d->temperature > 0.f && d->temperature < INFINITY, "distill_topk: temperature %g", (double)d->temperature);
    CVG_CHECK((d->logits_ld == 0 || d->logits_ld >= d->V) && (d->dlogits_ld == 0 || d->dlogits_ld >= d->V) &&
              (d->top_ld == 0 || d->top_ld >= d->top), "distill_topk: pitches %d, %d, %d", d->logits_ld, d->dlogits_ld, d->top_ld);
    CVG_CHECK(loss, "distill_topk: null loss");
    CVG_CHECK(d->R == 0 || (logits && top_val && top_idx && row_loss), "distill_topk: null tensor");
    const size_t es = d->dtype == CVG_BF16 ? 2 : 4;
    CVG_CHECK((uintptr_t)logits % es == 0 && (uintptr_t)dlogits % es == 0, "distill_topk: misaligned logits");
    DistillArgs a{};
    a.logits = logits; a.top_val = top_val; a.top_idx = top_idx; a.row_weight = row_weight;
    a.row_loss = row_loss; a.loss = loss; a.dlogits = dlogits;
    a.R = d->R; a.V = d->V; a.top = d->top;
    a.ld = d->logits_ld ? d->logits_ld : d->V;
    a.dld = d->dlogits_ld ? d->dlogits_ld : d->V;
    a.tld = d->top_ld ? d->top_ld : d->top;
    a.temp = d->temperature; a.inv_t = 1.f / d->temperature; a.scale = d->grad_scale;
    CVG_CHECK(dlogits != logits || a.ld == a.dld, "distill_topk: in place with different pitches");
    hipStream_t st = (hipStream_t)s;
    if (d->R > 0) {
        if (d->dtype == CVG_BF16) launch<bf16>(a, st); else launch<float>(a, st);
        CVG_LAUNCH_CHECK();
    }
    distill_total<<<1, 1024, 0, st>>>(row_loss, d->R, loss);
    CVG_LAUNCH_CHECK();
    return 0;
}
