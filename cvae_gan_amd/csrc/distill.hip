// Distillation from a teacher's top logits: loss and gradient of T^2 KL(p || q) in one pass over the student's rows.
//
//   p = softmax(t / T) over the row's `top` teacher entries, q = softmax(s / T) over the V classes,
//   row loss = w T^2 sum_j p_j (log p_j - s[i_j] / T + lse),  ds = scale w T (q - scatter(p)).
//
// One workgroup per row.  The row is held in registers between the maximum, the sum of exponentials and the gradient,
// so the logits are read once and the gradient is written once; the k teacher entries live in LDS.  The gradient of
// the k classes is written after a barrier, over the q the row pass left there.
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

// reductions over the TPR threads of a row (one wave, or the whole workgroup through LDS)
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
template <int TPR> __device__ __forceinline__ float row_max(float v, float* sh) {
    v = wave_max(v);
    if (TPR == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = sh[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) s = fmaxf(s, sh[i]);
    return s;
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

// simple form: three passes over the row from memory
template <typename T>
__global__ void __launch_bounds__(256) distill_row(const DistillArgs a) {
    __shared__ float sh[4];
    __shared__ float tv[MAX_TOP];
    __shared__ int32_t ti[MAX_TOP];
    const int r = blockIdx.x;
    const T* row = (const T*)a.logits + (size_t)r * a.ld;
    T* out = a.dlogits ? (T*)a.dlogits + (size_t)r * a.dld : nullptr;
    const int sh_in = (int)(((uintptr_t)row & 15) / sizeof(T));
    const bool whole = out && ((((uintptr_t)out) ^ (uintptr_t)row) & 15) == 0;
    const int nvec = (sh_in + a.V + 7) / 8;
    const float w = a.row_weight ? a.row_weight[r] : 1.f;
    // teacher
    float tm = -INFINITY;
    for (int j = threadIdx.x; j < a.top; j += 256) {
        const int i = a.top_idx[(size_t)r * a.tld + j];
        const float v = a.top_val[(size_t)r * a.tld + j] * a.inv_t;
        const bool in = i >= 0 && i < a.V && v != -INFINITY;
        ti[j] = in ? i : -1;
        tv[j] = in ? v : -INFINITY;
        tm = (in && !(v <= tm)) ? v : tm;             // (a NaN stays)
    }
    const float tmax = row_max<256>(tm, sh);
    float any_nan = 0.f, zs = 0.f;
    for (int j = threadIdx.x; j < a.top; j += 256)
        if (ti[j] >= 0) { zs += expf(tv[j] - tmax); any_nan = 1.f; }
    const float psum = row_sum<256>(zs, sh);
    const bool empty = row_sum<256>(any_nan, sh) == 0.f;
    if (w == 0.f || empty) {
        if (threadIdx.x == 0) a.row_loss[r] = 0.f;
        if (out) {
            const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int i = threadIdx.x; i < nvec; i += 256) vec_store<T>(out, sh_in, a.V, i, whole, z);
        }
        return;
    }
    float m = -INFINITY;
    for (int i = threadIdx.x; i < nvec; i += 256) {
        float v[8];
        vec_load<T>(row, sh_in, a.V, i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, v[j]);
    }
    m = row_max<256>(m, sh);
    float z = 0.f;
    for (int i = threadIdx.x; i < nvec; i += 256) {
        float v[8];
        vec_load<T>(row, sh_in, a.V, i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) z += expf((v[j] - m) * a.inv_t);
    }
    z = row_sum<256>(z, sh);
    const float logz = logf(z), logp0 = logf(psum);
    // loss terms; the student's logits at the teacher's classes are kept for the gradient
    float l = 0.f;
    for (int j = threadIdx.x; j < a.top; j += 256) {
        if (ti[j] < 0) continue;
        const float lp = tv[j] - tmax - logp0, p = expf(tv[j] - tmax) / psum;
        const float lq = (to_f32(row[ti[j]]) - m) * a.inv_t - logz;
        if (p > 0.f || p != p) l += p * (lp - lq);
        tv[j] = p;
    }
    l = row_sum<256>(l, sh);
    if (threadIdx.x == 0) a.row_loss[r] = w * a.temp * a.temp * l;
    if (!out) return;
    const float c = a.scale * w * a.temp, inv_z = 1.f / z;
    // q at the teacher's classes, read before the row is overwritten (dlogits may be logits)
    float qj[MAX_TOP / 256];
#pragma unroll
    for (int u = 0; u < MAX_TOP / 256; ++u) {
        const int j = threadIdx.x + u * 256;
        qj[u] = j < a.top && ti[j] >= 0 ? expf((to_f32(row[ti[j]]) - m) * a.inv_t) * inv_z : 0.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nvec; i += 256) {
        float v[8];
        vec_load<T>(row, sh_in, a.V, i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c * (expf((v[j] - m) * a.inv_t) * inv_z);
        vec_store<T>(out, sh_in, a.V, i, whole, v);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MAX_TOP / 256; ++u) {
        const int j = threadIdx.x + u * 256;
        if (j >= a.top || ti[j] < 0) continue;
        // an index that appears more than once: its first entry writes the sum
        float p = 0.f;
        bool first = true;
        for (int k = 0; k < a.top; ++k)
            if (ti[k] == ti[j]) { first &= k >= j; p += tv[k]; }
        if (first) out[ti[j]] = from_f32<T>(c * (qj[u] - p));
    }
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
        if (d->dtype == CVG_BF16) distill_row<bf16><<<d->R, 256, 0, st>>>(a);
        else distill_row<float><<<d->R, 256, 0, st>>>(a);
        CVG_LAUNCH_CHECK();
    }
    distill_total<<<1, 1024, 0, st>>>(row_loss, d->R, loss);
    CVG_LAUNCH_CHECK();
    return 0;
}
