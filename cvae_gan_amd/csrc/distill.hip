// Distillation from a teacher's top logits: loss and gradient of T^2 KL(p || q) in one pass over the student's rows.
//
//   p = softmax(t / T) over the row's `top` teacher entries, q = softmax(s / T) over the V classes,
//   row loss = w T^2 sum_j p_j (log p_j - s[i_j] / T + lse),  ds = scale w T (q - scatter(p)).
//
// TPR threads own a row (a wave, 256 threads or 1024) and hold it in registers, R vectors of 8 each: every vector goes
// into a running (maximum, sum of exponentials) as it arrives, so the sum is taken while the rest of the row is still on
// its way, and the gradient is computed from the same registers: the logits are read once, the gradient is written once.
// A workgroup walks over rows, and as soon as a vector's gradient is stored its registers take the same vector of the
// next row: loads, arithmetic and stores of two rows overlap although one row fills the register file.
// Rows that do not fit (131072 bf16 or 65536 f32 classes) are read twice, the second time mostly from the 256 MB cache.
// The k teacher entries sit in a hash table in LDS, keyed by the vector of 8 their class falls into; whoever computes
// that vector's gradient subtracts them and takes their part of the loss, so nothing is gathered or written twice.
// Bound by memory.  Call to call over rotating buffers, loss and total included: 4096 x 131072 bf16 472 us (4.55 TB/s; a copy
// reaches 5.0-5.4), 2048 x 32768 64 us (4.2 TB/s); the kernel alone under the profiler 480 to 540 and 59.  Rows that are
// no whole number of vectors take branches around their loads and stores: 4096 x 131071 660 us, 2048 x 32003 77.
#include "rowops.h"

namespace {

constexpr int MAX_TOP = 1024;

// e^(d / T) for d <= 0, as 2^(d k): k = log2(e) / T.  For f32 logits in two parts, hi rounded towards zero and lo > 0 (so
// -inf stays -inf): one part alone puts the same relative error times d k into every exponential, and none of it averages
// out (256 x 100, T = 2: 4.9e-7 of the gradient, against 2.3e-7).  bf16 logits carry 2^-9 of their own; there the
// multiply-add more per element would cost 3 % of the time.
struct Scale { float hi, lo; };
template <typename T> __device__ __forceinline__ float exp_t(const Scale& k, float d) {
    return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? fmaf(d, k.lo, d * k.hi) : d * k.hi);
}

struct DistillArgs {
    const void* logits;
    const float* top_val;
    const int32_t* top_idx;
    const float* row_weight;
    float *row_loss, *loss;
    void* dlogits;
    int R, V, top;
    size_t ld, dld, tld;
    Scale k;
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

// Running (maximum, sum of e^((v - maximum) / T)).  The maximum is subtracted before k is multiplied in: k times the lowest
// values of a type overflows, and a row that is masked throughout is uniform.  It starts at the lowest finite value, so
// that a row may begin with -inf; a NaN or +inf reaches the sum.
template <typename T> struct Running {
    float m, s;
    __device__ __forceinline__ void add(const float (&v)[8], const Scale& k) {
        const float before = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = v[j] > m ? v[j] : m;
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) t += exp_t<T>(k, v[j] - m);
        s = fmaf(s, exp_t<T>(k, before - m), t);
    }
    __device__ __forceinline__ void join(float m2, float s2, const Scale& k) {
        const float n = fmaxf(m, m2);
        s = s * exp_t<T>(k, m - n) + s2 * exp_t<T>(k, m2 - n);
        m = n;
    }
};

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
template <typename T> __device__ __forceinline__ void vec_raw(Raw8<T>& x, const T* row, int sh, int V, int i) {
    if (vec_inside<T>(sh, V, i)) {
        raw_load(x, row + i * 8 - sh);
    } else {
        float v[8];
        vec_load<T>(row, sh, V, i, v);
        raw_pack(x, v);
    }
}

template <int TPR> __device__ __forceinline__ void row_barrier() {
    if (TPR == 64) {                                      // (a wave's LDS accesses complete in order)
        asm volatile("" : : : "memory");
        return;
    }
    lds_barrier();
}

// EVEN: every row starts on a 16-byte border and is a whole number of vectors.  R = 0: the row is read from memory twice.
template <typename T, int TPR, int R, bool EVEN>
__global__ void __launch_bounds__(TPR == 64 ? 256 : TPR, 4) distill_row(const DistillArgs a) {
    constexpr int ROWS = TPR == 64 ? 4 : 1, HASH = TPR == 64 ? 256 : 2048;
    __shared__ float sh[64];
    __shared__ int32_t heads[ROWS][HASH];
    extern __shared__ float dyn[];                        // [ROWS][4][top]: value, class, p (of all entries of the class), next
    const int sub = ROWS == 1 ? 0 : threadIdx.x >> 6, tid = ROWS == 1 ? threadIdx.x : threadIdx.x & 63, lane = threadIdx.x & 63;
    int r = blockIdx.x * ROWS + sub;
    if (r >= a.R) return;                                 // (whole waves; only the wave form can have idle ones)
    float* tv = dyn + sub * 4 * a.top;
    int32_t* ti = (int32_t*)(tv + a.top);
    float* tp = tv + 2 * a.top;
    int32_t* next = (int32_t*)(tv + 3 * a.top);
    int32_t* head = heads[sub];
    const Scale k = a.k;
    const int stride = gridDim.x * ROWS;
    constexpr uint32_t VB = 8 * sizeof(T);               // bytes of a vector

    const T* row = (const T*)a.logits + (size_t)r * a.ld;
    int off = EVEN ? 0 : (int)(((uintptr_t)row & 15) / sizeof(T)), nvec = (off + a.V + 7) / 8;
    // this thread's first teacher entry (the only one where there are as many threads as entries) travels a row ahead
    const int my = min(tid, a.top - 1);
    float ev = a.top_val[(size_t)r * a.tld + my];
    int32_t ei = a.top_idx[(size_t)r * a.tld + my];
    float w = a.row_weight ? a.row_weight[r] : 1.f;
    // Loads and stores of the EVEN form are unconditional (lanes behind the row repeat its last vector, and store the same
    // values there): under a branch the compiler could not tell how many are in flight and would wait for all of them.
    Raw8<T> x[R > 0 ? R : 1];
    if constexpr (R > 0) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int i = tid + u * TPR;
            if constexpr (EVEN) raw_load(x[u], (const T*)((const char*)row + (uint32_t)min(i, nvec - 1) * VB));
            else if (i < nvec) vec_raw<T>(x[u], row, off, a.V, i);
        }
    }

    for (;;) {
        T* out = a.dlogits ? (T*)a.dlogits + (size_t)r * a.dld : nullptr;
        const bool whole = EVEN || (out && ((((uintptr_t)out) ^ (uintptr_t)row) & 15) == 0);
        // ---- the teacher: entries into LDS, their maximum and sum, chains by vector
        float v0 = ev;
        int c0 = ei;
        if (c0 < 0 || c0 >= a.V || v0 == -INFINITY) { c0 = -1; v0 = -INFINITY; }
        float s0 = to_f32(row[max(c0, 0)]);               // the student's logit at this thread's first class
        if (tid < a.top) { tv[tid] = v0; ti[tid] = c0; }
        for (int j = tid + TPR; j < a.top; j += TPR) {
            const float v = a.top_val[(size_t)r * a.tld + j];
            const int c = a.top_idx[(size_t)r * a.tld + j];
            const bool in = c >= 0 && c < a.V && v != -INFINITY;
            tv[j] = in ? v : -INFINITY;
            ti[j] = in ? c : -1;
        }
        for (int i = tid; i < HASH; i += TPR) head[i] = -1;
        row_barrier<TPR>();
        float tmax = -INFINITY, ps = 0.f;                 // (every wave takes them over all entries)
        for (int j = lane; j < a.top; j += 64) tmax = fmaxf(tmax, tv[j]);
        tmax = wave_max(tmax);
        for (int j = lane; j < a.top; j += 64)
            if (ti[j] >= 0) ps += expf((tv[j] - tmax) * a.inv_t);
        ps = wave_sum(ps);                                // 0: no entry at all (the largest adds 1, a NaN stays)
        const bool dead = w == 0.f || ps == 0.f;
        const float inv_ps = 1.f / ps;
        auto share = [&](int j) { return expf((tv[j] - tmax) * a.inv_t) * inv_ps; };      // p of entry j
        if (!dead)
            for (int j = tid; j < a.top; j += TPR) {
                const int c = ti[j];
                if (c < 0 || share(j) == 0.f) { next[j] = -2; continue; }      // (absent, or nothing to add)
                next[j] = atomicExch(&head[((c + off) >> 3) & (HASH - 1)], j);
            }
        row_barrier<TPR>();
        if (!dead)
            for (int j = tid; j < a.top; j += TPR) {
                // p of the class: where entries name it twice the first stands for all, added in their order, whatever the
                // order in which they were chained
                const int c = ti[j];
                float p = 0.f;
                if (next[j] != -2) {
                    for (int last = -1;;) {
                        int e = MAX_TOP;
                        for (int q = head[((c + off) >> 3) & (HASH - 1)]; q >= 0; q = next[q])
                            if (q > last && q < e && ti[q] == c) e = q;
                        if (last < 0 && e != j) break;    // (not the first)
                        if (e == MAX_TOP) break;
                        p += share(e);
                        last = e;
                    }
                }
                tp[j] = p;
            }
        // ---- maximum and sum
        Running<T> run{-3.402823466e38f, 0.f};
        if constexpr (R > 0) {
#pragma unroll
            for (int u = 0; u < R; ++u) {
                if (tid + u * TPR < nvec) {
                    float v[8];
                    pin(x[u]);
                    raw_f32(x[u], v);
                    run.add(v, k);
                }
            }
        } else {
            // 64 vectors at a time: in one sum of thousands (2^31 classes: 262144) terms below its last bit would all be lost,
            // 7e-4 of the whole where a thread's first vector holds the largest logit
            Running<T> whole = run;
            for (int i = tid; i < nvec;) {
                for (int n = 0; n < 64 && i < nvec; ++n, i += TPR) {
                    float v[8];
                    vec_load<T>(row, off, a.V, i, v);
                    run.add(v, k);
                }
                whole.join(run.m, run.s, k);
                run = Running<T>{-3.402823466e38f, 0.f};
            }
            run = whole;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) run.join(__shfl_xor(run.m, o, 64), __shfl_xor(run.s, o, 64), k);
        asm volatile("" : "+v"(s0));                      // (arrived: behind the barrier the row may be overwritten)
        if (TPR > 64) {
            if (lane == 0) { sh[tid >> 6] = run.m; sh[16 + (tid >> 6)] = run.s; }
            row_barrier<TPR>();                           // (publishes tp too)
            run.m = sh[0];
            run.s = sh[16];
#pragma unroll
            for (int i = 1; i < TPR / 64; ++i) run.join(sh[i], sh[16 + i], k);
        }
        const float m = run.m, inv_z = 1.f / run.s, c = a.scale * w * a.temp, cz = c * inv_z;
        // ---- the loss: T^2 p (log p - log q) as T p ((t - its maximum) - T log(its sum) - ((s - maximum) - T log z)), which
        // does not divide a masked logit by a temperature below one
        float l = 0.f;
        if (!dead) {
            const float tz = a.temp * logf(run.s), tp0 = a.temp * logf(ps), wt = w * a.temp;
            for (int j = tid; j < a.top; j += TPR) {
                if (next[j] == -2) continue;
                const float v = j == tid ? s0 : to_f32(row[ti[j]]);
                l += wt * share(j) * (((tv[j] - tmax) - tp0) - ((v - m) - tz));
            }
        }
        // ---- the gradient; the next row moves in
        const int rn = r + stride;
        const bool more = rn < a.R;
        const T* row_n = more ? (const T*)a.logits + (size_t)rn * a.ld : row;
        const int off_n = EVEN ? 0 : (int)(((uintptr_t)row_n & 15) / sizeof(T)), nvec_n = (off_n + a.V + 7) / 8;
        const int r_next = more ? rn : r;
        ev = a.top_val[(size_t)r_next * a.tld + my];
        ei = a.top_idx[(size_t)r_next * a.tld + my];
        w = a.row_weight ? a.row_weight[r_next] : 1.f;
        if (TPR > 64 && a.top > TPR) {                    // (the loads of the loop above have arrived in every wave)
            asm volatile("" : "+v"(l));
            row_barrier<TPR>();
        }
        auto gradient = [&](float (&v)[8], int i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = cz * exp_t<T>(k, v[j] - m);
            for (int q = head[i & (HASH - 1)]; q >= 0; q = next[q]) {
                const int at = ti[q] + off - 8 * i;
                const float p = c * tp[q];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] -= j == at ? p : 0.f;
            }
        };
        // (a fresh copy of tid per row: what depends on it is recomputed where it is used instead of being kept in R
        // registers across rows)
        int t = tid;
        asm volatile("" : "+v"(t));
        const int last_n = more ? nvec_n - 1 : 0;         // (no next row: one line, loaded and never used)
        if constexpr (R > 0 && EVEN) {
            // one path for every row (two would meet with the loads in different registers, and wait for them to move)
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int i = min(t + u * TPR, nvec - 1);
                float v[8];
                pin(x[u]);
                if (dead) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = 0.f;
                } else {
                    raw_f32(x[u], v);
                    gradient(v, i);
                }
                if (R > 4 || out) store8<T>((T*)((char*)out + (uint32_t)i * VB), v);       // (R > 4 is launched with an output)
                raw_load(x[u], (const T*)((const char*)row_n + (uint32_t)min(t + u * TPR, last_n) * VB));
            }
        } else if constexpr (R > 0) {
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int i = t + u * TPR;
                if (out && i < nvec) {
                    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    pin(x[u]);
                    if (!dead) {
                        raw_f32(x[u], v);
                        gradient(v, i);
                    }
                    vec_store<T>(out, off, a.V, i, whole, v);
                }
                if (more && i < nvec_n) vec_raw<T>(x[u], row_n, off_n, a.V, i);
            }
        } else if (out) {
            for (int i = tid; i < nvec; i += TPR) {
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (!dead) {
                    vec_load<T>(row, off, a.V, i, v);
                    gradient(v, i);
                }
                vec_store<T>(out, off, a.V, i, whole, v);
            }
        }
        l = wave_sum(l);
        if (TPR > 64) {
            if (lane == 0) sh[32 + (tid >> 6)] = l;
            row_barrier<TPR>();                           // (and the table may be cleared)
            l = 0.f;
#pragma unroll
            for (int i = 0; i < TPR / 64; ++i) l += sh[32 + i];
        }
        if (tid == 0) a.row_loss[r] = l;
        if (!more) return;
        r = rn;
        row = row_n;
        off = off_n;
        nvec = nvec_n;
    }
}

template <typename T, int TPR, int R>
void launch_as(const DistillArgs& a, bool even, int per_cu, hipStream_t st) {
    constexpr int ROWS = TPR == 64 ? 4 : 1;
    const size_t lds = (size_t)a.top * 16 * ROWS;
    // as many workgroups as the chip holds at once; each walks over its share of the rows
    const int blocks = min(ceil_div(a.R, ROWS), 256 * per_cu);
    if (even) distill_row<T, TPR, R, true><<<blocks, TPR == 64 ? 256 : TPR, lds, st>>>(a);
    else distill_row<T, TPR, R, false><<<blocks, TPR == 64 ? 256 : TPR, lds, st>>>(a);
}
template <typename T>
void launch(const DistillArgs& a, hipStream_t st) {
    constexpr bool B = sizeof(T) == 2;
    // (rows that do not all start on a 16-byte border may need one vector more)
    const bool aligned = aligned16(a.logits) && a.ld * sizeof(T) % 16 == 0;
    const bool even = aligned && a.V % 8 == 0 && (!a.dlogits || (aligned16(a.dlogits) && a.dld * sizeof(T) % 16 == 0));
    const int nvec = (a.V + 7) / 8 + (aligned ? 0 : 1);
    // A wave per row while 4 vectors per lane hold it; then as many threads as hold the row in 64 registers each, so that
    // a CU's registers are full of rows (four, two, one) at every size.
    constexpr int F = B ? 1 : 2;                          // (an f32 vector takes twice the registers)
    if (nvec <= 64) launch_as<T, 64, 1>(a, even, 8, st);
    else if (nvec <= 256) launch_as<T, 64, 4>(a, even, 4, st);
    else if (nvec <= 1024) launch_as<T, 256, 4>(a, even, 4, st);
    else if (!a.dlogits) launch_as<T, 1024, 0>(a, even, 2, st);        // (without a gradient the row is read once there too)
    else if (nvec * F <= 256 * 12) launch_as<T, 256, 12 / F>(a, even, 4, st);
    else if (nvec * F <= 256 * 16) launch_as<T, 256, 16 / F>(a, even, 4, st);
    else if (nvec * F <= 512 * 12) launch_as<T, 512, 12 / F>(a, even, 2, st);
    else if (nvec * F <= 512 * 16) launch_as<T, 512, 16 / F>(a, even, 2, st);
    else if (nvec * F <= 1024 * 12) launch_as<T, 1024, 12 / F>(a, even, 1, st);
    else if (nvec * F <= 1024 * 16) launch_as<T, 1024, 16 / F>(a, even, 1, st);
    else launch_as<T, 1024, 0>(a, even, 2, st);
}

__global__ void __launch_bounds__(1024) distill_total(const float* __restrict__ rows, int R, float* loss) {
    __shared__ float sh[16];
    float s = 0.f;
#pragma unroll 8
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
    CVG_CHECK(d->R <= 0x7fff0000 && d->V <= 0x7ffffff0, "distill_topk: R %d, V %d", d->R, d->V);   // (row loops step past the end)
    CVG_CHECK(d->top >= 1 && d->top <= MAX_TOP, "distill_topk: %d teacher entries (1..%d)", d->top, MAX_TOP);
    CVG_CHECK(d->temperature >= 1e-37f && d->temperature <= 1e20f, "distill_topk: temperature %g", (double)d->temperature);
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
    const double k = 1.4426950408889634 / (double)d->temperature;
    a.k.hi = (float)k;
    if (d->dtype == CVG_F32 && (double)a.k.hi > k) a.k.hi = nextafterf(a.k.hi, 0.f);
    a.k.lo = (float)(k - (double)a.k.hi);
    // (nothing left: any normal number far below hi's last bit; T <= 1e20 keeps both parts of k normal)
    if (!(a.k.lo > 0.f)) a.k.lo = a.k.hi * 0x1p-40f;
    CVG_CHECK(dlogits != logits || a.ld == a.dld, "distill_topk: in place with different pitches");
    CVG_CHECK(apart({row_loss, dlogits}, {top_val, top_idx, row_weight}) && apart({row_loss}, {logits}) &&
              apart({loss}, {logits, top_val, top_idx, row_weight, dlogits, d->R > 1 ? row_loss : nullptr}),
              "distill_topk: an output over another tensor");
    hipStream_t st = (hipStream_t)s;
    if (d->R > 0) {
        if (d->dtype == CVG_BF16) launch<bf16>(a, st); else launch<float>(a, st);
        CVG_LAUNCH_CHECK();
    }
    distill_total<<<1, 1024, 0, st>>>(row_loss, d->R, loss);
    CVG_LAUNCH_CHECK();
    return 0;
}
