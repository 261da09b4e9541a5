// tensor_list.hip -- the end of a training step over a LIST of tensors, in a few launches however many tensors the list has:
//   bfsr_list_write / bfsr_pointer_write : the device table of a list (rows of pointers and sizes, and the chunks they are cut into)
//   bfsr_grad_norm                       : global norm, sqrt(sum g^2) or max |g|
//   bfsr_clip_grads                      : out = min(1, max_norm / (norm + 1e-6)) g
//   bfsr_adam_step                       : Adam's update, with the clipping folded into its read of the gradients
// (the optimizer and loop body of LINF-LP/train.py:46-62, 118-160, which leave this to torch's per-tensor operations).
//
// Every tensor is dense memory of fp32 / fp16 / bf16, so a list is flat elements, cut into chunks of `chunk` elements that never cross a tensor.
// A workgroup finds its chunk's row with two dependent scalar loads, whatever the number of tensors.  Nothing asks for more than
// the element's own alignment: the vector types below say so and gfx950's global loads of 8 and 16 bytes take it.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include "../../include/bfsr_hip.h"
#include "launch_util.h"

namespace {

constexpr int T = 256;                        // threads of a workgroup
constexpr int WAVES = T / 64;
constexpr int CHUNK = 2048;                   // elements of a chunk: what one wave takes at a time
constexpr int MAX_PARTS = 1024;               // partial results of a norm, one for each of its workgroups

struct Row { const void* p[4]; float* step; long long n; int type, type_g; long long pad; };      // BFSR_LIST_ROW bytes
static_assert(sizeof(Row) == BFSR_LIST_ROW, "the row's size is part of the interface");

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned short h8u __attribute__((ext_vector_type(8), aligned(2)));
#define GLOBAL __attribute__((address_space(1)))          // the rows' pointers are of device memory, which the compiler cannot know: without it every access is a flat one

__device__ __forceinline__ float from_half(unsigned short h) { return __half2float(__ushort_as_half(h)); }
__device__ __forceinline__ float from_bf16(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ unsigned short to_half(float f) { return __half_as_ushort(__float2half_rn(f)); }
__device__ __forceinline__ unsigned short to_bf16(float f)               // round to nearest even; a NaN stays one
{
    const unsigned u = __float_as_uint(f);
    return f != f ? (unsigned short)((u >> 16) | 0x40) : (unsigned short)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
}

// The elements of a type, N to a load of 16 bytes.
template <int TYPE> struct Vec;
template <> struct Vec<BFSR_LIST_F32> { typedef f4u type; typedef float one; static constexpr int N = 4; __device__ static float wide(float f) { return f; } };
template <> struct Vec<BFSR_LIST_F16> { typedef h8u type; typedef unsigned short one; static constexpr int N = 8; __device__ static float wide(unsigned short h) { return from_half(h); } };
template <> struct Vec<BFSR_LIST_BF16> { typedef h8u type; typedef unsigned short one; static constexpr int N = 8; __device__ static float wide(unsigned short h) { return from_bf16(h); } };

// Four elements of a tensor of `type` from element i on; those from `count` on are 0 and are not touched.
struct Four { f4u f; h4u h; };

template <bool FULL>
__device__ __forceinline__ Four load4(const void* p, int type, int i, int count)
{
    Four r = {{0.f, 0.f, 0.f, 0.f}, {0, 0, 0, 0}};
    if (type == BFSR_LIST_F32) {
        const GLOBAL float* q = (const GLOBAL float*)p + i;
        if (FULL || i + 4 <= count) r.f = *(const GLOBAL f4u*)q;
        else for (int k = 0; k < 3; ++k) if (i + k < count) r.f[k] = q[k];
    } else {
        const GLOBAL unsigned short* q = (const GLOBAL unsigned short*)p + i;
        if (FULL || i + 4 <= count) r.h = *(const GLOBAL h4u*)q;
        else for (int k = 0; k < 3; ++k) if (i + k < count) r.h[k] = q[k];
    }
    return r;
}

__device__ __forceinline__ f4 floats(Four a, int type)
{
    if (type == BFSR_LIST_F32) return a.f;
    f4 r;
    for (int k = 0; k < 4; ++k) r[k] = type == BFSR_LIST_F16 ? from_half(a.h[k]) : from_bf16(a.h[k]);
    return r;
}

template <bool FULL>
__device__ __forceinline__ void store4(void* p, int type, int i, int count, f4 v)
{
    if (type == BFSR_LIST_F32) {
        GLOBAL float* q = (GLOBAL float*)p + i;
        if (FULL || i + 4 <= count) *(GLOBAL f4u*)q = v;
        else for (int k = 0; k < 3; ++k) if (i + k < count) q[k] = v[k];
        return;
    }
    GLOBAL unsigned short* q = (GLOBAL unsigned short*)p + i;
    h4u h;
    for (int k = 0; k < 4; ++k) h[k] = type == BFSR_LIST_F16 ? to_half(v[k]) : to_bf16(v[k]);
    if (FULL || i + 4 <= count) *(GLOBAL h4u*)q = h;
    else for (int k = 0; k < 3; ++k) if (i + k < count) q[k] = h[k];
}

__device__ __forceinline__ void* at_element(const void* p, int type, long long i) { return (char*)p + i * (type == BFSR_LIST_F32 ? 4 : 2); }

// The larger magnitude, where a NaN on either side wins (fmax would drop it).
__device__ __forceinline__ double worse(double a, double b) { return (b > a || b != b) ? b : a; }

template <bool MAX>
__device__ __forceinline__ double join(double a, double b) { return MAX ? (a != a ? a : worse(a, b)) : a + b; }

// The join of one value of each thread, in an order that depends on nothing but the number of threads; thread 0 has it.
template <bool MAX>
__device__ __forceinline__ double block_join(double v)
{
    __shared__ double part[T / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<MAX>(v, __shfl_down(v, o, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int k = 1; k < T / 64; ++k) v = join<MAX>(v, part[k]);
    return v;
}

// Squares are formed and added in 64 bits: fp32's largest value squared overflows 32 bits, its smallest vanish, and a norm of finite gradients has to be finite.
// Bound by memory: two instructions an element for the conversion and the multiply-add.  Each wave takes chunks of its own, 16 bytes a load and a chunk's loads all under way
// at once; loads of 8 bytes one at a time kept 8 KB in flight per CU and reached 2.7 TB/s.
template <bool MAX>
__device__ __forceinline__ double take(double acc, float g) { return MAX ? join<true>(acc, (double)fabsf(g)) : fma((double)g, (double)g, acc); }

template <bool MAX, int TYPE, bool FULL>
__device__ __forceinline__ double take_chunk(double acc, const void* p, long long begin, int count)
{
    typedef typename Vec<TYPE>::type V;
    constexpr int N = Vec<TYPE>::N, U = CHUNK / (64 * N);
    const GLOBAL typename Vec<TYPE>::one* q = (const GLOBAL typename Vec<TYPE>::one*)p + begin;
    const int lane = threadIdx.x & 63;
    V g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * 64 + lane) * N;
        if (FULL || i + N <= count) g[u] = *(const GLOBAL V*)(q + i);
        else {
            g[u] = V{};
            for (int k = 0; k < N - 1; ++k) if (i + k < count) g[u][k] = q[i + k];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        for (int k = 0; k < N; ++k) acc = take<MAX>(acc, Vec<TYPE>::wide(g[u][k]));
    return acc;
}

template <bool MAX, int TYPE>
__device__ __forceinline__ double take_chunk(double acc, const void* p, long long begin, int count)
{
    return count == CHUNK ? take_chunk<MAX, TYPE, true>(acc, p, begin, count) : take_chunk<MAX, TYPE, false>(acc, p, begin, count);
}

template <bool MAX>
__global__ __launch_bounds__(T) void norm_parts_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, const void* const* __restrict__ other,
                                                       int col, int count, double* __restrict__ parts)
{
    double acc = 0.0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int c = blockIdx.x * WAVES + wave; c < count; c += gridDim.x * WAVES) {
        const int2 at = chunks[c];
        const Row& r = rows[at.x];
        const void* p = other ? other[at.x] : r.p[col];
        const int type = col ? r.type_g : r.type;
        const long long begin = (long long)at.y * CHUNK, left = r.n - begin;
        const int here = left < CHUNK ? (int)left : CHUNK;
        acc = type == BFSR_LIST_F32 ? take_chunk<MAX, BFSR_LIST_F32>(acc, p, begin, here) : type == BFSR_LIST_F16 ? take_chunk<MAX, BFSR_LIST_F16>(acc, p, begin, here)
                                                                                                                 : take_chunk<MAX, BFSR_LIST_BF16>(acc, p, begin, here);
    }
    acc = block_join<MAX>(acc);
    if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

struct Final {
    const double* parts; int count, max;       // the norm's parts, or none (count 0) ...
    const float* given; float* out;            // ... and the norm that the caller has instead; where it goes
    float max_norm;                            // < 0: no clipping
    float* share;                              // what the gradients are multiplied by
};

// The norm from its parts and the share min(1, max_norm / (norm + 1e-6)), in 64 bits: a NaN norm gives a NaN share, an infinite one 0, as the quotient does.
__device__ double finish(const Final& f)
{
    __shared__ double whole;
    double v = 0.0;
    if (f.given) v = (double)*f.given;
    else {
        for (int k = threadIdx.x; k < f.count; k += T) v = f.max ? join<true>(v, f.parts[k]) : v + f.parts[k];
        v = f.max ? block_join<true>(v) : sqrt(block_join<false>(v));
    }
    if (threadIdx.x == 0) {
        whole = v;
        if (f.out) *f.out = (float)v;
        if (f.share) {
            const double s = (double)f.max_norm / (v + 1e-6);
            *f.share = f.max_norm < 0.f ? 1.f : (float)(s > 1.0 ? 1.0 : s);
        }
    }
    __syncthreads();
    return whole;
}

__global__ __launch_bounds__(T) void norm_finish_kernel(Final f) { finish(f); }

template <bool FULL>
__device__ __forceinline__ void clip_chunk(const void* from, void* to, int type, int count, float s)
{
    const int lane = threadIdx.x & 63;
    constexpr int U = CHUNK / 256;
    Four g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) g[u] = load4<FULL>(from, type, (u * 64 + lane) * 4, count);
#pragma unroll
    for (int u = 0; u < U; ++u) store4<FULL>(to, type, (u * 64 + lane) * 4, count, floats(g[u], type) * s);
}

__global__ __launch_bounds__(T) void clip_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, int count, const float* __restrict__ share)
{
    const int c = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (c >= count) return;
    const int2 at = chunks[c];
    const Row& r = rows[at.x];
    const float s = *share;
    if (s == 1.f && r.p[0] == r.p[1]) return;                  // in place, and nothing to change
    const long long begin = (long long)at.y * CHUNK, left = r.n - begin;
    const void* from = at_element(r.p[0], r.type, begin);
    void* to = at_element(r.p[1], r.type, begin);
    if (left >= CHUNK) clip_chunk<true>(from, to, r.type, CHUNK, s);
    else clip_chunk<false>(from, to, r.type, (int)left, s);
}

struct Hyper { double lr, beta1, beta2, weight_decay; float eps; int decoupled, skip; const float* lr_at; };
struct Factors { float size, root, keep, go; };                // of one row: lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), 1 - lr decay, whether it is updated

// One workgroup: the norm, and each row's step count and factors.  Powers and quotients in 64 bits: 1 - beta2^t loses what 32 bits have for small t.
__global__ __launch_bounds__(T) void adam_begin_kernel(const Row* __restrict__ rows, int n, Final f, Hyper h, Factors* __restrict__ factors)
{
    double norm = 0.0;
    if (f.given || f.count) norm = finish(f);
    else if (threadIdx.x == 0) *f.share = 1.f;
    const bool go = !(h.skip && !(norm <= 1.7976931348623157e308));
    const double lr = h.lr_at ? (double)*h.lr_at : h.lr;
    for (int k = threadIdx.x; k < n; k += T) {
        const float t = *rows[k].step + 1.f;
        if (go) *rows[k].step = t;
        factors[k] = {(float)(lr / (1.0 - pow(h.beta1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(h.beta2, (double)t))),
                      (float)(1.0 - lr * h.weight_decay), go ? 1.f : 0.f};
    }
}

struct Rule { float share, b1, c1, b2, c2, wd, eps; bool add, keep; Factors f; };

template <bool FULL>
__device__ __forceinline__ void adam_chunk(void* pp, const void* gp, float* mp, float* vp, int type, int type_g, int count, const Rule& w)
{
    const int lane = threadIdx.x & 63;
    constexpr int U = 2;
    for (int j = 0; j < CHUNK && (FULL || j < count); j += U * 256) {
        Four p[U], g[U], m[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = j + (u * 64 + lane) * 4;
            p[u] = load4<FULL>(pp, type, i, count);
            g[u] = load4<FULL>(gp, type_g, i, count);
            m[u] = load4<FULL>(mp, BFSR_LIST_F32, i, count);
            v[u] = load4<FULL>(vp, BFSR_LIST_F32, i, count);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = j + (u * 64 + lane) * 4;
            f4 x = floats(p[u], type), y = floats(g[u], type_g), m1, v1;
            for (int k = 0; k < 4; ++k) {
                float d = y[k] * w.share;
                if (w.add) d = fmaf(w.wd, x[k], d);
                if (w.keep) x[k] *= w.f.keep;
                m1[k] = fmaf(w.b1, m[u].f[k], w.c1 * d);
                v1[k] = fmaf(w.b2, v[u].f[k], w.c2 * d * d);
                x[k] -= w.f.size * (m1[k] / fmaf(sqrtf(v1[k]), w.f.root, w.eps));
            }
            store4<FULL>(pp, type, i, count, x);
            store4<FULL>(mp, BFSR_LIST_F32, i, count, m1);
            store4<FULL>(vp, BFSR_LIST_F32, i, count, v1);
        }
    }
}

__global__ __launch_bounds__(T) void adam_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, const void* const* __restrict__ other, int count,
                                                 Hyper h, const Factors* __restrict__ factors, const float* __restrict__ share)
{
    const int c = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (c >= count) return;
    const int2 at = chunks[c];
    const Row& r = rows[at.x];
    const Factors f = factors[at.x];
    if (f.go == 0.f) return;
    const float wd = (float)h.weight_decay;
    const Rule w = {*share, (float)h.beta1, (float)(1.0 - h.beta1), (float)h.beta2, (float)(1.0 - h.beta2), wd, h.eps, wd != 0.f && !h.decoupled, wd != 0.f && h.decoupled, f};
    const long long begin = (long long)at.y * CHUNK, left = r.n - begin;
    void* p = at_element(r.p[0], r.type, begin);
    const void* g = at_element(other ? other[at.x] : r.p[1], r.type_g, begin);
    float* m = (float*)r.p[2] + begin;
    float* v = (float*)r.p[3] + begin;
    if (left >= CHUNK) adam_chunk<true>(p, g, m, v, r.type, r.type_g, CHUNK, w);
    else adam_chunk<false>(p, g, m, v, r.type, r.type_g, (int)left, w);
}

// ---- the table: rows and chunks travel to the device as kernel arguments.  No host buffer has to outlive the call, nothing waits for the stream, and a
// captured graph holds what it needs.
template <int COLS>
struct Entry { const void* p[COLS]; long long n; int types, first; };          // first: the row's first chunk
constexpr int ARGS = 3584;                                                     // bytes of a kernel's arguments that hold entries, of 4096
template <int COLS>
struct Entries { Entry<COLS> e[ARGS / sizeof(Entry<COLS>)]; };

template <int COLS>
__global__ __launch_bounds__(T) void list_write_kernel(Entries<COLS> all, int row0, int chunk, Row* __restrict__ rows, int2* __restrict__ chunks)
{
    const Entry<COLS>& e = all.e[blockIdx.x];
    const int row = row0 + blockIdx.x;
    if (threadIdx.x == 0) {
        Row r = {};
        r.p[0] = e.p[0];
        r.p[1] = e.p[COLS > 1 ? 1 : 0];
        if constexpr (COLS == 5) { r.p[2] = e.p[2]; r.p[3] = e.p[3]; r.step = (float*)e.p[4]; }
        r.n = e.n; r.type = e.types & 15; r.type_g = e.types >> 4;
        rows[row] = r;
    }
    const int count = (int)((e.n + chunk - 1) / chunk);
    for (int k = threadIdx.x; k < count; k += T) chunks[e.first + k] = make_int2(row, k);
}

template <int COLS>
int write_rows(const void* const* const* cols, const long long* sizes, const int* types, int n, int chunk, Row* rows, int2* chunks, hipStream_t st)
{
    constexpr int PER = ARGS / sizeof(Entry<COLS>);
    long long first = 0;
    for (int k = 0; k < n; k += PER) {
        Entries<COLS> all = {};
        const int m = n - k < PER ? n - k : PER;
        for (int j = 0; j < m; ++j) {
            for (int c = 0; c < COLS; ++c) all.e[j].p[c] = cols[c][k + j];
            all.e[j].n = sizes[k + j]; all.e[j].types = types[k + j]; all.e[j].first = (int)first;
            first += (sizes[k + j] + chunk - 1) / chunk;
        }
        list_write_kernel<COLS><<<m, T, 0, st>>>(all, k, chunk, rows, chunks);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

constexpr int POINTERS = 480;
struct Pointers { const void* p[POINTERS]; };
__global__ __launch_bounds__(512) void pointer_write_kernel(Pointers all, int n, const void** __restrict__ to)
{
    if ((int)threadIdx.x < n) to[threadIdx.x] = all.p[threadIdx.x];
}

bool good(const BfsrListArgs& a) { return a.rows && a.chunks && a.n > 0 && a.count >= 0 && a.count < (1 << 24) && a.chunk == CHUNK; }

int blocks_of(int count) { return (count + WAVES - 1) / WAVES; }
int parts_of(int count) { return blocks_of(count) < MAX_PARTS ? blocks_of(count) : MAX_PARTS; }

int launch_parts(const BfsrListArgs& a, int col, double* parts, hipStream_t st)
{
    if (!a.count) return 0;
    const auto k = a.max ? norm_parts_kernel<true> : norm_parts_kernel<false>;
    k<<<parts_of(a.count), T, 0, st>>>((const Row*)a.rows, (const int2*)a.chunks, (const void* const*)a.other, col, a.count, parts);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int bfsr_list_chunk(long long total) { return total < 0 ? -1 : CHUNK; }

extern "C" long long bfsr_list_work(int n) { return n < 0 ? -1 : (long long)MAX_PARTS * 8 + 16 + (long long)n * (long long)sizeof(Factors); }

extern "C" int bfsr_list_write(const void* const* const* cols, int ncols, const long long* sizes, const int* types, int n, int chunk, void* rows, void* chunks, void* stream)
{
    if (!cols || !sizes || !types || n <= 0 || chunk != CHUNK || !rows || !chunks) return -1;
    if (ncols != 1 && ncols != 2 && ncols != 5) return -1;
    long long count = 0;
    for (int k = 0; k < n; ++k) {
        const int t = types[k] & 15, g = types[k] >> 4;
        if (sizes[k] < 0 || t > BFSR_LIST_BF16 || g < 0 || g > BFSR_LIST_BF16) return -1;
        for (int c = 0; c < ncols; ++c)
            if (!cols[c] || (sizes[k] && !cols[c][k])) return -1;
        if (ncols == 5 && !cols[4][k]) return -1;
        count += (sizes[k] + chunk - 1) / chunk;
        if (count >= (1 << 24)) return -1;
    }
    hipStream_t st = (hipStream_t)stream;
    Row* r = (Row*)rows;
    int2* c = (int2*)chunks;
    return ncols == 1 ? write_rows<1>(cols, sizes, types, n, chunk, r, c, st) : ncols == 2 ? write_rows<2>(cols, sizes, types, n, chunk, r, c, st)
                                                                                           : write_rows<5>(cols, sizes, types, n, chunk, r, c, st);
}

extern "C" int bfsr_pointer_write(const void* const* from, int n, void* to, void* stream)
{
    if (!from || !to || n <= 0) return -1;
    for (int k = 0; k < n; k += POINTERS) {
        Pointers all = {};
        const int m = n - k < POINTERS ? n - k : POINTERS;
        for (int j = 0; j < m; ++j) all.p[j] = from[k + j];
        pointer_write_kernel<<<1, 512, 0, (hipStream_t)stream>>>(all, m, (const void**)to + k);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

extern "C" int bfsr_grad_norm(const BfsrListArgs* a, void* stream)
{
    if (!a || !good(*a) || !a->work || !a->norm) return -1;
    hipStream_t st = (hipStream_t)stream;
    double* parts = (double*)a->work;
    const int err = launch_parts(*a, 0, parts, st);
    if (err) return err;
    norm_finish_kernel<<<1, T, 0, st>>>(Final{parts, parts_of(a->count), a->max, nullptr, a->norm, -1.f, nullptr});
    return (int)hipGetLastError();
}

extern "C" int bfsr_clip_grads(const BfsrListArgs* a, float max_norm, void* stream)
{
    if (!a || !good(*a) || !a->work || !a->norm || !(max_norm >= 0.f)) return -1;
    hipStream_t st = (hipStream_t)stream;
    double* parts = (double*)a->work;
    float* share = (float*)(parts + MAX_PARTS);
    const int err = launch_parts(*a, 0, parts, st);
    if (err) return err;
    norm_finish_kernel<<<1, T, 0, st>>>(Final{parts, parts_of(a->count), a->max, nullptr, a->norm, max_norm, share});
    if (a->count) clip_kernel<<<blocks_of(a->count), T, 0, st>>>((const Row*)a->rows, (const int2*)a->chunks, a->count, share);
    return (int)hipGetLastError();
}

extern "C" int bfsr_adam_step(const BfsrListArgs* a, const BfsrAdamArgs* h, void* stream)
{
    if (!a || !h || !good(*a) || !a->work) return -1;
    if (!(h->beta1 >= 0. && h->beta1 < 1.) || !(h->beta2 >= 0. && h->beta2 < 1.) || !(h->eps >= 0.f) || !(h->weight_decay >= 0.)) return -1;
    hipStream_t st = (hipStream_t)stream;
    double* parts = (double*)a->work;
    float* share = (float*)(parts + MAX_PARTS);
    Factors* factors = (Factors*)(share + 4);
    const bool norm = h->max_norm >= 0.f || h->skip_nonfinite;
    const bool own = norm && !h->given_norm;
    if (norm && !a->norm) return -1;
    if (own) {
        const int err = launch_parts(*a, 1, parts, st);
        if (err) return err;
    }
    const Hyper hy = {h->lr, h->beta1, h->beta2, h->weight_decay, h->eps, h->decoupled, h->skip_nonfinite, h->lr_at};
    adam_begin_kernel<<<1, T, 0, st>>>((const Row*)a->rows, a->n, Final{parts, own ? parts_of(a->count) : 0, a->max, norm ? h->given_norm : nullptr, norm ? a->norm : nullptr,
                                       h->max_norm >= 0.f ? h->max_norm : -1.f, share}, hy, factors);
    if (a->count) adam_kernel<<<blocks_of(a->count), T, 0, st>>>((const Row*)a->rows, (const int2*)a->chunks, (const void* const*)a->other, a->count, hy, factors, share);
    return (int)hipGetLastError();
}
