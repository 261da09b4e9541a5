// tensor_list.hip -- the end of a training step over a LIST of tensors, in one or two launches however many tensors the list has (and more where a call writes its table or brings
// other gradients: one for each 149, 112 or 64 rows of one, two or five columns, one for each 480 addresses):
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
#include <atomic>
#include <new>
#include "../../include/bfsr_hip.h"
#include "launch_util.h"

namespace {

constexpr int T = 256;                        // threads of a workgroup that updates
constexpr int TN = 1024;                      // threads of one that sums
constexpr int CHUNK = 2048;                   // elements of a chunk
constexpr int PARTS = 256;                    // partial results of a norm at most, one for each of its workgroups: one a CU, and four a lane for the wave that joins them
constexpr int ALONE = 48;                     // chunks up to which one workgroup finds a norm by itself: 8.0 us a call against 10.7 with a second launch; at 128 chunks 11.7 and 10.9
// ... and up to which (and bytes of tensors) it clips a list, or takes a step, in the same launch.  One workgroup / a launch for each part, us a call among others and (waited for):
// clipping 24 full chunks 7.6 (22.0) / 10.2 (21.0), 42 chunks of 0.5 MB 9.9 (24.1) / 10.6 (21.4);  a step of 11 chunks of 118 KB 6.6 (20.1) / 9.7 (20.5), clipped
// 8.5 (23.6) / 11.7 (22.4), of 12 full chunks 10.2 (24.0) / 9.4 (20.2).  Above, one CU's share of the bandwidth counts for more than a launch.
constexpr int ALONE_CLIP = 32, ALONE_CLIP_BYTES = 384 << 10, ALONE_ADAM = 12, ALONE_ADAM_BYTES = 192 << 10;
constexpr int ALONE_ROWS = 256;               // rows that such a step has room for
// Bytes of tensors up to which a call goes through the 256 MB cache that the card shares.  Reads past it still find there what others left.
// An update: half of the cache.  Lists in turn, the usual way / past the cache: 3 of 73 MB 20.4 / 25.2 us, 3 of 200 MB 70 / 62 us; one of 160 MB again and again 54 / 61 us, and
// with 1 GB of other work in between 74 / 64 us.
constexpr long long CACHE = 128ll << 20;
// A norm by itself, 64 MB: again and again 14.7 / 15.6 us, with other work in between 30 / 18 us; 32 MB: 15.3 / 16.0 and 19 / 13 us.
constexpr long long CACHE_NORM = 24ll << 20;

struct Row { const void* p[4]; float* step; long long n; int type, type_g; long long pad; };      // BFSR_LIST_ROW bytes
static_assert(sizeof(Row) == BFSR_LIST_ROW, "the row's size is part of the interface");

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short h2 __attribute__((ext_vector_type(2)));
typedef unsigned short h4 __attribute__((ext_vector_type(4)));
typedef unsigned short h8 __attribute__((ext_vector_type(8)));
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

// STREAM: past the shared cache, for lists that it cannot hold anyway.  Read that way 614 MB came in at 6.4 TB/s, the usual way at 4.1; what follows on a list
// that fits (an update after a norm, the next step) found it in the cache the usual way and lost 10 to 20 % the other.
// (written out for each type: a template's argument would lose the alignment that the typedefs carry)
#define ACCESS(V, ONE, LOAD, STORE) \
    template <bool STREAM> __device__ __forceinline__ V LOAD(const GLOBAL ONE* p) \
    { if constexpr (STREAM) return __builtin_nontemporal_load((const GLOBAL V##u*)p); else return *(const GLOBAL V##u*)p; } \
    template <bool STREAM> __device__ __forceinline__ void STORE(GLOBAL ONE* p, V v) \
    { if constexpr (STREAM) __builtin_nontemporal_store((V##u)v, (GLOBAL V##u*)p); else *(GLOBAL V##u*)p = v; }
ACCESS(f4, float, load16, store16)
ACCESS(h8, unsigned short, load16, store16)
ACCESS(h4, unsigned short, load8, store8)

// The elements of a type, N to a load of 16 bytes.
template <int TYPE> struct Vec;
template <> struct Vec<BFSR_LIST_F32> { typedef f4 type; typedef float one; static constexpr int N = 4; __device__ static float wide(float f) { return f; } __device__ static float narrow(float f) { return f; } };
template <> struct Vec<BFSR_LIST_F16> { typedef h8 type; typedef unsigned short one; static constexpr int N = 8; __device__ static float wide(unsigned short h) { return from_half(h); } __device__ static unsigned short narrow(float f) { return to_half(f); } };
template <> struct Vec<BFSR_LIST_BF16> { typedef h8 type; typedef unsigned short one; static constexpr int N = 8; __device__ static float wide(unsigned short h) { return from_bf16(h); } __device__ static unsigned short narrow(float f) { return to_bf16(f); } };

// Four elements of a tensor of `type` from element i on.
struct Four { f4 f; h4 h; };

template <bool STREAM>
__device__ __forceinline__ Four load4(const void* p, int type, int i)
{
    Four r;
    if (type == BFSR_LIST_F32) r.f = load16<STREAM>((const GLOBAL float*)p + i);
    else r.h = load8<STREAM>((const GLOBAL unsigned short*)p + i);
    return r;
}

__device__ __forceinline__ f4 floats(Four a, int type)
{
    if (type == BFSR_LIST_F32) return a.f;
    f4 r;
    for (int k = 0; k < 4; ++k) r[k] = type == BFSR_LIST_F16 ? from_half(a.h[k]) : from_bf16(a.h[k]);
    return r;
}

template <bool STREAM>
__device__ __forceinline__ void store4(void* p, int type, int i, f4 v)
{
    if (type == BFSR_LIST_F32) return store16<STREAM>((GLOBAL float*)p + i, v);
    h4 h;
    for (int k = 0; k < 4; ++k) h[k] = type == BFSR_LIST_F16 ? to_half(v[k]) : to_bf16(v[k]);
    store8<STREAM>((GLOBAL unsigned short*)p + i, h);
}

__device__ __forceinline__ float load1(const void* p, int type, int i)
{
    if (type == BFSR_LIST_F32) return ((const GLOBAL float*)p)[i];
    const unsigned short h = ((const GLOBAL unsigned short*)p)[i];
    return type == BFSR_LIST_F16 ? from_half(h) : from_bf16(h);
}

__device__ __forceinline__ void store1(void* p, int type, int i, float v)
{
    if (type == BFSR_LIST_F32) ((GLOBAL float*)p)[i] = v;
    else ((GLOBAL unsigned short*)p)[i] = type == BFSR_LIST_F16 ? to_half(v) : to_bf16(v);
}

// Elements of the chunk that begins at element `begin`.
__device__ __forceinline__ int left_in(const Row& r, long long begin) { return r.n - begin < CHUNK ? (int)(r.n - begin) : CHUNK; }

__device__ __forceinline__ void* at_element(const void* p, int type, long long i) { return (char*)p + i * (type == BFSR_LIST_F32 ? 4 : 2); }

// The sum of squares, or the largest magnitude, of what a thread has seen.
// Squares are formed and added in 64 bits: fp32's largest value squared overflows 32 bits, its smallest vanish, and a norm that 32 bits hold has to be found.
// Magnitudes are compared as whole numbers: without the sign, larger bits are a larger number, infinity is above them all and NaN above that, so a NaN stays (fmax
// would drop it), at one instruction an element; compared in 64 bits as the sums are, 38 M elements took 20 us and not the 12 that memory needs.
template <bool MAX> struct Acc;
template <> struct Acc<false> {
    double a = 0.0;
    __device__ __forceinline__ void join(double b) { a += b; }
    template <int TYPE> __device__ __forceinline__ void take(typename Vec<TYPE>::type g)
    {
#pragma unroll
        for (int k = 0; k < Vec<TYPE>::N; ++k) { const double d = (double)Vec<TYPE>::wide(g[k]); a = fma(d, d, a); }
    }
    __device__ __forceinline__ double part() const { return a; }
    // What 32 bits cannot hold is infinite, as in the norm that the caller gets: whether a list is clipped and skipped as one or by the norm of several is the same then.
    __device__ static double whole(double sum)
    {
        const double norm = sqrt(sum);
        return isinf((float)norm) ? (double)(float)norm : norm;
    }
};
template <> struct Acc<true> {
    unsigned a = 0;
    __device__ __forceinline__ void join(double b) { const unsigned u = __float_as_uint((float)b); a = max(a, u); }
    template <int TYPE> __device__ __forceinline__ void take(typename Vec<TYPE>::type g)
    {
        if constexpr (TYPE == BFSR_LIST_F32) {
            const auto bits = [](float f) { return __float_as_uint(f) & 0x7fffffffu; };
            a = max(max(a, max(bits(g.x), bits(g.y))), max(bits(g.z), bits(g.w)));
        } else {
            g &= (unsigned short)0x7fff;
            const h4 h = __builtin_elementwise_max(g.lo, g.hi);
            const h2 l = __builtin_elementwise_max(h.lo, h.hi);
            a = max(a, __float_as_uint(Vec<TYPE>::wide(l.x > l.y ? l.x : l.y)));
        }
    }
    __device__ __forceinline__ double part() const { return (double)__uint_as_float(a); }
    __device__ static double whole(double most) { return most; }
};

// The join over a wave, in an order that depends on nothing; every lane has it.
template <bool MAX>
__device__ __forceinline__ double wave_join(double v)
{
    Acc<MAX> acc;
    acc.join(v);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc.join(__shfl_xor(acc.part(), o, 64));
    return acc.part();
}

// One chunk for one wave, 16 bytes a load and all of them under way at once.  Bound by memory; with loads of 8 bytes one at a time 8 KB were in flight per CU
// and 2.7 TB/s came in.
template <bool MAX, bool STREAM, int TYPE>
__device__ __forceinline__ void take_chunk(Acc<MAX>& acc, const void* p, long long begin, int count)
{
    typedef typename Vec<TYPE>::type V;
    constexpr int N = Vec<TYPE>::N, U = CHUNK / (64 * N);
    const GLOBAL typename Vec<TYPE>::one* q = (const GLOBAL typename Vec<TYPE>::one*)p + begin;
    const int lane = threadIdx.x & 63;
    V g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * 64 + lane) * N;
        g[u] = V{};
        if (i + N <= count) g[u] = load16<STREAM>(q + i);
    }
    if (lane < count % N) {                               // what does not fill a load: an element a lane
        V last = {};
        last[0] = q[count / N * N + lane];
        acc.template take<TYPE>(last);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) acc.template take<TYPE>(g[u]);
}

// Where a norm comes from and goes, and what the gradients are multiplied by.
struct Norm {
    const double* parts; int count, max;       // its parts, or none (count 0) ...
    const float* given; float* out;            // ... and the norm that the caller has instead; where it is written
    float max_norm;                            // < 0: no clipping
};

// The norm from its parts.  Every wave of an update does this for itself, while its loads are under way: 2 KB that its L2 has, and no waiting for other waves.  A launch in between
// that does it once took 2 to 5 us.
__device__ __forceinline__ double whole(const Norm& f)
{
    if (f.given) return (double)*f.given;
    double v[PARTS / 64];
#pragma unroll
    for (int k = 0; k < PARTS / 64; ++k) { const int i = k * 64 + (threadIdx.x & 63); v[k] = i < f.count ? f.parts[i] : 0.0; }
    if (f.max) {
        Acc<true> acc;
        for (int k = 0; k < PARTS / 64; ++k) acc.join(v[k]);
        return Acc<true>::whole(wave_join<true>(acc.part()));
    }
    Acc<false> acc;
    for (int k = 0; k < PARTS / 64; ++k) acc.join(v[k]);
    return Acc<false>::whole(wave_join<false>(acc.part()));
}

// min(1, max_norm / (norm + 1e-6)): a NaN norm gives NaN, an infinite one 0, as the quotient does.
__device__ __forceinline__ float share_of(const Norm& f, double norm)
{
    const double s = (double)f.max_norm / (norm + 1e-6);
    return f.max_norm < 0.f ? 1.f : (float)(s > 1.0 ? 1.0 : s);
}

struct Hyper { double lr, beta1, beta2, weight_decay; float eps; int decoupled, skip; const float* lr_at; };
struct Factors { float size, root, decay, had; };              // of one row: lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), lr times the decay, the count before

// b^t for a whole number t by squaring, in 64 bits (a count is at most 2^24, where float stops counting): 1 - b^t loses what 32 bits have for small t.
__device__ __forceinline__ double power(double b, unsigned t)
{
    double r = 1.0;
    for (; t; t >>= 1) { if (t & 1) r *= b; b *= b; }
    return r;
}

__device__ __forceinline__ void begin_row(const Row& r, const Hyper& h, Factors* f)
{
    const float had = *r.step, t = had + 1.f;
    const double lr = h.lr_at ? (double)*h.lr_at : h.lr;
    *r.step = t;
    *f = {(float)(lr / (1.0 - power(h.beta1, (unsigned)t))), (float)(1.0 / sqrt(1.0 - power(h.beta2, (unsigned)t))), (float)(lr * h.weight_decay), had};
}

// A thread a row: 2.5 us for 8 rows, 4.8 for 702, which is three loads that depend on each other.
__global__ __launch_bounds__(T) void adam_begin_kernel(const Row* __restrict__ rows, int n, Hyper h, Factors* __restrict__ factors)
{
    const int k = blockIdx.x * T + threadIdx.x;
    if (k < n) begin_row(rows[k], h, factors + k);
}

// The part of workgroup `index` of `of` of them (of TN threads), for every thread of it.  All its reads have been made when it is known.
template <bool MAX, bool STREAM>
__device__ __forceinline__ double sum_chunks(const Row* __restrict__ rows, const int2* __restrict__ chunks, const void* const* __restrict__ other, int col, int count,
                                             int index, int of)
{
    constexpr int WAVES = TN / 64;
    __shared__ double part[WAVES];
    Acc<MAX> acc;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int c = index * WAVES + wave; c < count; c += of * WAVES) {
        const int2 at = chunks[c];
        const Row& r = rows[at.x];
        const void* p = other ? other[at.x] : r.p[col];
        const int type = col ? r.type_g : r.type;
        const long long begin = (long long)at.y * CHUNK;
        const int here = left_in(r, begin);
        if (type == BFSR_LIST_F32) take_chunk<MAX, STREAM, BFSR_LIST_F32>(acc, p, begin, here);
        else if (type == BFSR_LIST_F16) take_chunk<MAX, STREAM, BFSR_LIST_F16>(acc, p, begin, here);
        else take_chunk<MAX, STREAM, BFSR_LIST_BF16>(acc, p, begin, here);
    }
    const double mine = wave_join<MAX>(acc.part());
    if ((threadIdx.x & 63) == 0) part[wave] = mine;
    __syncthreads();
    return wave_join<MAX>((threadIdx.x & 63) < WAVES ? part[threadIdx.x & 63] : 0.0);
}

// Memory bounds it: 614 MB of fp32 in 93 us (6.6 TB/s, streaming), 77 MB of fp16 in 14 us (5.4), 18 MB of fp32 in 6.0 us and 33 MB of bf16 in 9.8.  Of
// those middle lists its start and end are a part, and idle CUs (2280 chunks at 16 a workgroup occupy 143 of them) and the rounds of a wave, one chunk after the other, are the rest.
// One part of the norm for each of the first `sums` workgroups (with one, the norm itself); those behind them, if any, begin a step of Adam.
template <bool MAX, bool STREAM>
__global__ __launch_bounds__(TN) void norm_parts_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, const void* const* __restrict__ other,
                                                        int col, int count, int sums, double* __restrict__ parts, float* __restrict__ out, int n, Hyper h,
                                                        Factors* __restrict__ factors)
{
    if ((int)blockIdx.x >= sums) {
        const int k = ((int)blockIdx.x - sums) * TN + threadIdx.x;
        if (k < n) begin_row(rows[k], h, factors + k);
        return;
    }
    const double all = sum_chunks<MAX, STREAM>(rows, chunks, other, col, count, blockIdx.x, sums);
    if (threadIdx.x == 0) {
        if (out) *out = (float)Acc<MAX>::whole(all);
        else parts[blockIdx.x] = all;
    }
}

// 1.5 us; 3.8 where what came before has emptied the caches.
__global__ __launch_bounds__(64) void norm_finish_kernel(Norm f)
{
    const double norm = whole(f);
    if (threadIdx.x == 0) *f.out = (float)norm;
}

template <bool STREAM, int TYPE, bool FULL, class SHARE>
__device__ __forceinline__ void clip_chunk(const SHARE& share, const void* from, void* to, int count)
{
    typedef typename Vec<TYPE>::type V;
    constexpr int N = Vec<TYPE>::N, U = CHUNK / (64 * N);
    const GLOBAL typename Vec<TYPE>::one* p = (const GLOBAL typename Vec<TYPE>::one*)from;
    GLOBAL typename Vec<TYPE>::one* q = (GLOBAL typename Vec<TYPE>::one*)to;
    const int lane = threadIdx.x & 63;
    V g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * 64 + lane) * N;
        if (FULL || i + N <= count) g[u] = load16<STREAM>(p + i);
    }
    const bool more = !FULL && lane < count % N;                   // what does not fill a load: an element a lane
    const int last = count / N * N + lane;
    typename Vec<TYPE>::one e = {};
    if (more) e = p[last];
    const float s = share();                                       // with the loads under way
    if (s == 1.f && from == to) return;                            // in place, and nothing to change
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * 64 + lane) * N;
#pragma unroll
        for (int k = 0; k < N; ++k) g[u][k] = Vec<TYPE>::narrow(Vec<TYPE>::wide(g[u][k]) * s);
        if (FULL || i + N <= count) store16<STREAM>(q + i, g[u]);
    }
    if (more) q[last] = Vec<TYPE>::narrow(Vec<TYPE>::wide(e) * s);
}

template <bool STREAM, class SHARE>
__device__ __forceinline__ void clip_one(const Row* __restrict__ rows, const int2 at, const SHARE& share)
{
    const Row& r = rows[at.x];
    const long long begin = (long long)at.y * CHUNK;
    const int left = left_in(r, begin);
    const void* from = at_element(r.p[0], r.type, begin);
    void* to = at_element(r.p[1], r.type, begin);
    const bool full = left == CHUNK;
    if (r.type == BFSR_LIST_F32) full ? clip_chunk<STREAM, BFSR_LIST_F32, true>(share, from, to, left) : clip_chunk<STREAM, BFSR_LIST_F32, false>(share, from, to, left);
    else if (r.type == BFSR_LIST_F16) full ? clip_chunk<STREAM, BFSR_LIST_F16, true>(share, from, to, left) : clip_chunk<STREAM, BFSR_LIST_F16, false>(share, from, to, left);
    else full ? clip_chunk<STREAM, BFSR_LIST_BF16, true>(share, from, to, left) : clip_chunk<STREAM, BFSR_LIST_BF16, false>(share, from, to, left);
}

// One chunk for each wave, and then the wave ends: one that went on to another chunk would wait for its stores before the next loads count as arrived.
// Chunks are taken from the end, where the cache holds what the norm has read last.  Memory bounds it: 307 MB of bf16 read and written in 98 us (6.2 TB/s), 18 MB of fp32 in 7.6.
template <bool STREAM>
__global__ __launch_bounds__(T) void clip_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, int count, Norm f)
{
    const int c = count - 1 - (int)blockIdx.x * (T / 64) - __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (c < 0) return;
    clip_one<STREAM>(rows, chunks[c], [&] {
        const double norm = whole(f);
        if (blockIdx.x == 0 && threadIdx.x == 0) *f.out = (float)norm;
        return share_of(f, norm);
    });
}

// A short list in one workgroup: the norm, and then the clipping of what its caches still hold.
template <bool MAX>
__global__ __launch_bounds__(TN) void clip_alone_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, int count, Norm f)
{
    const double norm = Acc<MAX>::whole(sum_chunks<MAX, false>(rows, chunks, nullptr, 0, count, 0, 1));
    if (threadIdx.x == 0) *f.out = (float)norm;
    const float s = share_of(f, norm);
    for (int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); c < count; c += TN / 64) clip_one<false>(rows, chunks[c], [=] { return s; });
}

struct Rule { float b1, c1, b2, c2, wd, eps; bool add, apart; Factors f; };

// Decoupled decay goes into the update before that is taken off: 1 - lr decay has 24 bits, of which a small decay leaves few or none (of 1e-6 it made 1.013e-6, in every step).
__device__ __forceinline__ void adam_element(const Rule& w, float share, float& p, float g, float& m, float& v)
{
    float d = g * share;
    if (w.add) d = fmaf(w.wd, p, d);
    m = fmaf(w.b1, m, w.c1 * d);
    v = fmaf(w.b2, v, w.c2 * d * d);
    const float step = m / fmaf(sqrtf(v), w.f.root, w.eps);
    p -= w.apart ? fmaf(w.f.size, step, w.f.decay * p) : w.f.size * step;
}

// One chunk for T threads; `share`: what its gradients are multiplied by, below 0 where the step is skipped.
template <bool STREAM, class SHARE>
__device__ __forceinline__ void adam_chunk(const SHARE& share_of_step, void* pp, const void* gp, float* mp, float* vp, int type, int type_g, int count, const Rule& w)
{
    constexpr int U = CHUNK / (T * 4), F32 = BFSR_LIST_F32;
    const int t = threadIdx.x & (T - 1);
    Four p[U], g[U], m[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * T + t) * 4;
        if (i + 4 <= count) {
            p[u] = load4<STREAM>(pp, type, i);
            g[u] = load4<STREAM>(gp, type_g, i);
            m[u] = load4<STREAM>(mp, F32, i);
            v[u] = load4<STREAM>(vp, F32, i);
        }
    }
    const float share = share_of_step();                           // with the loads under way
    if (share < 0.f) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * T + t) * 4;
        if (i + 4 <= count) {
            f4 x = floats(p[u], type), y = floats(g[u], type_g), m1 = m[u].f, v1 = v[u].f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float a = x[k], b = m1[k], c = v1[k];
                adam_element(w, share, a, y[k], b, c);
                x[k] = a; m1[k] = b; v1[k] = c;
            }
            store4<STREAM>(pp, type, i, x);
            store4<STREAM>(mp, F32, i, m1);
            store4<STREAM>(vp, F32, i, v1);
        }
    }
    if (t < (count & 3)) {                          // what does not fill a load
        const int i = (count & ~3) + t;
        float a = load1(pp, type, i), b = mp[i], c = vp[i];
        adam_element(w, share, a, load1(gp, type_g, i), b, c);
        store1(pp, type, i, a);
        mp[i] = b;
        vp[i] = c;
    }
}

template <bool STREAM, class SHARE>
__device__ __forceinline__ void adam_one(const Row* __restrict__ rows, const int2 at, const void* const* __restrict__ other, const Hyper& h, const Factors& factors,
                                         const SHARE& share)
{
    Rule w = {(float)h.beta1, (float)(1.0 - h.beta1), (float)h.beta2, (float)(1.0 - h.beta2), (float)h.weight_decay, h.eps};
    w.add = w.wd != 0.f && !h.decoupled;
    w.apart = w.wd != 0.f && h.decoupled;
    w.f = factors;
    const Row& r = rows[at.x];
    const long long begin = (long long)at.y * CHUNK;
    void* p = at_element(r.p[0], r.type, begin);
    const void* g = at_element(other ? other[at.x] : r.p[1], r.type_g, begin);
    adam_chunk<STREAM>(share, p, g, (float*)r.p[2] + begin, (float*)r.p[3] + begin, r.type, r.type_g, left_in(r, begin), w);
}

// The share of a step, or -1 where it is skipped: its norm is infinite or NaN, and the caller asked for that.
__device__ __forceinline__ float share_of_step(const Norm& f, const Hyper& h, double norm) { return h.skip && !isfinite(norm) ? -1.f : share_of(f, norm); }

// One chunk for each workgroup: two loads of 16 bytes from each of four arrays under way a thread, about fifty instructions an element, a division and a root among them.  Memory bounds
// it: 153 M fp32 parameters (28 bytes each, none moved twice) in 711 us (6.0 TB/s), 16.7 M bf16 ones (22 bytes) in 62 us (5.9); 512 threads a chunk 2 % less to 2 % more.
// The workgroup behind the chunks sees to the norm's output, and to the counts of a step that is skipped.
template <bool STREAM>
__global__ __launch_bounds__(T) void adam_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, const void* const* __restrict__ other, int count, int n,
                                                 Norm f, Hyper h, const Factors* __restrict__ factors)
{
    const int c = count - 1 - (int)blockIdx.x;
    if (c < 0) {
        if (!f.out) return;
        const double norm = whole(f);
        if (threadIdx.x == 0) *f.out = (float)norm;
        if (share_of_step(f, h, norm) < 0.f)
            for (int k = threadIdx.x; k < n; k += T) *rows[k].step = factors[k].had;
        return;
    }
    const int2 at = chunks[c];
    adam_one<STREAM>(rows, at, other, h, factors[at.x], [&] { return f.out ? share_of_step(f, h, whole(f)) : 1.f; });
}

// A short list in one workgroup: the counts, the norm if there is to be one, and the update of what its caches still hold.
template <bool MAX>
__global__ __launch_bounds__(TN) void adam_alone_kernel(const Row* __restrict__ rows, const int2* __restrict__ chunks, const void* const* __restrict__ other, int count, int n,
                                                        Norm f, Hyper h)
{
    __shared__ Factors factors[ALONE_ROWS];
    const int k = threadIdx.x;
    if (k < n) begin_row(rows[k], h, factors + k);
    float share = 1.f;
    if (f.out) {
        const double norm = f.given ? (double)*f.given : Acc<MAX>::whole(sum_chunks<MAX, false>(rows, chunks, other, 1, count, 0, 1));
        if (k == 0) *f.out = (float)norm;
        share = share_of_step(f, h, norm);
        if (share < 0.f) {
            if (k < n) *rows[k].step = factors[k].had;
            return;
        }
    }
    __syncthreads();
    for (int c = __builtin_amdgcn_readfirstlane(k / T); c < count; c += TN / T) {
        const int2 at = chunks[c];
        adam_one<false>(rows, at, other, h, factors[at.x], [=] { return share; });
    }
}

// ---- the table: rows and chunks travel to the device as kernel arguments.  No host buffer has to outlive the call, nothing waits for the stream, and a
// captured graph of a table made in it holds what it needs.  A launch takes 149 rows (one column), 112 (two) or 64 (five) and 2.4 us.
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

bool good(const BfsrListArgs& a) { return a.rows && a.chunks && a.n > 0 && a.count >= 0 && a.count < (1 << 24) && a.chunk == CHUNK && a.bytes >= 0; }

int sums_of(int count) { const int w = TN / 64, b = (count + w - 1) / w; return b < 1 ? 1 : b < PARTS ? b : PARTS; }

// Whether a call streams its tensors past the cache.
bool streams(const BfsrListArgs& a, long long bound) { return a.bytes > bound; }

// The parts of a norm; `out`: the norm itself, which one workgroup finds. `h`: with them, the beginning of a step of Adam.
int launch_parts(const BfsrListArgs& a, int col, bool stream, int sums, float* out, const Hyper* h, Factors* factors, hipStream_t st)
{
    const auto k = a.max ? stream ? norm_parts_kernel<true, true> : norm_parts_kernel<true, false> : stream ? norm_parts_kernel<false, true> : norm_parts_kernel<false, false>;
    k<<<sums + (h ? (a.n + TN - 1) / TN : 0), TN, 0, st>>>((const Row*)a.rows, (const int2*)a.chunks, h ? (const void* const*)a.other : nullptr, col, a.count, sums, (double*)a.work, out, a.n,
                                                        h ? *h : Hyper{}, factors);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int bfsr_list_chunk(long long total) { return total < 0 ? -1 : CHUNK; }

extern "C" long long bfsr_list_work(int n) { return n < 0 ? -1 : (long long)PARTS * 8 + (long long)n * (long long)sizeof(Factors); }

extern "C" long long bfsr_norm_work(int count) { return count < 0 ? -1 : count <= ALONE ? 0 : PARTS * 8; }

extern "C" int bfsr_list_write(const void* const* const* cols, int ncols, const long long* sizes, const int* types, int n, int chunk, void* rows, void* chunks, void* stream)
{
    if (!cols || !sizes || !types || n <= 0 || chunk != CHUNK || !rows || !chunks) return -1;
    if (ncols != 1 && ncols != 2 && ncols != 5) return -1;
    long long count = 0;
    for (int k = 0; k < n; ++k) {
        const int t = types[k] & 15, g = types[k] >> 4;
        if (sizes[k] < 0 || sizes[k] > ((long long)CHUNK << 24) || t > BFSR_LIST_BF16 || g < 0 || g > BFSR_LIST_BF16) return -1;
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
    if (!a || !good(*a) || !a->norm || (a->count > ALONE && !a->work)) return -1;
    hipStream_t st = (hipStream_t)stream;
    if (a->count <= ALONE) return launch_parts(*a, 0, false, 1, a->norm, nullptr, nullptr, st);
    const int sums = sums_of(a->count), err = launch_parts(*a, 0, streams(*a, CACHE_NORM), sums, nullptr, nullptr, nullptr, st);
    if (err) return err;
    norm_finish_kernel<<<1, 64, 0, st>>>(Norm{(const double*)a->work, sums, a->max, nullptr, a->norm, -1.f});
    return (int)hipGetLastError();
}

extern "C" int bfsr_clip_grads(const BfsrListArgs* a, float max_norm, void* stream)
{
    if (!a || !good(*a) || !a->work || !a->norm || !(max_norm >= 0.f)) return -1;
    hipStream_t st = (hipStream_t)stream;
    const Norm one = {nullptr, 0, a->max, nullptr, a->norm, max_norm};
    if (!a->count || (a->count <= ALONE_CLIP && a->bytes <= ALONE_CLIP_BYTES)) {
        (a->max ? clip_alone_kernel<true> : clip_alone_kernel<false>)<<<1, TN, 0, st>>>((const Row*)a->rows, (const int2*)a->chunks, a->count, one);
        return (int)hipGetLastError();
    }
    const bool past = streams(*a, CACHE);
    const int err = launch_parts(*a, 0, past, sums_of(a->count), nullptr, nullptr, nullptr, st), per = T / 64;
    if (err) return err;
    (past ? clip_kernel<true> : clip_kernel<false>)<<<(a->count + per - 1) / per, T, 0, st>>>((const Row*)a->rows, (const int2*)a->chunks, a->count,
                                                   Norm{(const double*)a->work, sums_of(a->count), a->max, nullptr, a->norm, max_norm});
    return (int)hipGetLastError();
}

extern "C" int bfsr_adam_step(const BfsrListArgs* a, const BfsrAdamArgs* h, void* stream)
{
    if (!a || !h || !good(*a) || !a->work) return -1;
    if (!(h->beta1 >= 0. && h->beta1 < 1.) || !(h->beta2 >= 0. && h->beta2 < 1.) || !(h->eps >= 0.f) || !(h->weight_decay >= 0.) || h->max_norm != h->max_norm) return -1;
    hipStream_t st = (hipStream_t)stream;
    Factors* factors = (Factors*)((double*)a->work + PARTS);
    const bool norm = h->max_norm >= 0.f || h->skip_nonfinite, own = norm && !h->given_norm;
    if (norm && !a->norm) return -1;
    const Hyper hy = {h->lr, h->beta1, h->beta2, h->weight_decay, h->eps, h->decoupled, h->skip_nonfinite, h->lr_at};
    const float* given = norm ? h->given_norm : nullptr;
    const float max_norm = h->max_norm >= 0.f ? h->max_norm : -1.f;
    if (a->count <= ALONE_ADAM && a->bytes <= ALONE_ADAM_BYTES && a->n <= ALONE_ROWS) {
        (a->max ? adam_alone_kernel<true> : adam_alone_kernel<false>)<<<1, TN, 0, st>>>((const Row*)a->rows, (const int2*)a->chunks, (const void* const*)a->other, a->count, a->n,
                                                                                       Norm{nullptr, 0, a->max, given, norm ? a->norm : nullptr, max_norm}, hy);
        return (int)hipGetLastError();
    }
    const bool past = streams(*a, CACHE);
    int err;
    if (own) err = launch_parts(*a, 1, past, sums_of(a->count), nullptr, &hy, factors, st);
    else {
        adam_begin_kernel<<<(a->n + T - 1) / T, T, 0, st>>>((const Row*)a->rows, a->n, hy, factors);
        err = (int)hipGetLastError();
    }
    if (err) return err;
    (past ? adam_kernel<true> : adam_kernel<false>)<<<a->count + 1, T, 0, st>>>((const Row*)a->rows, (const int2*)a->chunks, (const void* const*)a->other, a->count, a->n,
                                                   Norm{(const double*)a->work, own ? sums_of(a->count) : 0, a->max, given, norm ? a->norm : nullptr, max_norm}, hy, factors);
    return (int)hipGetLastError();
}

// ---- the life of a captured graph.  The graph owns a reference to a ticket, and so does every executable made from it; the runtime says when the last one is gone, on a thread of
// its choice and perhaps at the process's end, so that notice sets a flag in plain memory and nothing else.
extern "C" int bfsr_capture_ticket(void* stream, void** ticket)
{
    if (!ticket) return -1;
    *ticket = nullptr;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    hipGraph_t graph = nullptr;
    hipError_t err = hipStreamGetCaptureInfo_v2((hipStream_t)stream, &status, nullptr, &graph, nullptr, nullptr);
    if (err != hipSuccess || status != hipStreamCaptureStatusActive || !graph) return (int)err;
    std::atomic<int>* gone = new (std::nothrow) std::atomic<int>(0);
    if (!gone) return (int)hipErrorOutOfMemory;
    hipUserObject_t object = nullptr;
    err = hipUserObjectCreate(&object, gone, [](void* flag) { ((std::atomic<int>*)flag)->store(1, std::memory_order_release); }, 1, hipUserObjectNoDestructorSync);
    if (err != hipSuccess) { delete gone; return (int)err; }
    err = hipGraphRetainUserObject(graph, object, 1, hipGraphUserObjectMove);
    if (err != hipSuccess) return (int)err;                        // the flag stays the object's
    *ticket = gone;
    return 0;
}

extern "C" int bfsr_capture_gone(void* ticket)
{
    std::atomic<int>* gone = (std::atomic<int>*)ticket;
    if (!gone) return -1;
    if (!gone->load(std::memory_order_acquire)) return 0;
    delete gone;
    return 1;
}
