// The paged KV cache's operators for gfx950 (interface: kvcache.h).
//
//   append   rotary positions, new keys and values into the pages
//   attend   one new token over the cache, split over its length and joined;
//            each place's weight is added to the cache's mass
//   observe  the weight that a prompt's rows gave to the places
//   evict    which places stay once a sequence is too long, by mass
//
// Keys and values are 16-bit; queries are of the pool's type or float32 (over
// a bfloat16 pool). All scores, maxima, sums and masses are float32. Products
// run on v_mfma_f32_16x16x32: float32 operands go in as sums of 16-bit pieces
// (a float32 is three bfloat16 exactly), so nothing is lost to the matrix
// cores' types; the pieces cost matrix instructions only, and attention of
// one token has far more of those than it has bandwidth.
#include <algorithm>

#include "common.h"
#include "kvcache.h"

namespace cla {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f;

template <class To, class From>
__device__ __forceinline__ To bits(const From& x) {
    static_assert(sizeof(To) == sizeof(From), "same size");
    return __builtin_bit_cast(To, x);
}

// ------------------------------------------------------------- 16-bit types

struct Bf16 {
    // attention weights are taken relative to 2^-AHEAD of the largest
    static constexpr float AHEAD = 0.f;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            bits<bf16x8>(a), bits<bf16x8>(b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const bf16x2 v = {(__bf16)x, (__bf16)y};
        return bits<uint32_t>(v);
    }
    static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
        return f32x2{bits<float>(w << 16), bits<float>(w & 0xFFFF0000u)};
    }
    // The leading 8 bits of x and y as a packed pair; x and y become what is
    // left. Three calls take all 24 bits. What is left gets 2^-30 of x more: a
    // piece is then never 0, and of x's sign, so that it makes infinity of an
    // infinite operand as x does, and not NaN.
    static __device__ __forceinline__ uint32_t piece(float& x, float& y) {
        const uint32_t ux = bits<uint32_t>(x) & 0xFFFF0000u;
        const uint32_t uy = bits<uint32_t>(y) & 0xFFFF0000u;
        x = fmaf(x, 0x1p-30f, x - bits<float>(ux));
        y = fmaf(y, 0x1p-30f, y - bits<float>(uy));
        return (ux >> 16) | uy;
    }
};

struct F16 {
    // A weight of 1 would leave float16 only 24 bits of range below it: weights
    // go up to 2^14 (the type holds 2^16), so that 2^-39 of the largest counts.
    static constexpr float AHEAD = 14.f;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(
            bits<f16x8>(a), bits<f16x8>(b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const f16x2 v = {(_Float16)x, (_Float16)y};
        return bits<uint32_t>(v);
    }
    static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
        const f16x2 v = bits<f16x2>(w);
        return f32x2{(float)v.x, (float)v.y};
    }
    // As above, 11 bits a call, for attention weights: of [0, 2^14], in two
    // pieces. The second is at least 2^-24, the type's smallest (2^-38 of the
    // largest weight); weights below that are 0 or 2^-24 in all.
    static __device__ __forceinline__ uint32_t piece(float& x, float& y) {
        const auto v = __builtin_amdgcn_cvt_pkrtz(x, y);
        x = fmaxf(x - (float)v.x, fminf(x, 0x1p-24f));
        y = fmaxf(y - (float)v.y, fminf(y, 0x1p-24f));
        return bits<uint32_t>(v);
    }
};

struct Pages {
    uint16_t* pool;
    int64_t page_stride, table_stride;
    const int32_t* table;
    int32_t pages, max_pages, page;
    uint32_t per16, magic;   // page / 16, and ceil(2^32 / that)

    // Where 16 places from p on (p a multiple of 16) lie: the first one's
    // row; null where the table or the pool has no such page.
    __device__ __forceinline__ uint16_t* rows16(int b, int p, int head,
                                                int dim) const {
        const uint32_t p16 = (uint32_t)p >> 4;
        const uint32_t i = per16 == 1 ? p16 : __umulhi(p16, magic);
        const int32_t pg = kv_page_of(table + (int64_t)b * table_stride, i,
                                      max_pages, pages);
        if (pg < 0) return nullptr;
        return pool + (int64_t)pg * page_stride
               + (int64_t)head * 2 * page * dim
               + (int64_t)(p16 - i * per16) * 16 * dim;
    }
};

Pages pages_of(const KvPages& kv) {
    Pages p;
    p.pool = reinterpret_cast<uint16_t*>(kv.pool);
    p.page_stride = kv.page_stride;
    p.table_stride = kv.table_stride;
    p.table = kv.table;
    p.pages = kv.pages;
    p.max_pages = kv.max_pages;
    p.page = kv.page;
    p.per16 = (uint32_t)kv.page / 16;
    // exact for p16 * per16 < 2^32: pages have at most 1024 places and
    // sequences at most 2^30 (checked by check_pages)
    p.magic = p.per16 > 1 ? (uint32_t)((0xFFFFFFFFull + p.per16) / p.per16) : 0;
    return p;
}

void check_pages(const KvPages& kv, int q_heads, int reach) {
    if (kv.dim != 64 && kv.dim != 96 && kv.dim != 128)
        throw std::runtime_error("head_dim must be 64, 96 or 128");
    if (kv.page < 16 || kv.page > 1024 || kv.page % 16)
        throw std::runtime_error(
            "page size must be a multiple of 16, at most 1024");
    if (kv.type != KVT::BF16 && kv.type != KVT::F16)
        throw std::runtime_error("the pool must be bfloat16 or float16");
    if (kv.slots < 1 || kv.kv_heads < 1 || kv.pages < 1 || kv.max_pages < 1)
        throw std::runtime_error("empty pool or page table");
    if (reach < 0 || reach > (1 << 30) ||
        (int64_t)reach > (int64_t)kv.max_pages * kv.page)
        throw std::runtime_error("a sequence may have at most 2^30 places");
    if ((int64_t)kv.slots * kv.kv_heads * (reach / 128 + 1) >= (1ll << 31))
        throw std::runtime_error("too many places in all");
    if (q_heads && (q_heads % kv.kv_heads || q_heads / kv.kv_heads > 16))
        throw std::runtime_error(
            "query heads must be 1 to 16 times the kv heads");
}

void check_scale(float scale) {
    if (!(scale > 0.f && scale * LOG2E < INFINITY))
        throw std::runtime_error("scale must be positive and finite");
}

// a grid's threads must be fewer than 2^32
void check_grid(int64_t workgroups) {
    if (workgroups >= 1ll << 24)
        throw std::runtime_error("too many rows or sequences in one call");
}

void check_launch() {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        throw std::runtime_error(std::string("HIP error: ") +
                                 hipGetErrorString(e));
}

// Which sequence row t of packed rows belongs to: the last b whose
// starts[b] <= t. slots: behind the last sequence. All 64 lanes take part.
__device__ __forceinline__ int sequence_of(const int32_t* starts, int slots,
                                           int t) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base <= slots; base += 64) {
        const int i = base + lane;
        before += __popcll(__ballot(i <= slots && starts[i] <= t));
    }
    return before - 1;
}

__device__ __forceinline__ float wave_xor_max(float x, int mask) {
    return fmaxf(x, __shfl_xor(x, mask, 64));
}
__device__ __forceinline__ float wave_xor_sum(float x, int mask) {
    return x + __shfl_xor(x, mask, 64);
}

// x is there from here on: a loaded operand that a loop uses first is
// otherwise waited for in the loop, along with the loop's own loads that
// should still be on their way.
__device__ __forceinline__ void arrive(u32x4& x) {
    asm volatile("" : "+v"(x));
}

__device__ __forceinline__ float exp2_fast(float x) {
    return __builtin_amdgcn_exp2f(x);
}

// ------------------------------------------------------------------- append

struct AppendArgs {
    Pages kv;
    KvHeads k, v, q, q_out;
    KvRows mass, pos;
    const int32_t *starts, *lens, *next_pos;
    const float* inv_freq;
    int32_t q_heads, kv_heads, slots, reach;
};

template <KVT T>
__device__ __forceinline__ void load8(const void* p, int64_t at, float* x) {
    if constexpr (T == KVT::F32) {
        const f32x4* s = reinterpret_cast<const f32x4*>(
            reinterpret_cast<const float*>(p) + at);
        const f32x4 a = s[0], b = s[1];
        #pragma unroll
        for (int i = 0; i < 4; i++) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(
            reinterpret_cast<const uint16_t*>(p) + at);
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x2 f = T == KVT::BF16 ? Bf16::unpack(w[i])
                                           : F16::unpack(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

template <KVT T>
__device__ __forceinline__ void store8(void* p, int64_t at, const float* x) {
    if constexpr (T == KVT::F32) {
        f32x4* d = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + at);
        d[0] = f32x4{x[0], x[1], x[2], x[3]};
        d[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        u32x4 w;
        #pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = T == KVT::BF16 ? Bf16::pack(x[2 * i], x[2 * i + 1])
                                  : F16::pack(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p) + at) = w;
    }
}

// grid (rows, parts) x 256. A workgroup takes one row's heads (q, k, v side
// by side), 8 elements a thread and pass; the row's angles are shared by all
// heads through LDS. position * inv_freq is taken and reduced in 64 bits: in
// 32 it would be off by 2^-24 of the angle, 0.06 rad at position 10^6.
// Bound by memory: 7203 rows of 32 + 16 heads of 128 (177 MB) take 37.6 us, 4.7
// TB/s, nearly a large copy's rate; few rows by latency (3.4 us).
template <KVT T, KVT C, int D>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
    __shared__ float cs[D / 2], sn[D / 2];
    const int t = blockIdx.x, tid = threadIdx.x;
    int b = t, i = 0;
    if (a.starts) {
        b = sequence_of(a.starts, a.slots, t);
        if (b >= 0 && b < a.slots) i = t - a.starts[b];
    }
    const bool mine = b >= 0 && b < a.slots;
    const int64_t place = mine ? (int64_t)a.lens[b] + i : -1;
    const int position = mine ? a.next_pos[b] + i : 0;
    // rows behind the last sequence keep their queries as they are
    const bool turned = a.inv_freq && mine;
    if (turned && tid < D / 2) {
        const double turn = (double)position * (double)a.inv_freq[tid];
        const double whole = rint(turn * 0.15915494309189535);
        const float rest = (float)fma(whole, -6.283185307179586, turn);
        sincosf(rest, &sn[tid], &cs[tid]);
    }
    __syncthreads();

    const bool stored = place >= 0 && place < a.reach;
    int32_t page = -1;
    int row = 0;
    if (stored) {
        page = kv_page_of(a.kv.table + (int64_t)b * a.kv.table_stride,
                          place / a.kv.page, a.kv.max_pages, a.kv.pages);
        row = (int)(place % a.kv.page);
    }
    constexpr int PER = D / 8;
    const int heads = a.q_heads + 2 * a.kv_heads;
    for (int it = blockIdx.y * 256 + tid; it < heads * PER;
         it += gridDim.y * 256) {
        const int head = it / PER, d = it % PER * 8;
        const int kvh = head - a.q_heads;
        if (kvh >= 0 && page < 0) continue;
        const bool is_v = kvh >= a.kv_heads;
        const KvHeads& src = kvh < 0 ? a.q : is_v ? a.v : a.k;
        const int h = kvh < 0 ? head : is_v ? kvh - a.kv_heads : kvh;
        float x[8];
        load8<T>(src.data, t * src.row_stride + h * src.head_stride + d, x);
        if (turned && !is_v) {
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const float c = cs[d / 2 + j], s = sn[d / 2 + j];
                const float x0 = x[2 * j], x1 = x[2 * j + 1];
                x[2 * j] = x0 * c - x1 * s;
                x[2 * j + 1] = x0 * s + x1 * c;
            }
        }
        if (kvh < 0)
            store8<T>(a.q_out.data,
                      t * a.q_out.row_stride + h * a.q_out.head_stride + d, x);
        else
            store8<C>(a.kv.pool,
                      (int64_t)page * a.kv.page_stride
                          + ((int64_t)h * 2 + is_v) * a.kv.page * D
                          + (int64_t)row * D + d, x);
    }
    if (blockIdx.y == 0 && stored) {
        for (int h = tid; h < a.kv_heads; h += 256) {
            if (a.mass.data)
                reinterpret_cast<float*>(a.mass.data)[
                    b * a.mass.slot_stride + h * a.mass.head_stride + place] =
                    0.f;
            if (a.pos.data)
                reinterpret_cast<int32_t*>(a.pos.data)[
                    b * a.pos.slot_stride + h * a.pos.head_stride + place] =
                    position;
        }
    }
}

__global__ __launch_bounds__(64) void k_kv_step(
    int32_t* len, int32_t* step, const uint8_t* active, int slots) {
    for (int b = threadIdx.x; b < slots; b += 64) {
        step[b] = active[b] ? len[b] : -1;
        if (active[b]) len[b]++;
    }
}

// ------------------------------------------------------------------- attend

constexpr int TILE = 32;          // places a wave takes at a time
constexpr int WAVES = 4;
constexpr int UNIT = TILE * WAVES;

// How many workgroups the whole of the batch's places are split into, about:
// two a CU, which stream as fast as more and leave less to join (one sequence
// of 131071 places: 125 us, 133 with 2048; 16 x 8 rows of up to 4096: 33 us, 35
// with 2048). With as many rows (sequences x kv heads) as CUs most rows would
// stay whole, and the CUs that get long ones finish late: finer parts even that
// out (16 x 32 rows of up to 8191 places: 172 us, 208 with 512; 64 x 4 of up to
// 4096: 50 us, 55 with 512).
inline int attend_target(const KvPages& kv) {
    return (int64_t)kv.slots * kv.kv_heads >= 256 ? 2048 : 512;
}

// The lengths on the device decide how the work is split: every kv head's
// places are cut into equally many units of 128 for each workgroup, as many
// as make about `target` workgroups of all of them. A ragged batch's long
// sequences get more workgroups than its short ones, and the host needs no
// length. Workgroup `id` takes part j of n of (b, head).
struct Part {
    int b, head, j, n, first, lo, hi, there;
};

struct AttendArgs {
    Pages kv;
    KvHeads q, out;
    KvRows mass;
    const int32_t* lens;
    int32_t add, q_heads, kv_heads, slots, reach, target;
    float scale2;             // scale * log2(e)
    float* scores;            // [slots][kv heads][ld / 32][G][32], of log2
    int64_t ld;
    float* part_o;            // [workgroup][G][D], relative to part_m
    float* part_ml;           // [workgroup][G][2]
    Part* parts;              // [workgroup], for the second kernel
};

__device__ __forceinline__ bool find_part(const AttendArgs& a, int id,
                                          Part& p) {
    const int lane = threadIdx.x & 63;
    auto len_of = [&](int b) {
        return b < a.slots ? kv_clamp_len(a.lens[b] + a.add, a.reach) : 0;
    };
    const int len0 = len_of(lane);
    int all = (len0 + UNIT - 1) / UNIT;
    for (int b = 64 + lane; b - lane < a.slots; b += 64)
        all += (len_of(b) + UNIT - 1) / UNIT;
    #pragma unroll
    for (int m = 32; m; m >>= 1) all += __shfl_xor(all, m, 64);
    all = __builtin_amdgcn_readfirstlane(all);
    const int per = max(1u, ((uint32_t)all * a.kv_heads + a.target - 1)
                                / (uint32_t)a.target);
    int before = 0;
    for (int base = 0; base < a.slots; base += 64) {
        const int b = base + lane;
        const int len = base ? len_of(b) : len0;
        const int units = (len + UNIT - 1) / UNIT;
        const int n = max(1u, (uint32_t)(units + per - 1) / (uint32_t)per);
        int upto = b < a.slots ? n * a.kv_heads : 0;
        #pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int x = __shfl_up(upto, m, 64);
            if (lane >= m) upto += x;
        }
        const uint64_t over = __ballot(before + upto > id);
        if (over) {
            // scalars, as all that follows from them
            const int at = __builtin_ctzll(over);
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
            const int len_b = of(len);
            p.b = base + at;
            p.n = of(n);
            const int rest = id - before - (of(upto) - p.n * a.kv_heads);
            p.head = rest / p.n;
            p.j = rest - p.head * p.n;
            p.first = id - p.j;
            // n = ceil(units / per) parts of ceil(units / n): none is empty
            const int each = ((len_b + UNIT - 1) / UNIT + p.n - 1) / p.n
                * UNIT;
            p.lo = p.j * each;
            p.hi = min(p.lo + each, len_b);
            p.there = 1;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// The queries of one kv head as the B operand of 16x16x32 products, in NQ
// pieces: column n is query head n (zero past the last), k runs over d.
template <class C, int NQ, int D>
__device__ __forceinline__ void load_q(const void* q, int64_t at, bool there,
                                       int g, u32x4 (*f)[D / 32]) {
    #pragma unroll
    for (int kk = 0; kk < D / 32; kk++) {
        const int64_t d = at + kk * 32 + g * 8;
        if constexpr (NQ == 1) {
            f[0][kk] = there ? *reinterpret_cast<const u32x4*>(
                reinterpret_cast<const uint16_t*>(q) + d) : u32x4{0, 0, 0, 0};
        } else {
            float x[8];
            if (there) {
                load8<KVT::F32>(q, d, x);
            } else {
                #pragma unroll
                for (int i = 0; i < 8; i++) x[i] = 0.f;
            }
            #pragma unroll
            for (int s = 0; s < NQ; s++)
                #pragma unroll
                for (int i = 0; i < 4; i++)
                    f[s][kk][i] = C::piece(x[2 * i], x[2 * i + 1]);
        }
    }
}

// One wave's 32 places: keys as the A operand (two products of 16 places),
// values as a lane's 8 places of EL elements.
template <int D>
struct Tile {
    static constexpr int EL = D / 16;
    u32x4 k[2][D / 32];
    uint32_t v[8][EL / 2];
};

template <int D>
__device__ __forceinline__ void load_tile(const uint16_t* r0,
                                          const uint16_t* r1, int64_t to_v,
                                          int n, int g, Tile<D>& t) {
    constexpr int EL = D / 16;
    #pragma unroll
    for (int u = 0; u < 2; u++) {
        const uint16_t* r = u ? r1 : r0;
        const uint16_t* kp = r + n * D + g * 8;
        #pragma unroll
        for (int kk = 0; kk < D / 32; kk++)
            t.k[u][kk] = *reinterpret_cast<const u32x4*>(kp + kk * 32);
        const uint16_t* vp = r + to_v + g * 4 * D + n * EL;
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t* d = t.v[u * 4 + j];
            if constexpr (EL == 8) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(vp + j * D);
                d[0] = w.x; d[1] = w.y; d[2] = w.z; d[3] = w.w;
            } else if constexpr (EL == 6) {
                // 12 bytes at a multiple of 4
                const uint32_t* s =
                    reinterpret_cast<const uint32_t*>(vp + j * D);
                d[0] = s[0]; d[1] = s[1]; d[2] = s[2];
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2*>(vp + j * D);
                d[0] = w.x; d[1] = w.y;
            }
        }
    }
}

// What a lane has of its query head: the reference m of its weights 2^(score -
// m), which is AHEAD below the maximum of the wave's places; the sum of its own
// places' weights; and its outputs.
template <int D>
struct Softmax {
    float m = -INFINITY, l = 0.f;
    f32x4 o[D / 16];
    __device__ Softmax() {
        #pragma unroll
        for (int e = 0; e < D / 16; e++) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
};

// 32 places from p0 on: S = K Q^T and O^T = V^T P^T, so that in both results a
// lane's column is its query head: maximum, sum and rescaling stay in the
// lane. S's rows (places) then are just the k index of the second product,
// and V needs no transposition through LDS: a lane holds 8 places x EL
// elements, and product e takes element e of each (MFMA row r is d = r*EL+e).
// t0, t1: whether the first and the second 16 have a page. Scores go to
// put(place, 4 of them).
template <class C, int NQ, int NP, int D, class Put>
__device__ __forceinline__ void use_tile(Tile<D>& t, bool t0, bool t1, int p0,
                                         int hi, float scale2, int g,
                                         const u32x4 (*q)[D / 32],
                                         Softmax<D>& x, Put put) {
    constexpr int EL = D / 16;
    float &m = x.m, &l = x.l;
    f32x4* o = x.o;
    const bool whole = t0 && t1 && p0 + TILE <= hi;
    float s[8];
    #pragma unroll
    for (int u = 0; u < 2; u++) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int y = NQ - 1; y >= 0; y--)
            #pragma unroll
            for (int kk = 0; kk < D / 32; kk++)
                acc = C::mfma(t.k[u][kk], q[y][kk], acc);
        #pragma unroll
        for (int i = 0; i < 4; i++) s[u * 4 + i] = acc[i] * scale2;
    }
    if (!whole) {
        #pragma unroll
        for (int j = 0; j < 8; j++) {
            const int u = j >> 2;
            const bool seen = (u ? t1 : t0) &&
                p0 + u * 16 + g * 4 + (j & 3) < hi;
            if (!seen) {
                s[j] = -INFINITY;
                // what lies there may be anything: 0 * inf is NaN
                #pragma unroll
                for (int e = 0; e < EL / 2; e++) t.v[j][e] = 0;
            }
        }
    }
    #pragma unroll
    for (int u = 0; u < 2; u++)
        put(u * 16 + g * 4, f32x4{s[u * 4], s[u * 4 + 1], s[u * 4 + 2],
                                  s[u * 4 + 3]});
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                      fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    top = wave_xor_max(wave_xor_max(top, 16), 32) - C::AHEAD;
    if (__any(top > m)) {
        const float now = fmaxf(m, top);
        const float f = exp2_fast(m - now);   // 0 from -inf
        m = now;
        if (now > -INFINITY) {
            l *= f;
            #pragma unroll
            for (int e = 0; e < EL; e++) o[e] *= f;
        }
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float w[8];
    #pragma unroll
    for (int j = 0; j < 8; j++) {
        w[j] = exp2_fast(s[j] - ref);
        l += w[j];
    }
    u32x4 pf[NP];
    #pragma unroll
    for (int y = 0; y < NP; y++)
        #pragma unroll
        for (int i = 0; i < 4; i++)
            pf[y][i] = y + 1 < NP ? C::piece(w[2 * i], w[2 * i + 1])
                                  : C::pack(w[2 * i], w[2 * i + 1]);
    #pragma unroll
    for (int e = 0; e < EL; e++) {
        u32x4 vf;
        #pragma unroll
        for (int i = 0; i < 4; i++)
            vf[i] = __builtin_amdgcn_perm(
                t.v[2 * i + 1][e >> 1], t.v[2 * i][e >> 1],
                (e & 1) ? 0x07060302u : 0x05040100u);
        #pragma unroll
        for (int y = NP - 1; y >= 0; y--) o[e] = C::mfma(vf, pf[y], o[e]);
    }
}

template <class C, bool F32>
__device__ __forceinline__ void put_out(const AttendArgs& a, int b, int head,
                                        int d, float y) {
    const int64_t at = b * a.out.row_stride
        + (int64_t)head * a.out.head_stride + d;
    if constexpr (F32)
        reinterpret_cast<float*>(a.out.data)[at] = y;
    else
        reinterpret_cast<uint16_t*>(a.out.data)[at] =
            (uint16_t)C::pack(y, 0.f);
}

// A workgroup's waves join: s_m, s_l, s_o take what its lanes have, a lane's
// l being of its own places only.
template <int D>
__device__ __forceinline__ void give(const Softmax<D>& x, int n, int g,
                                     float* s_m, float* s_l, float (*s_o)[D]) {
    const float l = wave_xor_sum(wave_xor_sum(x.l, 16), 32);
    if (g == 0) { s_m[n] = x.m; s_l[n] = l; }
    #pragma unroll
    for (int e = 0; e < D / 16; e++)
        #pragma unroll
        for (int i = 0; i < 4; i++)
            s_o[n][(g * 4 + i) * (D / 16) + e] = x.o[e][i];
}

// One workgroup takes one part of one kv head's places, its four waves 32 at
// a time in turn.
//
// Bound by the reads of K and V: one sequence of 131071 places of 8 kv heads of
// 128 (537 MB) takes 102 us without a mass, with its join, 5.3 TB/s; a stream
// that is only read reaches 5.5. Its scores go out as they are where a mass is
// wanted, since the weights are known only once all parts are; those 17 MB, out
// and back, cost another 23 us. The products take a third of that (three
// pieces), so loading a tile ahead gains nothing (119 us for 112).
template <class C, int NQ, int NP, int D, bool MASS>
__global__ __launch_bounds__(256) void k_kv_attend(AttendArgs a) {
    __shared__ float s_m[WAVES][16], s_l[WAVES][16];
    __shared__ float s_o[WAVES][16][D];
    Part p;
    const bool there = find_part(a, blockIdx.x, p);
    if (threadIdx.x == 0) {
        if (there) a.parts[blockIdx.x] = p;
        else a.parts[blockIdx.x].there = 0;
    }
    if (!there) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int G = a.q_heads / a.kv_heads;
    const int head = p.head * G + n;

    u32x4 q[NQ][D / 32];
    load_q<C, NQ, D>(a.q.data,
                     p.b * a.q.row_stride + head * a.q.head_stride, n < G, g,
                     q);
    Softmax<D> sm;
    float* scores = MASS && n < G
        ? a.scores + ((int64_t)p.b * a.kv_heads + p.head) * G * a.ld + n * 32
        : nullptr;
    const int64_t to_v = (int64_t)a.kv.page * D;

    for (int p0 = p.lo + wave * TILE; p0 < p.hi; p0 += UNIT) {
        const uint16_t* r0 = a.kv.rows16(p.b, p0, p.head, D);
        const uint16_t* r1 = p0 + 16 < p.hi
            ? a.kv.rows16(p.b, p0 + 16, p.head, D) : nullptr;
        // places that are not there are read from the pool's first page,
        // and count for nothing
        Tile<D> t;
        load_tile<D>(r0 ? r0 : a.kv.pool, r1 ? r1 : a.kv.pool, to_v, n, g, t);
        use_tile<C, NQ, NP, D>(
            t, r0, r1, p0, p.hi, a.scale2, g, q, sm, [&](int x, f32x4 s) {
                // a tile's scores lie together
                if (MASS && scores)
                    *reinterpret_cast<f32x4*>(scores + (int64_t)p0 * G + x) = s;
            });
    }

    give<D>(sm, n, g, s_m[wave], s_l[wave], s_o[wave]);
    __syncthreads();
    for (int x = tid; x < G * D; x += 256) {
        const int h = x / D, d = x % D;
        float top = s_m[0][h];
        #pragma unroll
        for (int w = 1; w < WAVES; w++) top = fmaxf(top, s_m[w][h]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f, acc = 0.f;
        #pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = exp2_fast(s_m[w][h] - ref);
            sum += f * s_l[w][h];
            acc += f * s_o[w][h][d];
        }
        if (p.n == 1) {
            put_out<C, (NQ > 1)>(a, p.b, p.head * G + h, d,
                                 sum == 0.f ? 0.f : acc / sum);
        } else {
            a.part_o[((int64_t)blockIdx.x * G + h) * D + d] = acc;
        }
        if (d == 0) {
            a.part_ml[((int64_t)blockIdx.x * G + h) * 2] = top;
            a.part_ml[((int64_t)blockIdx.x * G + h) * 2 + 1] = sum;
        }
    }
}

// Short rows, grid (kv heads, slots): eight waves take all of a row's places,
// and its mass in the same launch, from scores in LDS. Bound by what one CU can
// have under way (601 places of heads of 128: 11.7 us); the next tile's loads
// ahead of a tile's products gain nothing.
constexpr int ROW_WAVES = 8, ROW_PLACES = 1024;

template <class C, int NQ, int NP, int D, bool MASS>
__global__ __launch_bounds__(64 * ROW_WAVES) void k_kv_attend_row(
    AttendArgs a) {
    __shared__ float s_m[ROW_WAVES][16], s_l[ROW_WAVES][16];
    __shared__ float s_ref[16], s_r[16];
    __shared__ float s_o[ROW_WAVES][16][D];
    __shared__ __align__(16) float s_s[MASS ? ROW_PLACES * 16 : 4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4, b = blockIdx.y;
    const int G = a.q_heads / a.kv_heads, first = blockIdx.x * G;
    const int len = kv_clamp_len(a.lens[b] + a.add, a.reach);
    u32x4 q[NQ][D / 32];
    load_q<C, NQ, D>(a.q.data, b * a.q.row_stride
                         + (int64_t)(first + n) * a.q.head_stride, n < G, g, q);
    const int64_t to_v = (int64_t)a.kv.page * D;
    Softmax<D> sm;
    for (int p0 = wave * TILE; p0 < len; p0 += TILE * ROW_WAVES) {
        const uint16_t* r0 = a.kv.rows16(b, p0, blockIdx.x, D);
        const uint16_t* r1 = p0 + 16 < len
            ? a.kv.rows16(b, p0 + 16, blockIdx.x, D) : nullptr;
        Tile<D> t;
        load_tile<D>(r0 ? r0 : a.kv.pool, r1 ? r1 : a.kv.pool, to_v, n, g, t);
        use_tile<C, NQ, NP, D>(
            t, r0, r1, p0, len, a.scale2, g, q, sm, [&](int x, f32x4 s) {
                if (MASS && n < G)
                    *reinterpret_cast<f32x4*>(s_s + p0 * G + n * 32 + x) = s;
            });
    }
    give<D>(sm, n, g, s_m[wave], s_l[wave], s_o[wave]);
    __syncthreads();
    for (int x = tid; x < G * D; x += 64 * ROW_WAVES) {
        const int h = x / D, d = x % D;
        float top = s_m[0][h];
        #pragma unroll
        for (int w = 1; w < ROW_WAVES; w++) top = fmaxf(top, s_m[w][h]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f, acc = 0.f;
        #pragma unroll
        for (int w = 0; w < ROW_WAVES; w++) {
            const float f = exp2_fast(s_m[w][h] - ref);
            sum += f * s_l[w][h];
            acc += f * s_o[w][h][d];
        }
        const float r = sum == 0.f ? 0.f : 1.f / sum;
        if (d == 0) { s_ref[h] = ref; s_r[h] = r; }
        put_out<C, (NQ > 1)>(a, b, first + h, d,
                             sum == 0.f ? 0.f : acc / sum);
    }
    if constexpr (MASS) {
        __syncthreads();
        float* mass = reinterpret_cast<float*>(a.mass.data)
            + b * a.mass.slot_stride + blockIdx.x * a.mass.head_stride;
        for (int x = tid; x < len; x += 64 * ROW_WAVES) {
            const float* sc = s_s + (x & ~31) * G + (x & 31);
            float w = 0.f;
            for (int h = 0; h < G; h++)
                w += exp2_fast(sc[h * 32] - s_ref[h]) * s_r[h];
            mass[x] += w;
        }
    }
}

// Join the parts: the same workgroups once more. Each makes its share of the
// head's outputs (the parts' sums, in their order) and, from the scores, the
// weights of its own places. Latency and the scores' 17 MB: 10.7 us for the
// sequence above.
template <class C, bool F32OUT, int D, bool MASS>
__global__ __launch_bounds__(256) void k_kv_join(AttendArgs a) {
    __shared__ float s_m[16], s_r[16];
    __shared__ float s_acc[256];
    const Part p = a.parts[blockIdx.x];
    if (!p.there || (!MASS && p.n == 1)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int G = a.q_heads / a.kv_heads;
    const float* ml = a.part_ml + (int64_t)p.first * G * 2;
    for (int h = wave; h < G; h += WAVES) {
        float m = -INFINITY, l = 0.f;
        for (int j = lane; j < p.n; j += 64) {
            const float mj = ml[((int64_t)j * G + h) * 2];
            const float lj = ml[((int64_t)j * G + h) * 2 + 1];
            const float now = fmaxf(m, mj);
            const float ref = now == -INFINITY ? 0.f : now;
            l = l * exp2_fast(m - ref) + lj * exp2_fast(mj - ref);
            m = now;
        }
        float top = m;
        #pragma unroll
        for (int x = 32; x; x >>= 1) top = wave_xor_max(top, x);
        const float ref = top == -INFINITY ? 0.f : top;
        l *= exp2_fast(m - ref);
        #pragma unroll
        for (int x = 32; x; x >>= 1) l = wave_xor_sum(l, x);
        if (lane == 0) { s_m[h] = ref; s_r[h] = l == 0.f ? 0.f : 1.f / l; }
    }
    __syncthreads();
    if constexpr (MASS) {
        // 4 places a thread, 4 heads' scores at a time
        float* mass = reinterpret_cast<float*>(a.mass.data)
            + p.b * a.mass.slot_stride + p.head * a.mass.head_stride;
        const float* sc = a.scores
            + ((int64_t)p.b * a.kv_heads + p.head) * G * a.ld;
        for (int x = p.lo + tid * 4; x < p.hi; x += 1024) {
            const float* at = sc + (int64_t)(x & ~31) * G + (x & 31);
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
            for (int h = 0; h < G; h += 4) {
                f32x4 s[4];
                #pragma unroll
                for (int i = 0; i < 4; i++)
                    s[i] = *reinterpret_cast<const f32x4*>(
                        at + min(h + i, G - 1) * 32);
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int hi = min(h + i, G - 1);
                    const float m = s_m[hi], r = s_r[hi];
                    #pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float w = exp2_fast(s[i][e] - m) * r;
                        sum[e] += h + i < G ? w : 0.f;
                    }
                }
            }
            #pragma unroll
            for (int e = 0; e < 4; e++)
                if (x + e < p.hi) mass[x + e] += sum[e];
        }
    }
    if (p.n > 1) {
        // `each` of the head's G * D outputs; width (a power of two) of them
        // at a time, the parts dealt to 256 / width threads of each
        const int each = (G * D + p.n - 1) / p.n;
        const int lo = p.j * each, hi = min(lo + each, G * D);
        int width = 8;
        while (width < each && width < 256) width <<= 1;
        const int y = tid / width, deal = 256 / width;
        const float* po = a.part_o + (int64_t)p.first * G * D;
        for (int x0 = lo; x0 < hi; x0 += width) {
            const int x = x0 + (tid & (width - 1)), h = x / D;
            float acc = 0.f;
            if (x < hi) {
                const float ref = s_m[h];
                #pragma unroll 4
                for (int j = y; j < p.n; j += deal)
                    acc += po[(int64_t)j * G * D + x]
                        * exp2_fast(ml[((int64_t)j * G + h) * 2] - ref);
            }
            __syncthreads();
            s_acc[tid] = acc;
            __syncthreads();
            if (tid < width && x < hi) {
                for (int i = 1; i < deal; i++) acc += s_acc[i * width + tid];
                put_out<C, F32OUT>(a, p.b, p.head * G + h, x % D,
                                   acc * s_r[h]);
            }
        }
    }
}

// ------------------------------------------------------------------ observe

// x / d for x * d < 2^32
struct Div {
    uint32_t d, magic;
    __device__ __forceinline__ int of(int x) const {
        return d == 1 ? x : (int)__umulhi((uint32_t)x, magic);
    }
};

Div div_by(int d) {
    return {(uint32_t)d,
            d > 1 ? (uint32_t)((0xFFFFFFFFull + (uint32_t)d) / d) : 0u};
}

// Groups of 16 places that a wave of the second pass holds, where there is
// work for many. Three leave room for a third wave a SIMD with heads of 128 and
// one piece (8192 rows of 32 heads, both passes: 633 us, 653 with four); more
// pieces have more to do for each row that is read (3 x 500 rows over 16000
// places: 466 us, 482 with three).
constexpr int obs_groups(bool one_piece, int dim) {
    return one_piece && dim == 128 ? 3 : 4;
}

struct ObserveArgs {
    Pages kv;
    KvHeads q;
    KvRows mass;
    const int32_t *starts, *lens;
    int32_t q_heads, kv_heads, slots, rows, reach;
    float scale2;
    Div group;
    // first pass: places in parts of `part`, of which there are `parts`
    int32_t part, parts;
    // second pass: a sequence's rows in chunks of `chunk`, at most `chunks` in
    // the batch, and places in blocks of `block`
    int32_t chunk, chunks, block;
    float* sums;       // [parts][kv heads][rows][G][2]: maximum, sum
    float* norm;       // [kv heads][rows][G][2]: what a row's weights are of
    float* partial;    // [chunks][kv heads][ld]
    int64_t ld;
};

// A sequence's rows as the kernels see them: r = i * G + h, query head h of
// row i, so that one pass over the keys serves the kv head's queries.
struct Seq {
    int b, t0, m, len;   // its first packed row, its rows, its places
    int before;          // places before its first row's own, negative if that
                         // has none; row i sees the first before + i + 1, of len
};

__device__ __forceinline__ Seq sequence_at(const ObserveArgs& a, int b) {
    Seq s;
    s.b = b;
    s.t0 = max(0, min(a.starts[b], a.rows));
    s.m = max(0, min(a.starts[b + 1], a.rows) - s.t0);
    // a length past the last place is that of a longer sequence, whose later
    // tokens were not stored: its rows' places are counted from there (as far
    // as it matters: where each row sees all places)
    const int len = max(a.lens[b], 0);
    s.len = min(len, a.reach);
    s.before = min(len, a.reach + s.m) - s.m;
    return s;
}

// How many places row i of the sequence sees.
__device__ __forceinline__ int sees(const Seq& s, int i) {
    return min(s.before + i + 1, s.len);
}

// Rows are staged in LDS with 16 bytes more than they have: an odd number of
// 16-byte units, so that 16 lanes that read one unit each of 16 rows meet in
// no bank.
template <int D> constexpr int LDS_ROW = D + 8;

struct True { constexpr operator bool() const { return true; } };
struct False { constexpr operator bool() const { return false; } };

template <int D>
__device__ __forceinline__ u32x4 lds_unit(const uint16_t* rows, int r,
                                          int unit) {
    return *reinterpret_cast<const u32x4*>(rows + r * LDS_ROW<D> + unit * 8);
}

// A row whose weights 2^(s - m) sum to l: each is 2^(s - x) * y of it, x a whole
// number, so that the exponent is as exact as s is near to it. (One number,
// m + log2(l), would be rounded to 2^-20 for a sum of thousands, and so would
// all of a row's weights, the same way.) A row that sees nothing gives nothing:
// x is infinite.
__device__ __forceinline__ f32x2 row_norm(float m, float l) {
    if (l == 0.f) return f32x2{INFINITY, 0.f};
    const float x = rintf(m + __log2f(l));
    return f32x2{x, exp2_fast(x - m) / l};
}

// The x-th block of `rows` rows, counted over the batch: which sequence's it
// is, which of its blocks, and of how many. -1: there is no such.
struct RowBlock {
    int id, all;
};

__device__ __forceinline__ RowBlock row_block(const ObserveArgs& a, int rows,
                                              int at_x, Seq& s) {
    if (a.slots == 1) {
        s = sequence_at(a, 0);
        const int all = (s.m * (int)a.group.d + rows - 1) / rows;
        return {at_x < all ? at_x : -1, all};
    }
    const int lane = threadIdx.x & 63;
    for (int base = 0, before = 0; base < a.slots; base += 64) {
        const int b = min(base + lane, a.slots - 1);
        const Seq own = sequence_at(a, b);
        const int all = base + lane < a.slots
            ? (own.m * (int)a.group.d + rows - 1) / rows : 0;
        int upto = all;
        #pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int x = __shfl_up(upto, m, 64);
            if (lane >= m) upto += x;
        }
        const uint64_t over = __ballot(before + upto > at_x);
        if (over) {
            // scalars, as all that follows from them
            const int at = __builtin_ctzll(over);
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
            s = {base + at, of(own.t0), of(own.m), of(own.len),
                 of(own.before)};
            return {at_x - before - of(upto) + of(all), of(all)};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return {-1, 0};
}

// The first pass's: a sequence's last rows, which see the most, go first.
template <int ROWS>
__device__ __forceinline__ int late_block(const ObserveArgs& a, Seq& s) {
    const RowBlock x = row_block(a, ROWS, blockIdx.x, s);
    return x.id < 0 ? -1 : x.all - 1 - x.id;
}

// A row's sum over a part of the places, to where it belongs.
__device__ __forceinline__ void store_sum(const ObserveArgs& a, const Seq& s,
                                          int head, int r, float top,
                                          float sum) {
    const int64_t at = ((int64_t)head * a.rows + s.t0) * a.group.d + r;
    if (a.parts == 1) {
        *reinterpret_cast<f32x2*>(a.norm + at * 2) = row_norm(top, sum);
    } else {
        float* d = a.sums + ((int64_t)blockIdx.z * a.q_heads * a.rows + at) * 2;
        // a part without a weight must not set the others' reference
        d[0] = sum == 0.f ? -INFINITY : top;
        d[1] = sum;
    }
}

// Pass 1, grid (row blocks, kv heads, parts): 16 * RW rows a wave, whose
// queries stay in registers, over the part's places, which the workgroup
// stages 64 at a time. Each lane keeps a sum (and a maximum, where it needs
// one) of its own for each of its columns; they meet at the end.
//
// A score costs a multiplication, an exponential and an addition: 16 + 32 + 16
// cycles of the SIMD for 4 x 64 of them, beside 64 of matrix products, which
// run at the same time in part. 312 us for 8192 rows of 32 heads (275 GFLOP).
//
// One piece leaves room for three waves a SIMD; with three pieces they would
// spill (both passes for 3 x 500 rows over 16000 places: 466 us with two waves,
// 502 with three).
template <class C, int NQ, int D, int RW>
__global__ __launch_bounds__(256, NQ > 1 ? 2 : 3) void k_kv_observe_sums(
    ObserveArgs a) {
    constexpr int ROWS = 16 * RW * WAVES, KT = 64, PER = 16 * D / 8 / 64;
    __shared__ __align__(16) uint16_t s_k[2][KT * LDS_ROW<D>];
    __shared__ int s_there[2][4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4, head = blockIdx.y;
    const int G = a.group.d;
    Seq s{};
    const int id = late_block<ROWS>(a, s);
    if (id < 0) return;
    const int R = s.m * G;
    const int r0 = id * ROWS + wave * 16 * RW;
    // places that the workgroup's last row, and the wave's first, see
    const int most = sees(s, a.group.of(min(id * ROWS + ROWS, R) - 1));
    const int least = sees(s, a.group.of(r0));
    const int begin = blockIdx.z * a.part, end = min(begin + a.part, most);

    u32x4 q[RW][NQ][D / 32];
    float m[RW], l[RW];
    int seen[RW];          // places that the lane's column sees
    #pragma unroll
    for (int w = 0; w < RW; w++) {
        const int r = r0 + w * 16 + n, i = a.group.of(r), h = r - i * G;
        const bool there = r < R;
        load_q<C, NQ, D>(a.q.data, (int64_t)(s.t0 + i) * a.q.row_stride
                             + (int64_t)(head * G + h) * a.q.head_stride,
                         there, g, q[w]);
        seen[w] = there ? sees(s, i) : 0;
    }
    #pragma unroll
    for (int w = 0; w < RW; w++)
        #pragma unroll
        for (int x = 0; x < NQ; x++)
            #pragma unroll
            for (int kk = 0; kk < D / 32; kk++) arrive(q[w][x][kk]);

    u32x4 next[PER];
    bool next_there;
    auto fetch = [&](int p0) {
        const int p = p0 + wave * 16;
        const uint16_t* rows = p < end ? a.kv.rows16(s.b, p, head, D)
                                       : nullptr;
        next_there = rows != nullptr;
        if (!rows) rows = a.kv.pool;
        #pragma unroll
        for (int x = 0; x < PER; x++)
            next[x] = reinterpret_cast<const u32x4*>(rows)[x * 64 + lane];
    };
    auto stage = [&](int buf) {
        #pragma unroll
        for (int x = 0; x < PER; x++) {
            const int u = x * 64 + lane;
            *reinterpret_cast<u32x4*>(
                &s_k[buf][(wave * 16 + u / (D / 8)) * LDS_ROW<D>
                          + u % (D / 8) * 8]) = next[x];
        }
        if (lane == 0) s_there[buf][wave] = next_there;
    };
    // 32 places (the tile's half `half`) against the wave's rows. CUT: some
    // row does not see them all, or (t0, t1) 16 of them have no page. MAX:
    // relative to a running maximum, else to 0.
    auto half_tile = [&](int buf, int half, int pu, bool t0, bool t1,
                         auto CUT, auto MAX) {
        u32x4 k[2][D / 32];
        #pragma unroll
        for (int u = 0; u < 2; u++)
            #pragma unroll
            for (int kk = 0; kk < D / 32; kk++)
                k[u][kk] = lds_unit<D>(s_k[buf], half * 32 + u * 16 + n,
                                       kk * 4 + g);
        #pragma unroll
        for (int w = 0; w < RW; w++) {
            f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            #pragma unroll
            for (int x = NQ - 1; x >= 0; x--)
                #pragma unroll
                for (int kk = 0; kk < D / 32; kk++)
                    #pragma unroll
                    for (int u = 0; u < 2; u++)
                        acc[u] = C::mfma(k[u][kk], q[w][x][kk], acc[u]);
            float e[8];
            #pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = acc[j >> 2][j & 3] * a.scale2;
                if (CUT && (!(j < 4 ? t0 : t1) ||
                            pu + (j >> 2) * 16 + g * 4 + (j & 3) >= seen[w]))
                    e[j] = -INFINITY;
            }
            if (MAX) {
                float top = m[w];
                #pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, e[j]);
                const float ref = top == -INFINITY ? 0.f : top;
                l[w] *= exp2_fast(m[w] - ref);
                m[w] = top;
                #pragma unroll
                for (int j = 0; j < 8; j++) e[j] -= ref;
            }
            #pragma unroll
            for (int j = 0; j < 8; j++) e[j] = exp2_fast(e[j]);
            l[w] += ((e[0] + e[1]) + (e[2] + e[3]))
                + ((e[4] + e[5]) + (e[6] + e[7]));
        }
    };
    auto pass = [&](auto MAX_) {
        constexpr bool MAX = MAX_;
        #pragma unroll
        for (int w = 0; w < RW; w++) {
            m[w] = MAX ? -INFINITY : 0.f;
            l[w] = 0.f;
        }
        if (begin < end) {
            fetch(begin);
            stage(0);
        }
        __syncthreads();
        int buf = 0;
        for (int p0 = begin; p0 < end; p0 += KT, buf ^= 1) {
            const bool more = p0 + KT < end;
            if (more) fetch(p0 + KT);
            #pragma unroll
            for (int half = 0; half < 2; half++) {
                const int pu = p0 + half * 32;
                if constexpr (MAX) {
                    const bool t0 = s_there[buf][half * 2];
                    const bool t1 = s_there[buf][half * 2 + 1];
                    if (t0 || t1)
                        half_tile(buf, half, pu, t0, t1, True{}, MAX_);
                } else if (pu + 32 <= least) {
                    half_tile(buf, half, pu, true, true, False{}, MAX_);
                } else {
                    half_tile(buf, half, pu, true, true, True{}, MAX_);
                }
            }
            if (more) stage(buf ^ 1);
            __syncthreads();
        }
    };
    // Exponentials relative to 0 need no maximum, and are as exact where
    // they neither overflow nor vanish; where some row's might have, or where
    // a page is missing, the workgroup goes the general way.
    bool odd = false;
    for (int p = begin + tid * 16; p < end; p += 256 * 16)
        odd |= !a.kv.rows16(s.b, p, head, D);
    if (!__syncthreads_or(odd)) {
        pass(False{});
        #pragma unroll
        for (int w = 0; w < RW; w++) {
            const float sum = wave_xor_sum(wave_xor_sum(l[w], 16), 32);
            odd |= begin < min(end, seen[w]) &&
                !(sum > 0x1p-60f && sum < 0x1p120f);
        }
        odd = __syncthreads_or(odd);
    } else {
        odd = true;
    }
    if (odd) pass(True{});
    #pragma unroll
    for (int w = 0; w < RW; w++) {
        const float top = wave_xor_max(wave_xor_max(m[w], 16), 32);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = l[w] * exp2_fast(m[w] - ref);
        sum = wave_xor_sum(wave_xor_sum(sum, 16), 32);
        const int r = r0 + w * 16 + n;
        if (g == 0 && r < R) store_sum(a, s, head, r, top, sum);
    }
}

// Pass 1 for few rows, grid as above: 16 * RW rows a workgroup, whose four
// waves take 32 places each in turn, with keys that go straight to registers.
// Bound by the reads of the keys.
template <class C, int NQ, int D, int RW>
__global__ __launch_bounds__(256) void k_kv_observe_few(ObserveArgs a) {
    constexpr int ROWS = 16 * RW;
    __shared__ float s_m[WAVES][ROWS], s_l[WAVES][ROWS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4, head = blockIdx.y;
    const int G = a.group.d;
    Seq s{};
    const int id = late_block<ROWS>(a, s);
    if (id < 0) return;
    const int R = s.m * G, r0 = id * ROWS;
    const int most = sees(s, a.group.of(min(r0 + ROWS, R) - 1));
    const int least = sees(s, a.group.of(r0));
    const int begin = blockIdx.z * a.part, end = min(begin + a.part, most);

    u32x4 q[RW][NQ][D / 32];
    float m[RW], l[RW];
    int seen[RW];
    #pragma unroll
    for (int w = 0; w < RW; w++) {
        const int r = r0 + w * 16 + n, i = a.group.of(r), h = r - i * G;
        load_q<C, NQ, D>(a.q.data, (int64_t)(s.t0 + i) * a.q.row_stride
                             + (int64_t)(head * G + h) * a.q.head_stride,
                         r < R, g, q[w]);
        seen[w] = r < R ? sees(s, i) : 0;
        m[w] = -INFINITY;
        l[w] = 0.f;
    }
    for (int p0 = begin + wave * TILE; p0 < end; p0 += UNIT) {
        const uint16_t* rows[2];
        rows[0] = a.kv.rows16(s.b, p0, head, D);
        rows[1] = p0 + 16 < end ? a.kv.rows16(s.b, p0 + 16, head, D)
                                : nullptr;
        u32x4 k[2][D / 32];
        #pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint16_t* kp = (rows[u] ? rows[u] : a.kv.pool) + n * D
                + g * 8;
            #pragma unroll
            for (int kk = 0; kk < D / 32; kk++)
                k[u][kk] = *reinterpret_cast<const u32x4*>(kp + kk * 32);
        }
        const bool whole = rows[0] && rows[1] && p0 + TILE <= least;
        #pragma unroll
        for (int w = 0; w < RW; w++) {
            f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            #pragma unroll
            for (int x = NQ - 1; x >= 0; x--)
                #pragma unroll
                for (int kk = 0; kk < D / 32; kk++)
                    #pragma unroll
                    for (int u = 0; u < 2; u++)
                        acc[u] = C::mfma(k[u][kk], q[w][x][kk], acc[u]);
            float e[8], top = m[w];
            #pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = acc[j >> 2][j & 3] * a.scale2;
                if (!whole && (!rows[j >> 2] ||
                        p0 + (j >> 2) * 16 + g * 4 + (j & 3) >= seen[w]))
                    e[j] = -INFINITY;
                top = fmaxf(top, e[j]);
            }
            const float ref = top == -INFINITY ? 0.f : top;
            l[w] *= exp2_fast(m[w] - ref);
            m[w] = top;
            #pragma unroll
            for (int j = 0; j < 8; j++) l[w] += exp2_fast(e[j] - ref);
        }
    }
    #pragma unroll
    for (int w = 0; w < RW; w++) {
        const float top = wave_xor_max(wave_xor_max(m[w], 16), 32);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = l[w] * exp2_fast(m[w] - ref);
        sum = wave_xor_sum(wave_xor_sum(sum, 16), 32);
        if (g == 0) {
            s_m[wave][w * 16 + n] = top;
            s_l[wave][w * 16 + n] = sum;
        }
    }
    __syncthreads();
    if (tid < ROWS && r0 + tid < R) {
        float top = -INFINITY, sum = 0.f;
        #pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, s_m[w][tid]);
        const float ref = top == -INFINITY ? 0.f : top;
        #pragma unroll
        for (int w = 0; w < WAVES; w++)
            sum += s_l[w][tid] * exp2_fast(s_m[w][tid] - ref);
        store_sum(a, s, head, r0 + tid, top, sum);
    }
}

// Join the parts of the rows' sums: 32 rows a workgroup, the parts dealt to 8
// threads of each. A part that its row does not see gave (-inf, 0).
__global__ __launch_bounds__(256) void k_kv_observe_join(ObserveArgs a) {
    __shared__ float s_m[8][32], s_l[8][32];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t at = (int64_t)blockIdx.x * 32 + x;
    const int64_t all = (int64_t)a.q_heads * a.rows;
    float m = -INFINITY, l = 0.f;
    auto join = [&](float mp, float lp) {
        const float now = fmaxf(m, mp);
        const float ref = now == -INFINITY ? 0.f : now;
        l = l * exp2_fast(m - ref) + lp * exp2_fast(mp - ref);
        m = now;
    };
    if (at < all) {
        #pragma unroll 4
        for (int p = y; p < a.parts; p += 8) {
            const f32x2 s = *reinterpret_cast<const f32x2*>(
                a.sums + (p * all + at) * 2);
            join(s.x, s.y);
        }
    }
    s_m[y][x] = m;
    s_l[y][x] = l;
    __syncthreads();
    if (y || at >= all) return;
    for (int i = 1; i < 8; i++) join(s_m[i][x], s_l[i][x]);
    *reinterpret_cast<f32x2*>(a.norm + at * 2) = row_norm(m, l);
}

// Pass 2, grid (place blocks x chunks, kv heads): 16 * PW places a
// wave, whose keys stay in registers, over the chunk's rows, which the
// workgroup stages QT at a time; a lane sums its columns' weights for its
// places. The same work a score as in pass 1. Where a sequence's rows are one
// chunk the sums go to the mass, else to `partial`, and the last kernel adds
// them in order.
template <class C, int NQ, int D, int PW>
__global__ __launch_bounds__(256) void k_kv_observe_mass(ObserveArgs a) {
    constexpr int QT = NQ == 1 ? 64 : 32, UNITS = QT * D / 8;
    constexpr int PER = (UNITS + 255) / 256;
    __shared__ __align__(16) uint16_t s_q[2][NQ][QT * LDS_ROW<D>];
    __shared__ f32x2 s_norm[2][QT];
    __shared__ int s_seen[2][QT];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4, head = blockIdx.y;
    const int G = a.group.d;
    // chunks differ in their work (late ones are seen by more places, short
    // sequences have less): turned by one from block to block and from head to
    // head, so that no XCD (every eighth workgroup) gets the long ones (both
    // passes for 7 x 251 rows of 32 kv heads: 270 us, 279 turned by block alone,
    // 370 not turned; 4 x 282 float32 rows of 8: 89, 104 and 85; 3 x 500 over
    // 16000 places: 466, 461 and 469)
    const int block = blockIdx.x / a.chunks;
    const int at = (blockIdx.x + block + head) % a.chunks;
    Seq s{};
    const RowBlock x = row_block(a, a.chunk, at, s);
    if (x.id < 0) return;
    const int chunk = x.id;
    const int first = block * 16 * PW * WAVES, p0 = first + wave * 16 * PW;
    const int R = s.m * G;
    // rows from the first that sees the block's first place on
    const int from = max(0, first - s.before) * G;
    const int begin = max(chunk * a.chunk, from / QT * QT);
    const int end = min(chunk * a.chunk + a.chunk, R);
    if (first >= s.len || begin >= end) return;

    u32x4 k[PW][D / 32];
    bool there[PW];
    #pragma unroll
    for (int u = 0; u < PW; u++) {
        const uint16_t* rows = p0 + u * 16 < s.len
            ? a.kv.rows16(s.b, p0 + u * 16, head, D) : nullptr;
        there[u] = rows != nullptr;
        if (!rows) rows = a.kv.pool;
        #pragma unroll
        for (int kk = 0; kk < D / 32; kk++)
            k[u][kk] = *reinterpret_cast<const u32x4*>(
                rows + n * D + kk * 32 + g * 8);
    }
    f32x4 sum[PW];
    #pragma unroll
    for (int u = 0; u < PW; u++) sum[u] = f32x4{0.f, 0.f, 0.f, 0.f};

    // a thread's units of a tile of queries: where they are, and their rows'
    // heads, both moved on from tile to tile
    constexpr int FULL = NQ > 1 ? 2 : 1;
    const char* from_q[PER];
    int h_of[PER];
    u32x4 next[PER][FULL];
    const int64_t size = NQ > 1 ? 4 : 2;
    const int step_i = a.group.of(QT), step_h = QT - step_i * G;
    const int64_t step = (step_i * a.q.row_stride
                          + step_h * a.q.head_stride) * size;
    const int64_t wrap = (a.q.row_stride - G * a.q.head_stride) * size;
    #pragma unroll
    for (int x = 0; x < PER; x++) {
        const int u = x * 256 + tid, r = begin + u / (D / 8);
        const int i = a.group.of(r);
        h_of[x] = r - i * G;
        from_q[x] = reinterpret_cast<const char*>(a.q.data)
            + ((int64_t)(s.t0 + i) * a.q.row_stride
               + (int64_t)(head * G + h_of[x]) * a.q.head_stride
               + u % (D / 8) * 8) * size;
    }
    const f32x2* from_norm = reinterpret_cast<const f32x2*>(a.norm)
        + ((int64_t)head * a.rows + s.t0) * G;
    f32x2 next_norm = {INFINITY, 0.f};
    int next_seen = 0;
    auto fetch = [&](int r0) {
        #pragma unroll
        for (int x = 0; x < PER; x++) {
            const int u = x * 256 + tid;
            const bool there = (UNITS % 256 == 0 || u < UNITS)
                && r0 + u / (D / 8) < R;
            #pragma unroll
            for (int y = 0; y < FULL; y++)
                next[x][y] = there
                    ? reinterpret_cast<const u32x4*>(from_q[x])[y]
                    : u32x4{0, 0, 0, 0};
            from_q[x] += step;
            if (step_h) {
                h_of[x] += step_h;
                if (h_of[x] >= G) {
                    h_of[x] -= G;
                    from_q[x] += wrap;
                }
            }
        }
        if (tid < QT) {
            const int r = r0 + tid;
            next_norm = r < R ? from_norm[r] : f32x2{INFINITY, 0.f};
            next_seen = r < R ? sees(s, a.group.of(r)) : 0;
        }
    };
    auto stage = [&](int buf) {
        #pragma unroll
        for (int x = 0; x < PER; x++) {
            const int u = x * 256 + tid;
            if (UNITS % 256 && u >= UNITS) break;
            const int at = u / (D / 8) * LDS_ROW<D> + u % (D / 8) * 8;
            if constexpr (NQ == 1) {
                *reinterpret_cast<u32x4*>(&s_q[buf][0][at]) = next[x][0];
            } else {
                const f32x4 f0 = bits<f32x4>(next[x][0]);
                const f32x4 f1 = bits<f32x4>(next[x][1]);
                float f[8] = {f0[0], f0[1], f0[2], f0[3],
                              f1[0], f1[1], f1[2], f1[3]};
                #pragma unroll
                for (int p = 0; p < NQ; p++) {
                    u32x4 w;
                    #pragma unroll
                    for (int i = 0; i < 4; i++)
                        w[i] = C::piece(f[2 * i], f[2 * i + 1]);
                    *reinterpret_cast<u32x4*>(&s_q[buf][p][at]) = w;
                }
            }
        }
        if (tid < QT) {
            s_norm[buf][tid] = next_norm;
            s_seen[buf][tid] = next_seen;
        }
    };
    // 16 rows against the wave's places. CUT: some row does not see them all
    auto rows16 = [&](const u32x4 (*q)[D / 32], f32x2 norm, int seen,
                      auto CUT) {
        f32x4 acc[PW];
        #pragma unroll
        for (int u = 0; u < PW; u++) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int x = NQ - 1; x >= 0; x--)
            #pragma unroll
            for (int kk = 0; kk < D / 32; kk++)
                #pragma unroll
                for (int u = 0; u < PW; u++)
                    acc[u] = C::mfma(k[u][kk], q[x][kk], acc[u]);
        #pragma unroll
        for (int u = 0; u < PW; u++)
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                const float w = exp2_fast(fmaf(acc[u][e], a.scale2, -norm.x));
                if (!CUT || p0 + u * 16 + g * 4 + e < seen)
                    sum[u][e] = fmaf(w, norm.y, sum[u][e]);
            }
    };
    fetch(begin);
    stage(0);
    #pragma unroll
    for (int u = 0; u < PW; u++)
        #pragma unroll
        for (int kk = 0; kk < D / 32; kk++) arrive(k[u][kk]);
    __syncthreads();
    int buf = 0;
    for (int r0 = begin; r0 < end; r0 += QT, buf ^= 1) {
        const bool more = r0 + QT < end;
        if (more) fetch(r0 + QT);
        #pragma unroll
        for (int t = 0; t < QT / 16; t++) {
            const int r = r0 + t * 16;
            u32x4 q[NQ][D / 32];
            #pragma unroll
            for (int x = 0; x < NQ; x++)
                #pragma unroll
                for (int kk = 0; kk < D / 32; kk++)
                    q[x][kk] = lds_unit<D>(s_q[buf][x], t * 16 + n,
                                           kk * 4 + g);
            const f32x2 norm = s_norm[buf][t * 16 + n];
            const int seen = s_seen[buf][t * 16 + n];
            // the first of 16 rows sees the least; rows past the last see none
            if (r + 16 <= R &&
                p0 + 16 * PW <= sees(s, a.group.of(r)))
                rows16(q, norm, seen, False{});
            else
                rows16(q, norm, seen, True{});
        }
        if (more) stage(buf ^ 1);
        __syncthreads();
    }
    float* to = x.all == 1
        ? reinterpret_cast<float*>(a.mass.data) + s.b * a.mass.slot_stride
            + head * a.mass.head_stride
        : a.partial + ((int64_t)at * a.kv_heads + head) * a.ld;
    #pragma unroll
    for (int u = 0; u < PW; u++)
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            float w = sum[u][e];
            #pragma unroll
            for (int x = 1; x < 16; x <<= 1) w = wave_xor_sum(w, x);
            const int p = p0 + u * 16 + g * 4 + e;
            if (n == 0 && p < s.len) {
                if (x.all > 1) to[p] = there[u] ? w : 0.f;
                else if (there[u]) to[p] += w;
            }
        }
}

// Add a sequence's chunks, of which it has more than one: those that the second
// pass made, in their order.
__global__ __launch_bounds__(256) void k_kv_observe_add(ObserveArgs a) {
    const int p = blockIdx.x * 256 + threadIdx.x, head = blockIdx.y;
    const int lane = threadIdx.x & 63, b = blockIdx.z;
    const Seq s = sequence_at(a, b);
    const int G = a.group.d, R = s.m * G;
    if ((int)blockIdx.x * 256 >= s.len || R <= a.chunk) return;
    // (`starts` out of order may make more chunks than there are)
    int before = 0;
    for (int x = lane; x < b; x += 64)
        before = min(before + (sequence_at(a, x).m * G + a.chunk - 1) / a.chunk,
                     a.chunks);
    #pragma unroll
    for (int x = 1; x < 64; x <<= 1) before += __shfl_xor(before, x, 64);
    const int from = max(0, p / a.block * a.block - s.before) * G;
    if (p >= s.len || from >= R) return;
    const int64_t step = (int64_t)a.kv_heads * a.ld;
    const float* part = a.partial + before * step + (int64_t)head * a.ld + p;
    const int end = min((R - 1) / a.chunk + 1, a.chunks - before);
    float w = 0.f;
    #pragma unroll 8
    for (int c = from / a.chunk; c < end; c++) w += part[c * step];
    reinterpret_cast<float*>(a.mass.data)[
        s.b * a.mass.slot_stride + head * a.mass.head_stride + p] += w;
}

// -------------------------------------------------------------------- evict

struct EvictArgs {
    Pages kv;
    int64_t layer_stride;
    KvLayers mass, pos, mass_out, pos_out;
    const int32_t *lens, *next_pos;
    int32_t* lens_out;
    int32_t layers, slots, kv_heads, keep, recent, limit, reach, most;
    int32_t *count, *dst, *src;    // [rows], [rows][most] twice
};

__device__ __forceinline__ int64_t row_at(const KvLayers& t, int layer, int b,
                                          int h) {
    return layer * t.layer_stride + b * t.slot_stride + h * t.head_stride;
}

// Sums over the workgroup's NW waves, in their order.
struct WaveSums {
    uint32_t before, all;
};

template <int NW>
__device__ __forceinline__ WaveSums wave_sums(uint32_t x, uint32_t* red,
                                              int wave) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = x;
    __syncthreads();
    WaveSums s{0, 0};
    #pragma unroll
    for (int w = 0; w < NW; w++) {
        const uint32_t y = red[w];
        if (w < wave) s.before += y;
        s.all += y;
    }
    return s;
}

// Pass 1, one workgroup of NT a row (layer, sequence, kv head): which places
// stay, and who moves where. Each wave has a stretch of the row, of which a
// thread holds the keys of up to KPT places, or, with KPT = 0, computes them
// each time it goes through them. The keep-th largest key is found eight bits
// at a time, by counting the digits of the keys that begin as it does in LDS;
// that ends early once exactly `keep` keys are at or above a digit. Then each
// wave counts its free places and those that come into them, and numbers them
// on from the counts of the waves before it.
//
// With the moves, NT 1024: KPT 8 serves rows of up to 8192 places (256 rows of
// 8192: 131 us, 133 with KPT 32, 145 with 0), 32 up to 32768 (128 of 20000: 170
// us, 215 with 0). NT 256, KPT 8 up to 2048 places (2304 rows of 318: 26 us, 66
// with 1024 threads; 8 of 512: 11.3, 13.5; 192 of 2048: 23 either way). The 256
// rows of 8192 are selected in 22.6 us, bound by the counting: keys of one
// exponent meet in few digits (the first one's lanes are added at once). Two
// bits a round, by ballots over three candidates, took 28.
template <int NT, int KPT>
__global__ __launch_bounds__(NT) void k_kv_evict_select(EvictArgs a) {
    constexpr int NW = NT / 64;
    __shared__ __align__(16) uint32_t digits[4][256];
    __shared__ uint32_t tot[NW];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x;
    const int h = row % a.kv_heads, b = row / a.kv_heads % a.slots,
              layer = row / a.kv_heads / a.slots;
    const float* mass = reinterpret_cast<const float*>(a.mass.data)
        + row_at(a.mass, layer, b, h);
    const int32_t* pos = reinterpret_cast<const int32_t*>(a.pos.data)
        + row_at(a.pos, layer, b, h);
    float* mass_out = reinterpret_cast<float*>(a.mass_out.data)
        + row_at(a.mass_out, layer, b, h);
    int32_t* pos_out = reinterpret_cast<int32_t*>(a.pos_out.data)
        + row_at(a.pos_out, layer, b, h);
    const int len = kv_clamp_len(a.lens[b], a.reach);
    const int64_t late = (int64_t)a.next_pos[b] - a.recent;
    const bool copies = mass_out != mass, copied = pos_out != pos;
    const bool full = len > a.limit;
    if (!full && tid == 0) a.count[row] = -1;
    if (!full && !copies && !copied) return;

    const int blocks = (len + NT - 1) / NT;
    const int p0 = wave * blocks * 64 + lane;     // places p0 + k * 64
    auto key_at = [&](int p) {
        return kv_rank_key(mass[p], pos[p] >= late);
    };
    uint32_t held[KPT ? KPT : 1];
    int copied_to = 0;
    if constexpr (KPT > 0) {
        // eight at a time without a branch between their loads
        #pragma unroll
        for (int k0 = 0; k0 < KPT; k0 += 8) {
            #pragma unroll
            for (int k = k0; k < k0 + 8; k++) held[k] = 0;
            if (k0 >= blocks) continue;
            float m[8];
            int32_t at[8];
            #pragma unroll
            for (int k = 0; k < 8; k++) {
                const int p = min(p0 + (k0 + k) * 64, len - 1);
                m[k] = mass[p];
                at[k] = pos[p];
            }
            #pragma unroll
            for (int k = 0; k < 8; k++) {
                const int p = p0 + (k0 + k) * 64;
                if (k0 + k < blocks && p < len) {
                    if (copies) mass_out[p] = m[k];
                    if (copied) pos_out[p] = at[k];
                    held[k0 + k] = kv_rank_key(m[k], at[k] >= late);
                }
            }
        }
        copied_to = len;
    }
    for (int p = copied_to + tid; p < a.reach; p += NT) {
        if (copies) mass_out[p] = mass[p];
        if (copied) pos_out[p] = pos[p];
    }
    if (!full) return;
    for (int i = tid; i < 4 * 256; i += NT) digits[i >> 8][i & 255] = 0;
    __syncthreads();
    // the wave's keys in order
    auto each = [&](auto f) {
        if constexpr (KPT > 0) {
            #pragma unroll
            for (int k = 0; k < KPT; k++)
                if (k < blocks) f(p0 + k * 64, held[k]);
        } else {
            for (int k = 0; k < blocks; k++) {
                const int p = p0 + k * 64;
                f(p, p < len ? key_at(p) : 0u);
            }
        }
    };

    // `want` of the keys that begin as `least` does are still to be found. A
    // key past the end is 0, as a NaN's: as there are more than `keep` places,
    // counting it too makes no group of the lowest keys exact
    uint32_t least = 0, want = a.keep;
    bool exact = false;
    #pragma unroll 1
    for (int turn = 0; turn < 4 && !exact; turn++) {
        const int shift = 24 - 8 * turn;
        each([&](int, uint32_t key) {
            // 64 bits: in the first turn nothing is left to compare
            const bool of = !((uint64_t)(key ^ least) >> (shift + 8));
            const uint32_t digit = key >> shift & 255;
            const uint64_t all = __ballot(of);
            if (!all) return;
            // the first one's digit, which many may share, is added at once
            const int first = __builtin_ctzll(all);
            const bool same =
                digit == (uint32_t)__builtin_amdgcn_readlane(digit, first);
            const uint64_t sames = __ballot(of && same);
            if (of && (!same || lane == first))
                atomicAdd(&digits[turn][digit],
                          same ? (uint32_t)__popcll(sames) : 1u);
        });
        __syncthreads();
        // the digit at which the count from the highest down reaches `want`:
        // four digits a lane
        const u32x4 n =
            *reinterpret_cast<const u32x4*>(&digits[turn][lane * 4]);
        uint32_t from = n.x + n.y + n.z + n.w;
        #pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t x = __shfl_down(from, m, 64);
            if (lane + m < 64) from += x;
        }
        const int at = 63 - __builtin_clzll(__ballot(from >= want));
        const uint32_t n3 = __builtin_amdgcn_readlane(n.w, at),
                       n2 = __builtin_amdgcn_readlane(n.z, at),
                       n1 = __builtin_amdgcn_readlane(n.y, at),
                       n0 = __builtin_amdgcn_readlane(n.x, at);
        uint32_t left = want - (__builtin_amdgcn_readlane(from, at)
                                - n0 - n1 - n2 - n3);
        uint32_t digit = at * 4 + 3, count = n3;
        if (left > count) { left -= count; digit--; count = n2; }
        if (left > count) { left -= count; digit--; count = n1; }
        if (left > count) { left -= count; digit--; count = n0; }
        least |= digit << shift;
        want = left;
        exact = count == left;
    }
    // of the keys equal to `least`, the first `ties` of the wave's stay
    int ties = INT_MAX;
    if (!exact) {
        uint32_t equal = 0;
        each([&](int p, uint32_t key) {
            equal += __popcll(__ballot(p < len && key == least));
        });
        ties = (int)want - (int)wave_sums<NW>(equal, tot, wave).before;
    }

    const uint64_t below = (1ull << lane) - 1;
    // f(place, whether it is free, whether it comes): ballots of the two
    auto walk = [&](auto f) {
        int left = ties;
        each([&](int p, uint32_t key) {
            bool stays = p < len && key >= least;
            if (!exact) {
                const uint64_t eqs = __ballot(p < len && key == least);
                // negative where the waves before have them all
                if (key == least) stays &= (int)__popcll(eqs & below) < left;
                left -= (int)__popcll(eqs);
            }
            f(p, __ballot(p < min(len, a.keep) && !stays),
              __ballot(stays && p >= a.keep));
        });
    };
    uint32_t free = 0, come = 0;
    walk([&](int, uint64_t fs, uint64_t cs) {
        free += __popcll(fs);
        come += __popcll(cs);
    });
    free = wave_sums<NW>(free, tot, wave).before;
    const WaveSums comes = wave_sums<NW>(come, tot, wave);
    come = comes.before;
    int32_t* dst = a.dst + (int64_t)row * a.most;
    int32_t* src = a.src + (int64_t)row * a.most;
    walk([&](int p, uint64_t fs, uint64_t cs) {
        if (fs >> lane & 1) dst[free + __popcll(fs & below)] = p;
        if (cs >> lane & 1) src[come + __popcll(cs & below)] = p;
        free += __popcll(fs);
        come += __popcll(cs);
    });
    come = comes.all;
    if (tid == 0) a.count[row] = come;
    __syncthreads();
    for (uint32_t i = tid; i < come; i += NT) {
        const int d = dst[i], s = src[i];
        mass_out[d] = mass[s];
        pos_out[d] = pos[s];
    }
}

// Pass 2, grid (rows, blocks of moves): the movers' keys and values, 16
// lanes a row. Sources are at or above keep and destinations below it, so
// no order is needed. 2048 places of 256 rows (537 MB read and written) take
// 108 us, the rate of a large copy.
__global__ __launch_bounds__(256) void k_kv_evict_move(EvictArgs a, int dim) {
    const int row = blockIdx.x;
    const int h = row % a.kv_heads, b = row / a.kv_heads % a.slots,
              layer = row / a.kv_heads / a.slots;
    const int count = a.count[row];
    if (blockIdx.y == 0 && h == 0 && layer == 0 && threadIdx.x == 0)
        a.lens_out[b] = count < 0 ? a.lens[b] : a.keep;
    const int32_t* table = a.kv.table + (int64_t)b * a.kv.table_stride;
    const int l16 = threadIdx.x & 15;
    auto where = [&](int p) -> uint16_t* {
        const int32_t pg = kv_page_of(table, p / a.kv.page, a.kv.max_pages,
                                      a.kv.pages);
        if (pg < 0) return nullptr;
        return a.kv.pool + layer * a.layer_stride
            + (int64_t)pg * a.kv.page_stride
            + (int64_t)h * 2 * a.kv.page * dim
            + (int64_t)(p % a.kv.page) * dim;
    };
    const int64_t to_v = (int64_t)a.kv.page * dim;
    for (int i = blockIdx.y * 16 + (threadIdx.x >> 4); i < count;
         i += gridDim.y * 16) {
        const uint16_t* s = where(a.src[(int64_t)row * a.most + i]);
        uint16_t* d = where(a.dst[(int64_t)row * a.most + i]);
        if (!s || !d || l16 * 8 >= dim) continue;
        const u32x4 k = *reinterpret_cast<const u32x4*>(s + l16 * 8);
        const u32x4 v = *reinterpret_cast<const u32x4*>(s + to_v + l16 * 8);
        *reinterpret_cast<u32x4*>(d + l16 * 8) = k;
        *reinterpret_cast<u32x4*>(d + to_v + l16 * 8) = v;
    }
}

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

#define KV_DIM(D_, ...)                                                       \
    do {                                                                      \
        if ((D_) == 128) { constexpr int D = 128; __VA_ARGS__; }              \
        else if ((D_) == 96) { constexpr int D = 96; __VA_ARGS__; }           \
        else { constexpr int D = 64; __VA_ARGS__; }                           \
    } while (0)

// q's type over the pool's: the pool's own, or float32 over bfloat16. NQ and NP
// pieces of queries and weights. All 24 bits of a weight over bfloat16, also
// where the output has 8: two pieces were cut by up to 2^-15, all the same way,
// which changed one output in 200, and took as long (64 sequences of up to
// 4096 places: 49.3 us)
#define KV_TYPES(Q_, C_, ...)                                                 \
    do {                                                                      \
        if ((C_) == KVT::F16) {                                               \
            if ((Q_) != KVT::F16) bad_types();                                \
            typedef F16 C; constexpr int NQ = 1, NP = 2; (void)NP;            \
            __VA_ARGS__;                                                      \
        } else if ((Q_) == KVT::BF16) {                                       \
            typedef Bf16 C; constexpr int NQ = 1, NP = 3; (void)NP;           \
            __VA_ARGS__;                                                      \
        } else {                                                              \
            if ((Q_) != KVT::F32) bad_types();                                \
            typedef Bf16 C; constexpr int NQ = 3, NP = 3; (void)NP;           \
            __VA_ARGS__;                                                      \
        }                                                                     \
    } while (0)

[[noreturn]] void bad_types() {
    throw std::runtime_error(
        "queries must have the pool's type, or float32 over bfloat16");
}

}  // namespace

void launch_kv_append(const KvPages& kv, const KvHeads& k, const KvHeads& v,
                      const KvHeads& q, const KvHeads& q_out, int q_heads,
                      KVT type, int rows, const int32_t* starts,
                      const int32_t* lens, const int32_t* next_pos,
                      const float* inv_freq, const KvRows& mass,
                      const KvRows& pos, int reach, hipStream_t stream) {
    check_pages(kv, 0, reach);
    if (rows <= 0) return;
    if (!starts && rows != kv.slots)
        throw std::runtime_error("append: one row for each sequence");
    check_grid(rows);
    AppendArgs a{pages_of(kv), k, v, q, q_out, mass, pos, starts, lens,
                 next_pos, inv_freq, q.data ? q_heads : 0, kv.kv_heads,
                 kv.slots, reach};
    // few rows: a row's heads over several workgroups
    const int items = (a.q_heads + 2 * kv.kv_heads) * (kv.dim / 8);
    const dim3 grid(rows, rows < 256 ? (items + 255) / 256 : 1);
    #define APPEND(T, C)                                                      \
        KV_DIM(kv.dim, hipLaunchKernelGGL((k_kv_append<T, C, D>), grid,       \
                                          dim3(256), 0, stream, a))
    if (kv.type == KVT::F16) {
        if (type != KVT::F16) bad_types();
        APPEND(KVT::F16, KVT::F16);
    } else if (type == KVT::BF16) {
        APPEND(KVT::BF16, KVT::BF16);
    } else {
        if (type != KVT::F32) bad_types();
        APPEND(KVT::F32, KVT::BF16);
    }
    #undef APPEND
    check_launch();
}

void launch_kv_step(int32_t* len, int32_t* step, const uint8_t* active,
                    int slots, hipStream_t stream) {
    hipLaunchKernelGGL(k_kv_step, dim3(1), dim3(64), 0, stream, len, step,
                       active, slots);
    check_launch();
}

namespace {
int64_t attend_wgs(const KvPages& kv, int reach) {
    const int64_t rows = (int64_t)kv.slots * kv.kv_heads;
    return std::min(attend_target(kv) + rows,
                    rows * std::max(1, (reach + UNIT - 1) / UNIT));
}
// Whether a row's places, which `reach` bounds, are one workgroup's: one launch
// and no join then take less time than more workgroups save. 8 rows of up to 300
// places 8.8 us, 12.1 in parts; 64 of 700, 14 and 14; 8 of 1000, 15.4 and 12.1;
// 128 of 1000, 17 and 19.5; 256 of 1000, 19 and 28; 1024 of 300, 36 and 38; but
// 2048 of 200, 61 and 52 (its LDS leaves a CU one workgroup).
bool attend_rows(const KvPages& kv, int reach) {
    const int64_t rows = (int64_t)kv.slots * kv.kv_heads;
    return rows <= 1024 && reach <= (rows < 128 ? 768 : ROW_PLACES);
}
int64_t scores_ld(int reach) { return (int64_t)(reach + 31) / 32 * 32; }
}  // namespace

size_t kv_attend_workspace(const KvPages& kv, int q_heads, int reach,
                           bool mass) {
    check_pages(kv, q_heads, reach);
    if (attend_rows(kv, reach)) return 0;
    const int64_t wgs = attend_wgs(kv, reach), G = q_heads / kv.kv_heads;
    return aligned(wgs * G * kv.dim * 4) + aligned(wgs * G * 2 * 4)
        + aligned(wgs * sizeof(Part)) + (mass ? aligned((size_t)kv.slots * q_heads * scores_ld(reach) * 4)
                : 0);
}

void launch_kv_attend(const KvPages& kv, const KvHeads& q, const KvHeads& out,
                      int q_heads, KVT type, const int32_t* lens, int add,
                      const KvRows& mass, int reach, float scale, void* ws,
                      hipStream_t stream) {
    check_pages(kv, q_heads, reach);
    check_scale(scale);
    const int64_t wgs = attend_wgs(kv, reach), G = q_heads / kv.kv_heads;
    check_grid(wgs);
    char* w = reinterpret_cast<char*>(ws);
    AttendArgs a{pages_of(kv), q, out, mass, lens, add, q_heads, kv.kv_heads,
                 kv.slots, reach, attend_target(kv), scale * LOG2E, nullptr,
                 scores_ld(reach), nullptr, nullptr, nullptr};
    a.part_o = reinterpret_cast<float*>(w);
    w += aligned(wgs * G * kv.dim * 4);
    a.part_ml = reinterpret_cast<float*>(w);
    w += aligned(wgs * G * 2 * 4);
    a.parts = reinterpret_cast<Part*>(w);
    w += aligned(wgs * sizeof(Part));
    a.scores = reinterpret_cast<float*>(w);
    if (attend_rows(kv, reach)) {
        #define ATTEND(M)                                                     \
            KV_TYPES(type, kv.type, KV_DIM(kv.dim,                            \
                hipLaunchKernelGGL((k_kv_attend_row<C, NQ, NP, D, M>),        \
                                   dim3(kv.kv_heads, kv.slots),               \
                                   dim3(64 * ROW_WAVES), 0, stream, a)))
        if (mass.data) ATTEND(true); else ATTEND(false);
        #undef ATTEND
        check_launch();
        return;
    }
    const dim3 grid((uint32_t)wgs), block(256);
    #define ATTEND(M)                                                         \
        KV_TYPES(type, kv.type, KV_DIM(kv.dim, {                              \
            hipLaunchKernelGGL((k_kv_attend<C, NQ, NP, D, M>), grid, block,   \
                               0, stream, a);                                 \
            hipLaunchKernelGGL((k_kv_join<C, (NQ > 1), D, M>), grid, block,   \
                               0, stream, a);                                 \
        }))
    if (mass.data) ATTEND(true); else ATTEND(false);
    #undef ATTEND
    check_launch();
}

namespace {

// How the two passes of observe are cut: into workgroups of OBSERVE_TILES
// tiles (64 x 256 scores of a kv head) at least, but 512 and no more than 4096
// of them: a pass with fewer waits for its longest ones (causal rows and
// places are uneven), one with more begins too often.
constexpr int OBSERVE_TILES_1 = 8, OBSERVE_TILES_2 = 8;

inline int64_t observe_wgs(int64_t tiles, int per) {
    return std::min<int64_t>(4096, std::max<int64_t>(512, tiles / per));
}

struct ObserveCut {
    int64_t blocks, parts, part, chunks, chunk, block, place_blocks;
    bool two;                       // a wave holds two groups of places
    bool several;                   // a sequence may have several chunks
    int64_t sums, norm, partial;    // bytes
};

// Rows of a workgroup of the first pass in its form for few rows; 0: the other
// form. For few rows a sequence on average (both passes for up to 4 rows of 8
// sequences of up to 3867 places, 32 kv heads: 86 us, 120 in the other form; 16
// x 4 tokens of 32 / 8 heads over up to 131071 places: 1147 us, 1472), and where
// the other form would not have 256 workgroups (4 x 100 tokens over 500 places:
// 26 us, 32 in the other form; 500 rows, 2000 places, 16 heads of 64: 28 us, 33;
// with more of them it loses, 512 tokens over 8000 places: 142 us, 97).
int64_t observe_few(const KvPages& kv, int q_heads, int rows, int reach,
                    KVT type) {
    const int64_t R = (int64_t)rows * (q_heads / kv.kv_heads);
    const int64_t most = type == KVT::F32 ? 32 : 64;   // what registers hold
    if (R <= 16ll * kv.slots) return 16;
    const int64_t per = 4 * most;                      // the other form's
    const int64_t wgs = ((R + per - 1) / per + kv.slots - 1) * kv.kv_heads
        * ((reach + 511) / 512);
    return R <= most * kv.slots || wgs < 256 ? most : 0;
}

ObserveCut observe_cut(const KvPages& kv, int q_heads, int rows, int reach,
                       KVT type) {
    if ((int64_t)rows * (q_heads / kv.kv_heads) >= (1ll << 28))
        throw std::runtime_error("observe: too many rows");
    const int64_t G = q_heads / kv.kv_heads, R = std::max<int64_t>(rows, 1) * G;
    const int64_t few = observe_few(kv, q_heads, rows, reach, type);
    const int64_t per = few ? few : 16 * WAVES * (type == KVT::F32 ? 2 : 4);
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    ObserveCut c;
    c.blocks = up(R, per) + kv.slots - 1;
    const int64_t places = std::max(reach, 1);
    const int64_t row_blocks = c.blocks * kv.kv_heads;
    c.parts = std::min(
        up(observe_wgs(row_blocks * up(places, 64), OBSERVE_TILES_1),
           row_blocks), up(places, 512));
    c.part = up(up(places, c.parts), 64) * 64;
    c.parts = up(places, c.part);
    // Two groups of 16 places a wave where that many workgroups' worth of
    // tiles of 64 rows would leave most of the chip idle (both passes for 300
    // float32 tokens of 32 / 8 heads: 26 us, 30 with four; 500 rows of 2000
    // places, 16 heads of 64: 28 us, 30.5 with four; 900 float32 tokens of 32 /
    // 8 heads, 1824 tiles: 65 us, 60 with four).
    int64_t blocks;
    for (int groups : {obs_groups(type != KVT::F32, kv.dim), 2}) {
        c.block = 16 * WAVES * groups;
        c.place_blocks = up(places, c.block);
        blocks = c.place_blocks * kv.kv_heads;
        c.two = groups == 2;
        if (blocks * up(R, 64) > 1024) break;
    }
    const int64_t cuts = up(observe_wgs(blocks * up(R, 64), OBSERVE_TILES_2),
                            blocks);
    c.chunk = up(up(R, cuts), 64) * 64;
    c.several = R > c.chunk;
    c.chunks = up(R, c.chunk) + kv.slots - 1;
    c.sums = c.parts > 1 ? aligned((size_t)c.parts * rows * q_heads * 8) : 0;
    c.norm = aligned((size_t)std::max(rows, 1) * q_heads * 8);
    c.partial = c.several
        ? aligned((size_t)c.chunks * kv.kv_heads * c.place_blocks * c.block
                  * 4) : 0;
    return c;
}

}  // namespace

size_t kv_observe_workspace(const KvPages& kv, int q_heads, int rows,
                            int reach, KVT type) {
    check_pages(kv, q_heads, reach);
    const ObserveCut c = observe_cut(kv, q_heads, rows, reach, type);
    return c.sums + c.norm + c.partial;
}

void launch_kv_observe(const KvPages& kv, const KvHeads& q, int q_heads,
                       KVT type, int rows, const int32_t* starts,
                       const int32_t* lens, const KvRows& mass, int reach,
                       float scale, void* ws, hipStream_t stream) {
    check_pages(kv, q_heads, reach);
    check_scale(scale);
    if (rows <= 0 || reach == 0) return;
    const ObserveCut c = observe_cut(kv, q_heads, rows, reach, type);
    if (c.parts > 65535 || kv.kv_heads > 65535 || kv.slots > 65535)
        throw std::runtime_error("observe: too many sequences or kv heads");
    check_grid(c.blocks);
    check_grid(c.place_blocks * c.chunks);
    check_grid((int64_t)rows * q_heads / 32 + 1);
    char* w = reinterpret_cast<char*>(ws);
    ObserveArgs a{pages_of(kv), q, mass, starts, lens, q_heads, kv.kv_heads,
                  kv.slots, rows, reach, scale * LOG2E,
                  div_by(q_heads / kv.kv_heads), (int32_t)c.part,
                  (int32_t)c.parts, (int32_t)c.chunk, (int32_t)c.chunks,
                  (int32_t)c.block,
                  reinterpret_cast<float*>(w),
                  reinterpret_cast<float*>(w + c.sums),
                  reinterpret_cast<float*>(w + c.sums + c.norm),
                  c.place_blocks * c.block};
    KV_TYPES(type, kv.type, KV_DIM(kv.dim, {
        constexpr int RW = NQ > 1 ? 2 : 4, PW = obs_groups(NQ == 1, D);
        const int64_t few = observe_few(kv, q_heads, rows, reach, type);
        auto* sums = few == 16 ? k_kv_observe_few<C, NQ, D, 1>
            : few ? k_kv_observe_few<C, NQ, D, RW>
                  : k_kv_observe_sums<C, NQ, D, RW>;
        hipLaunchKernelGGL(sums, dim3((uint32_t)c.blocks, kv.kv_heads,
                                      (uint32_t)c.parts),
                           dim3(256), 0, stream, a);
        if (c.parts > 1)
            hipLaunchKernelGGL(k_kv_observe_join,
                               dim3((uint32_t)(((int64_t)rows * q_heads + 31)
                                               / 32)),
                               dim3(256), 0, stream, a);
        auto* mass_of = c.two ? k_kv_observe_mass<C, NQ, D, 2>
                              : k_kv_observe_mass<C, NQ, D, PW>;
        hipLaunchKernelGGL(mass_of,
                           dim3((uint32_t)(c.place_blocks * c.chunks),
                                kv.kv_heads),
                           dim3(256), 0, stream, a);
        if (c.several)
            hipLaunchKernelGGL(k_kv_observe_add,
                               dim3((reach + 255) / 256, kv.kv_heads,
                                    kv.slots),
                               dim3(256), 0, stream, a);
    }));
    check_launch();
}

size_t kv_evict_workspace(const KvPages& kv, int layers, int keep, int reach) {
    check_pages(kv, 0, reach);
    const size_t rows = (size_t)layers * kv.slots * kv.kv_heads;
    const size_t most = std::max(0, std::min(keep, reach - keep));
    return aligned(rows * 4) + 2 * aligned(rows * most * 4 + 4);
}

void launch_kv_evict(const KvPages& kv, int layers, int64_t layer_stride,
                     const int32_t* lens, int32_t* lens_out,
                     const int32_t* next_pos, const KvLayers& mass,
                     const KvLayers& pos, const KvLayers& mass_out,
                     const KvLayers& pos_out, int keep, int recent, int limit,
                     int reach, void* ws, hipStream_t stream) {
    check_pages(kv, 0, reach);
    const int64_t rows = (int64_t)layers * kv.slots * kv.kv_heads;
    if (layers < 1 || rows >= 1 << 22)
        throw std::runtime_error("evict: 1 to 2^22 - 1 rows (layers x "
                                 "sequences x kv heads)");
    if (keep < 1 || recent < 0 || limit < keep)
        throw std::runtime_error("evict: keep >= 1, recent >= 0 and "
                                 "limit >= keep");
    const int most = std::max(0, std::min(keep, reach - keep));
    char* w = reinterpret_cast<char*>(ws);
    EvictArgs a{pages_of(kv), layer_stride, mass, pos, mass_out, pos_out,
                lens, next_pos, lens_out, layers, kv.slots, kv.kv_heads, keep,
                recent, limit, reach, most, nullptr, nullptr, nullptr};
    a.count = reinterpret_cast<int32_t*>(w);
    w += aligned(rows * 4);
    a.dst = reinterpret_cast<int32_t*>(w);
    w += aligned((size_t)rows * most * 4 + 4);
    a.src = reinterpret_cast<int32_t*>(w);
    const dim3 grid((uint32_t)rows), block(1024);
    if (reach <= 8 * 256)
        hipLaunchKernelGGL((k_kv_evict_select<256, 8>), grid, dim3(256), 0,
                           stream, a);
    else if (reach <= 8 * 1024)
        hipLaunchKernelGGL((k_kv_evict_select<1024, 8>), grid, block, 0,
                           stream, a);
    else if (reach <= 32 * 1024)
        hipLaunchKernelGGL((k_kv_evict_select<1024, 32>), grid, block, 0,
                           stream, a);
    else
        hipLaunchKernelGGL((k_kv_evict_select<1024, 0>), grid, block, 0,
                           stream, a);
    hipLaunchKernelGGL(k_kv_evict_move,
                       dim3((uint32_t)rows,
                            std::min(65535, std::max(1, (most + 63) / 64))),
                       dim3(256), 0, stream, a, kv.dim);
    check_launch();
}

}  // namespace cla
