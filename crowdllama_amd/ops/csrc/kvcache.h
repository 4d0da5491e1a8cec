// The paged KV cache's operators: append, attend, observe and evict
// (kvcache.hip). Host-side launch interface, shared by the engine and by the
// Python bindings.
//
// A pool holds pages [page][layer][kv head][K, V][place in page][D]; place p
// of sequence b lies in row p % page of page table[b][p / page]. Each (layer,
// sequence, kv head) has `mass` (f32: the attention weight that each place
// has received) and `pos` (i32: the position of the token in each place).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace cla {

// Element types of q/k/v and of the pool.
enum class KVT : int32_t { F32 = 0, F16 = 1, BF16 = 2 };

// One layer's pages of all sequences.
struct KvPages {
    void* pool = nullptr;        // the layer's first page
    int64_t page_stride = 0;     // elements from page to page
    int32_t pages = 0;           // pages in the pool
    const int32_t* table = nullptr;   // [slots][max_pages]
    int64_t table_stride = 0;
    int32_t max_pages = 0;
    int32_t page = 0;            // places in a page (a multiple of 16)
    int32_t slots = 0;
    int32_t kv_heads = 0;
    int32_t dim = 0;             // 64, 96 or 128
    KVT type = KVT::BF16;
};

// A tensor [slots][kv heads][places] of 4-byte values (mass, pos).
struct KvRows {
    void* data = nullptr;
    int64_t slot_stride = 0, head_stride = 0;
};

// A tensor [rows][heads][D].
struct KvHeads {
    void* data = nullptr;
    int64_t row_stride = 0, head_stride = 0;
};

// Pages are only followed where the table and the pool have them: -1 for a
// place past the table's end and for a page number outside the pool. Such
// places have no weight, and no keys and values are stored there.
__host__ __device__ inline int32_t kv_page_of(const int32_t* row,
                                              int64_t index,
                                              int32_t max_pages,
                                              int32_t pages) {
    if (index < 0 || index >= max_pages) return -1;
    const int32_t p = row[index];
    return (p < 0 || p >= pages) ? -1 : p;
}

// A length as the operators use it: never negative, never past the places
// that the table (and the mass, where there is one) reaches.
__host__ __device__ inline int32_t kv_clamp_len(int32_t len, int32_t reach) {
    return len < 0 ? 0 : (len > reach ? reach : len);
}

// Order of eviction as one unsigned key, larger keys first: tokens of late
// (`recent`) before all others, the others by mass. NaN comes last, -0 is 0.
__host__ __device__ inline uint32_t kv_rank_key(float mass, bool recent) {
    if (recent) return 0xFFFFFFFFu;
    union { float f; uint32_t u; } v;
    v.f = mass + 0.0f;
    if (v.f != v.f) return 0u;
    const uint32_t k = (v.u & 0x80000000u) ? ~v.u : (v.u | 0x80000000u);
    return k == 0xFFFFFFFFu ? 0xFFFFFFFEu : k;
}

// Rotate q and k (adjacent pairs, inv_freq [D/2], or not at all where that
// is null) and store k and v of `rows` new tokens at places lens[b]... of
// their sequences; starts [slots + 1] says which rows are whose (null: row b
// belongs to sequence b). q, mass and pos may be null.
void launch_kv_append(const KvPages& kv, const KvHeads& k, const KvHeads& v,
                      const KvHeads& q, const KvHeads& q_out, int q_heads,
                      KVT type, int rows, const int32_t* starts,
                      const int32_t* lens, const int32_t* next_pos,
                      const float* inv_freq, const KvRows& mass,
                      const KvRows& pos, int reach, hipStream_t stream);

// A decode step's places: step[b] is where slot b's next token goes, -1 for a
// slot that takes no part; len counts the tokens of those that do.
void launch_kv_step(int32_t* len, int32_t* step, const uint8_t* active,
                    int slots, hipStream_t stream);

// One new token's attention over each sequence's first lens[b] places;
// mass (may be null) gets each place's weight added, summed over the query
// heads of the kv head. `add` is added to each length.
size_t kv_attend_workspace(const KvPages& kv, int q_heads, int reach,
                           bool mass);
void launch_kv_attend(const KvPages& kv, const KvHeads& q, const KvHeads& out,
                      int q_heads, KVT type, const int32_t* lens, int add,
                      const KvRows& mass, int reach, float scale, void* ws,
                      hipStream_t stream);

// The weight that `rows` tokens at the ends of their sequences gave to each
// place they see, added to mass.
size_t kv_observe_workspace(const KvPages& kv, int q_heads, int rows,
                            int reach, KVT type);
void launch_kv_observe(const KvPages& kv, const KvHeads& q, int q_heads,
                       KVT type, int rows, const int32_t* starts,
                       const int32_t* lens, const KvRows& mass, int reach,
                       float scale, void* ws, hipStream_t stream);

// Keep `keep` places of each sequence that has more than `limit`, in all
// layers. mass, pos and lens are written to the *_out tensors, which may be
// the same ones. Places are ordered and moved whether they have a page or not;
// keys and values move where both places have one.
struct KvLayers {              // [layers][slots][kv heads][places]
    void* data = nullptr;
    int64_t layer_stride = 0, slot_stride = 0, head_stride = 0;
};
size_t kv_evict_workspace(const KvPages& kv, int layers, int keep, int reach);
void launch_kv_evict(const KvPages& kv, int layers, int64_t layer_stride,
                     const int32_t* lens, int32_t* lens_out,
                     const int32_t* next_pos, const KvLayers& mass,
                     const KvLayers& pos, const KvLayers& mass_out,
                     const KvLayers& pos_out, int keep, int recent, int limit,
                     int reach, void* ws, hipStream_t stream);

}  // namespace cla
