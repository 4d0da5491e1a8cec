// Python face of the paged cache's operators. crowdllama_amd/ops/kv.py checks
// the tensors and passes addresses, strides (in elements) and sizes.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <tuple>

#include "common.h"
#include "kvcache.h"

namespace py = pybind11;

namespace cla {

namespace {

// address, page stride, pages, table, table stride, max_pages, page, slots,
// kv heads, dim, type, device
using PagesArg = std::tuple<uintptr_t, int64_t, int32_t, uintptr_t, int64_t,
                            int32_t, int32_t, int32_t, int32_t, int32_t,
                            int32_t, int32_t>;
// address, row stride, head stride
using HeadsArg = std::tuple<uintptr_t, int64_t, int64_t>;
// address, layer stride, slot stride, head stride
using LayersArg = std::tuple<uintptr_t, int64_t, int64_t, int64_t>;

template <class T>
T* at(uintptr_t p) { return reinterpret_cast<T*>(p); }

KvPages pages(const PagesArg& a) {
    KvPages kv;
    kv.pool = at<void>(std::get<0>(a));
    kv.page_stride = std::get<1>(a);
    kv.pages = std::get<2>(a);
    kv.table = at<const int32_t>(std::get<3>(a));
    kv.table_stride = std::get<4>(a);
    kv.max_pages = std::get<5>(a);
    kv.page = std::get<6>(a);
    kv.slots = std::get<7>(a);
    kv.kv_heads = std::get<8>(a);
    kv.dim = std::get<9>(a);
    kv.type = static_cast<KVT>(std::get<10>(a));
    return kv;
}

KvHeads heads(const HeadsArg& a) {
    return {at<void>(std::get<0>(a)), std::get<1>(a), std::get<2>(a)};
}
KvRows rows(const HeadsArg& a) {
    return {at<void>(std::get<0>(a)), std::get<1>(a), std::get<2>(a)};
}
KvLayers layers(const LayersArg& a) {
    return {at<void>(std::get<0>(a)), std::get<1>(a), std::get<2>(a),
            std::get<3>(a)};
}
hipStream_t stream(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }

// Work is launched on the tensors' device, whatever the current one is.
struct OnDevice {
    int before = 0;
    bool other = false;
    explicit OnDevice(const PagesArg& a) {
        const int dev = std::get<11>(a);
        HIP_CHECK(hipGetDevice(&before));
        other = dev != before;
        if (other) HIP_CHECK(hipSetDevice(dev));
    }
    ~OnDevice() {
        if (other) (void)hipSetDevice(before);
    }
};

}  // namespace

void bind_kv(py::module_& m) {
    m.def("kv_append", [](const PagesArg& kv, const HeadsArg& k,
                          const HeadsArg& v, const HeadsArg& q,
                          const HeadsArg& q_out, int q_heads, int type,
                          int n, uintptr_t starts, uintptr_t lens,
                          uintptr_t next_pos, uintptr_t inv_freq,
                          const HeadsArg& mass, const HeadsArg& pos,
                          int reach, uintptr_t s) {
        OnDevice on(kv);
        launch_kv_append(pages(kv), heads(k), heads(v), heads(q),
                         heads(q_out), q_heads, static_cast<KVT>(type), n,
                         at<const int32_t>(starts), at<const int32_t>(lens),
                         at<const int32_t>(next_pos),
                         at<const float>(inv_freq), rows(mass), rows(pos),
                         reach, stream(s));
    });
    m.def("kv_attend_workspace", [](const PagesArg& kv, int q_heads,
                                    int reach, bool mass) {
        return kv_attend_workspace(pages(kv), q_heads, reach, mass);
    });
    m.def("kv_attend", [](const PagesArg& kv, const HeadsArg& q,
                          const HeadsArg& out, int q_heads, int type,
                          uintptr_t lens, const HeadsArg& mass, int reach,
                          float scale, uintptr_t ws, uintptr_t s) {
        OnDevice on(kv);
        launch_kv_attend(pages(kv), heads(q), heads(out), q_heads,
                         static_cast<KVT>(type), at<const int32_t>(lens), 0,
                         rows(mass), reach, scale, at<void>(ws), stream(s));
    });
    m.def("kv_observe_workspace", [](const PagesArg& kv, int q_heads, int n,
                                     int reach, int type) {
        return kv_observe_workspace(pages(kv), q_heads, n, reach,
                                    static_cast<KVT>(type));
    });
    m.def("kv_observe", [](const PagesArg& kv, const HeadsArg& q, int q_heads,
                           int type, int n, uintptr_t starts, uintptr_t lens,
                           const HeadsArg& mass, int reach, float scale,
                           uintptr_t ws, uintptr_t s) {
        OnDevice on(kv);
        launch_kv_observe(pages(kv), heads(q), q_heads,
                          static_cast<KVT>(type), n,
                          at<const int32_t>(starts), at<const int32_t>(lens),
                          rows(mass), reach, scale, at<void>(ws), stream(s));
    });
    m.def("kv_evict_workspace", [](const PagesArg& kv, int n_layers, int keep,
                                   int reach) {
        return kv_evict_workspace(pages(kv), n_layers, keep, reach);
    });
    m.def("kv_evict", [](const PagesArg& kv, int n_layers,
                         int64_t layer_stride, uintptr_t lens,
                         uintptr_t lens_out, uintptr_t next_pos,
                         const LayersArg& mass, const LayersArg& pos,
                         const LayersArg& mass_out, const LayersArg& pos_out,
                         int keep, int recent, int limit, int reach,
                         uintptr_t ws, uintptr_t s) {
        OnDevice on(kv);
        launch_kv_evict(pages(kv), n_layers, layer_stride,
                        at<const int32_t>(lens), at<int32_t>(lens_out),
                        at<const int32_t>(next_pos), layers(mass),
                        layers(pos), layers(mass_out), layers(pos_out), keep,
                        recent, limit, reach, at<void>(ws), stream(s));
    });

    // what the kernels decide from values on the device, for CPU tests
    m.def("test_kv_page_of", [](std::vector<int32_t> row, int64_t index,
                                int32_t pages) {
        return kv_page_of(row.data(), index, (int32_t)row.size(), pages);
    });
    m.def("test_kv_clamp_len", &kv_clamp_len);
    m.def("test_kv_rank_key", &kv_rank_key);
}

}  // namespace cla
