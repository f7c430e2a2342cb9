// The nodes and functions of tannic_hip_functions.hpp for a cache in pages and the attention, over the stand-in of the front end (frontend_standin.hpp) and through adapter.cpp.
//     adapter_attention inputs outputs    float32 operands from a file, one after the other; what comes of them into another
// Compiled with RECORD the four entry points of the C ABI are replaced by functions that write down what they were handed, and nothing needs a device.
#include <cstdio>
#include <cstdlib>
#include <fstream>

#include "tannic_hip_functions.hpp"

using namespace tannic;

#ifdef RECORD
extern "C" {
// (memory and streams as well: an address is as many as there were before it)
void* tannic_hip_allocate(const tannic_device_t*, size_t) {
    static uintptr_t last = 0;
    return reinterpret_cast<void*>(++last);
}
void* tannic_hip_deallocate(const tannic_device_t*, void*) { return nullptr; }
int tannic_hip_copy_from_host(const tannic_device_t*, const void*, void*, size_t) { return TANNIC_SUCCESS; }
int tannic_hip_copy_device_to_host(const tannic_device_t*, const void*, void*, size_t) { return TANNIC_SUCCESS; }
tannic_stream_t tannic_hip_pop_stream(const tannic_device_t*) { return {77}; }
void tannic_hip_put_stream(const tannic_device_t*, tannic_stream_t) {}
static int answer = TANNIC_SUCCESS;
static int number(const tannic_tensor_t* t) { return t ? static_cast<int>(reinterpret_cast<uintptr_t>(t->address)) : 0; }
int tannic_hip_append_pages(const tannic_tensor_t* k, const tannic_tensor_t* v, const tannic_tensor_t* table, const tannic_tensor_t* starts, const tannic_tensor_t* context,
                            const tannic_tensor_t* cos, const tannic_tensor_t* sin, const tannic_tensor_t* q, tannic_tensor_t* keys, tannic_tensor_t* values, tannic_tensor_t* turned,
                            tannic_stream_t stream) {
    std::printf("append_pages %d %d %d %d %d %d %d %d %d %d %d stream %d\n", number(k), number(v), number(table), number(starts), number(context), number(cos), number(sin), number(q),
                number(keys), number(values), number(turned), static_cast<int>(stream.address));
    return answer;
}
int tannic_hip_attend_pages(const tannic_tensor_t* q, const tannic_tensor_t* keys, const tannic_tensor_t* values, const tannic_tensor_t* table, const tannic_tensor_t* starts,
                            const tannic_tensor_t* context, tannic_tensor_t* dst, tannic_stream_t stream, float scale) {
    std::printf("attend_pages %d %d %d %d %d %d %d stream %d scale %g\n", number(q), number(keys), number(values), number(table), number(starts), number(context), number(dst),
                static_cast<int>(stream.address), scale);
    return answer;
}
int tannic_hip_copy_pages(tannic_tensor_t* pool, tannic_stream_t stream, const int32_t* sources, const int32_t* targets, size_t count) {
    std::printf("copy_pages %d stream %d", number(pool), static_cast<int>(stream.address));
    for (size_t i = 0; i < count; ++i) std::printf(" %d>%d", sources[i], targets[i]);
    std::printf("\n");
    return answer;
}
int tannic_hip_attend(const tannic_tensor_t* q, const tannic_tensor_t* k, const tannic_tensor_t* v, const tannic_tensor_t* lengths, tannic_tensor_t* dst, tannic_stream_t stream,
                      float scale) {
    std::printf("attend %d %d %d %d %d stream %d scale %g\n", number(q), number(k), number(v), number(lengths), number(dst), static_cast<int>(stream.address), scale);
    return answer;
}
}
#endif

static Tensor on_device(type dtype, Shape const& shape, const void* values) {
    Tensor t(dtype, shape);
    t.initialize(Device{});
    device_t device{0};
    if (tannic_hip_copy_from_host(&device, values, get_tensor(t.id())->address, t.bytes()) != TANNIC_SUCCESS) std::exit(2);
    return t;
}

template <class Call> static void throws(const char* what, Call&& call) {
    try {
        call();
        std::printf("%s: nothing thrown\n", what);
    } catch (Exception const& e) {
        std::printf("%s: %s\n", what, e.what());
    }
}

int main(int, char** argument) {
    std::ifstream inputs(argument[1], std::ios::binary);
    auto given = [&](Shape const& shape) {
        Tensor described(float32, shape);
        std::vector<char> values(described.bytes());
        inputs.read(values.data(), static_cast<std::streamsize>(values.size()));
        return on_device(float32, shape, values.data());
    };
    auto numbers = [&](std::vector<int32_t> const& values, Shape const& shape) { return on_device(int32, shape, values.data()); };
    std::ofstream outputs(argument[2], std::ios::binary);
    auto put = [&](Tensor const& t) {
        device_t device{0};
        std::vector<char> values(t.bytes());
        if (tannic_hip_copy_device_to_host(&device, get_tensor(t.id())->address, values.data(), values.size()) != TANNIC_SUCCESS) std::exit(3);
        outputs.write(values.data(), static_cast<std::streamsize>(values.size()));
    };
    const Context context{};

    // two sequences of 9 states, 3 tokens, 4 / 2 heads of 16
    Tensor q = given({2, 3, 4, 16}), k = given({2, 9, 2, 16}), v = given({2, 9, 2, 16}), lengths = numbers({9, 4}, {2});
    put(attend(q, k, v, 0.25f).forward(context));
    put(attend(q, k, v, lengths, -0.5f).forward(context));

    // a cache of 6 pages of 4 tokens; 3 and 2 new tokens behind 2 and 4
    Tensor keys = given({6, 2, 4, 16}), values = given({6, 2, 4, 16}), new_k = given({5, 2, 16}), new_v = given({5, 2, 16}), new_q = given({5, 4, 16}), cosines = given({8, 8}),
           sines = given({8, 8});
    Tensor table = numbers({1, 3, 0, 4}, {2, 2}), starts = numbers({0, 3, 5}, {3}), before = numbers({2, 4}, {2});
    append_pages(new_k, new_v, keys, values, table, starts, before);
    put(keys), put(values);
    put(append_pages(new_k, new_v, keys, values, table, starts, before, cosines, sines, new_q));
    put(keys), put(values);
    put(attend_pages(new_q, keys, values, table, starts, before, 0.125f).forward(context));
    copy_pages(keys, {1, 5}, {5, 2});
    put(keys);

#ifdef RECORD
    Tensor on_host(float32, {2, 3, 4, 16});
    on_host.initialize(Host{});
    throws("host", [&] { attend(on_host, k, v, 1.0f).forward(context); });
    throws("mixed", [&] { attend_pages(q, keys, values, table, on_host, before, 1.0f).forward(context); });
    throws("lists", [&] { copy_pages(keys, {1}, {2, 3}); });
    answer = TANNIC_UNSUPPORTED_DTYPE;
    throws("types", [&] { attend(q, k, v, 1.0f).forward(context); });
    answer = TANNIC_ERROR;
    throws("refused", [&] { append_pages(new_k, new_v, keys, values, table, starts, before); });
#endif
    return 0;
}
