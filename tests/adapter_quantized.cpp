// The nodes and functions of tannic_hip_functions.hpp for rows in 8-bit integers and their product, over the stand-in of the front end (frontend_standin.hpp) and through adapter.cpp.
//     adapter_quantized inputs outputs    float32 operands from a file, one after the other; what comes of them into another
// Compiled with RECORD the entry points of the C ABI are replaced by functions that write down what they were handed, and nothing needs a device.
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
static void record(const char* name, std::initializer_list<const tannic_tensor_t*> tensors, tannic_stream_t stream) {
    std::printf("%s", name);
    for (const tannic_tensor_t* t : tensors) {
        if (!t) {
            std::printf(" -");
            continue;
        }
        std::printf(" %d:%d[", static_cast<int>(reinterpret_cast<uintptr_t>(t->address)), static_cast<int>(t->dtype));
        for (int d = 0; d < t->rank; ++d) std::printf(d ? ",%d" : "%d", static_cast<int>(t->shape.sizes[d]));
        std::printf("]");
    }
    std::printf(" stream %d", static_cast<int>(stream.address));
}
int tannic_hip_quantize(const tannic_tensor_t* x, tannic_tensor_t* dst, tannic_tensor_t* scales, tannic_stream_t stream) {
    record("quantize", {x, dst, scales}, stream);
    std::printf("\n");
    return answer;
}
int tannic_hip_swiglu_quantize(const tannic_tensor_t* gate, const tannic_tensor_t* up, tannic_tensor_t* dst, tannic_tensor_t* scales, tannic_stream_t stream) {
    record("swiglu_quantize", {gate, up, dst, scales}, stream);
    std::printf("\n");
    return answer;
}
int tannic_hip_add_rms_norm(const tannic_tensor_t* x, const tannic_tensor_t* residual, const tannic_tensor_t* gain, tannic_tensor_t* total, tannic_tensor_t* dst, tannic_tensor_t* scales,
                            tannic_stream_t stream, float eps) {
    record("add_rms_norm", {x, residual, gain, total, dst, scales}, stream);
    std::printf(" eps %g\n", eps);
    return answer;
}
int tannic_hip_dequantize(const tannic_tensor_t* values, const tannic_tensor_t* scales, tannic_tensor_t* dst, tannic_stream_t stream) {
    record("dequantize", {values, scales, dst}, stream);
    std::printf("\n");
    return answer;
}
int tannic_hip_gemm_quantized(const tannic_tensor_t* a, const tannic_tensor_t* a_scales, const tannic_tensor_t* b, const tannic_tensor_t* b_scales, tannic_tensor_t* dst,
                              tannic_stream_t stream) {
    record("gemm_quantized", {a, a_scales, b, b_scales, dst}, stream);
    std::printf("\n");
    return answer;
}
}
#endif

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
        Tensor t(float32, shape);
        t.initialize(Device{});
        std::vector<char> values(t.bytes());
        inputs.read(values.data(), static_cast<std::streamsize>(values.size()));
        device_t device{0};
        if (tannic_hip_copy_from_host(&device, values.data(), get_tensor(t.id())->address, values.size()) != TANNIC_SUCCESS) std::exit(2);
        return t;
    };
    std::ofstream outputs(argument[2], std::ios::binary);
    auto put = [&](Tensor const& t) {
        device_t device{0};
        std::vector<char> values(t.bytes());
        if (tannic_hip_copy_device_to_host(&device, get_tensor(t.id())->address, values.data(), values.size()) != TANNIC_SUCCESS) std::exit(3);
        outputs.write(values.data(), static_cast<std::streamsize>(values.size()));
    };
    const Context context{};

    // two sequences of 3 tokens of 40 elements, a square matrix of weights
    Tensor x = given({2, 3, 40}), residual = given({2, 3, 40}), gain = given({40}), w = given({40, 40});
    auto q = quantize(x), weights = quantize(w);
    put(q.scales);
    put(dequantize(q.values, q.scales, float32).forward(context));
    put(matmul_quantized(q.values, q.scales, weights.values, weights.scales, float32).forward(context));
    auto gated = swiglu_quantized(x, residual);
    put(dequantize(gated.values, gated.scales, float32).forward(context));
    auto alone = rms_norm_quantized(x, gain, 0.5f);
    put(dequantize(alone.values, alone.scales, float32).forward(context));
    auto [normed, total] = add_rms_norm(x, residual, gain, 0.25f);
    put(normed), put(total);
    auto [in_8_bits, sum] = add_rms_norm_quantized(x, residual, gain, 0.25f);
    put(dequantize(in_8_bits.values, in_8_bits.scales, float32).forward(context)), put(sum);

#ifdef RECORD
    Tensor on_host(float32, {2, 3, 40}), scalar(float32, {});
    on_host.initialize(Host{});
    scalar.initialize(Device{});
    throws("host", [&] { quantize(on_host); });
    throws("mixed", [&] { swiglu_quantized(x, on_host); });
    throws("scalar", [&] { quantize(scalar); });
    throws("ranks", [&] { matmul_quantized(gain, gain, w, gain, float32).forward(context); });
    throws("inner", [&] { matmul_quantized(x, gain, residual, gain, float32).forward(context); });
    answer = TANNIC_UNSUPPORTED_DTYPE;
    throws("types", [&] { add_rms_norm(x, residual, gain, 1.0f); });
    answer = TANNIC_ERROR;
    throws("refused", [&] { dequantize(x, residual, float32).forward(context); });
#endif
    return 0;
}
