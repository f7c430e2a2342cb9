// What tannic_hip_functions.hpp and adapter.cpp need of Tannic's front end, in the smallest form that compiles: for checking the expression nodes where the front end's sources
// are not at hand.  The names are the front end's; the rest is made up: the runtime structs are the C ABI's, a tensor is a contiguous float32 or int32 block on device 0 (or on the
// host, without memory), an expression holds copies of its operands.  Every header of the front end that those two files include is this one.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <memory>
#include <stdexcept>
#include <string>
#include <tuple>
#include <type_traits>
#include <utility>
#include <variant>
#include <vector>

#include "tannic_hip.h"

namespace tannic {

using tensor_t = ::tannic_tensor_t;
using scalar_t = ::tannic_scalar_t;
using stream_t = ::tannic_stream_t;
using device_t = ::tannic_device_t;
enum type { int32 = TANNIC_INT32, float16 = TANNIC_FLOAT16, float32 = TANNIC_FLOAT32, complex128 = TANNIC_COMPLEX128, TYPES = TANNIC_TYPES };
enum status { SUCCESS, ERROR, UNSUPPORTED_DTYPE, NULL_ALLOCATOR, INCOMPATIBLE_DEVICES };
enum layout { SINGLETON, CONTIGUOUS, STRIDED };
enum environment { HOST, DEVICE };
enum host { PAGEABLE = 1, PINNED };

struct Exception : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Context {};
struct Host {};
struct Device {
    int id() const { return 0; }
};
using Environment = std::variant<Host, Device>;

class Shape {
public:
    constexpr Shape() = default;
    constexpr Shape(std::initializer_list<size_t> sizes) {
        for (size_t size : sizes) expand(size);
    }
    constexpr size_t rank() const { return rank_; }
    constexpr size_t operator[](size_t dim) const { return sizes_[dim]; }
    constexpr void expand(size_t size) { sizes_[rank_++] = size; }

private:
    size_t sizes_[TANNIC_DIMENSIONS] = {}, rank_ = 0;
};
struct Strides {
    constexpr Strides() = default;
    constexpr explicit Strides(Shape const&) {}
};

// Memory and description of a tensor; tensors that are copies share it.
struct Node {
    tensor_t tensor{};
    Environment environment = Host{};
    bool initialized = false;
    ~Node() {
        device_t device{0};
        if (tensor.address && std::holds_alternative<Device>(environment)) tannic_hip_deallocate(&device, tensor.address);
    }
};
using uuid = Node*;
inline tensor_t* get_tensor(uuid id) { return &id->tensor; }
inline stream_t pop_stream(const device_t* device) { return tannic_hip_pop_stream(device); }
inline void put_stream(const device_t* device, stream_t stream) { tannic_hip_put_stream(device, stream); }

class Tensor {
public:
    Tensor(type dtype, Shape const& shape) : shape_(shape), node_(std::make_shared<Node>()) {
        tensor_t& t = node_->tensor;
        t.rank = static_cast<uint8_t>(shape.rank());
        t.dtype = static_cast<tannic_type>(dtype);
        t.layout = TANNIC_CONTIGUOUS;
        t.size = 1;
        for (size_t dim = shape.rank(); dim-- > 0;) {
            t.shape.sizes[dim] = shape[dim];
            t.strides.sizes[dim] = static_cast<int64_t>(t.size);
            t.size *= shape[dim];
        }
    }
    type dtype() const { return static_cast<type>(node_->tensor.dtype); }
    Shape const& shape() const { return shape_; }
    uuid id() const { return node_.get(); }
    Environment const& environment() const { return node_->environment; }
    bool is_initialized() const { return node_->initialized; }
    void initialize(Environment const& environment) {
        node_->environment = environment;
        node_->initialized = true;
        if (!std::holds_alternative<Device>(environment)) return;
        device_t device{0};
        node_->tensor.address = tannic_hip_allocate(&device, bytes());
        node_->tensor.environment.kind = TANNIC_DEVICE;
        node_->tensor.environment.resource.device.id = 0;
    }
    size_t bytes() const { return node_->tensor.size * 4; }
    Tensor const& forward(Context const&) const { return *this; }

private:
    Shape shape_;
    std::shared_ptr<Node> node_;
};

template <class T> concept Composable = true;
template <class T> struct Trait {
    using Reference = std::remove_cvref_t<T>;
};

namespace operation {
constexpr type promote(type first, type second) { return first < second ? second : first; }
constexpr Shape broadcast(Shape const& first, Shape const&) { return first; }
}  // namespace operation
namespace indexing {
constexpr int normalize(int axis, size_t rank) { return axis < 0 ? axis + static_cast<int>(rank) : axis; }
}  // namespace indexing
namespace expression {
template <class Operation, class... Operands> struct Expression {
    Operation operation;
    std::tuple<typename Trait<Operands>::Reference...> operands;
    Expression(Operation op, typename Trait<Operands>::Reference... each) : operation(op), operands(each...) {}
};
template <class Operation, class First, class Second> struct Binary {};
template <class Operation, class Source> struct Reduction {};
}  // namespace expression

}  // namespace tannic
