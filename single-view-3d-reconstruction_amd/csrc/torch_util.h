// What the operator registrations share (torch_ops.cpp, torch_train_ops.cpp): status checks, device and stream of
// a call, dispatcher handles.
#pragma once
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "sv3d_hip.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using IntList = at::IntArrayRef;

// ---- small helpers ---------------------------------------------------------------------------
void check_status(int st, const char *what)
{
    TORCH_CHECK(st == SV3D_OK, what, " failed: ", sv3d_strerror(st), " (status ", st, ")");
}

struct Launch {
    c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
    void *stream;
    explicit Launch(const Tensor &t) : guard(t.device())
    {
        stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
    }
};

void same_device(const Tensor &ref, const Tensor &t, const char *name)
{
    // a tensor on the host or on another GPU would reach the kernels as a foreign pointer
    TORCH_CHECK(t.device() == ref.device(), name, " is on ", t.device(), ", expected ", ref.device());
}

template <class Sig>
c10::TypedOperatorHandle<Sig> find_op(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

Tensor cast_like(const Tensor &g, at::ScalarType t) { return g.scalar_type() == t ? g : g.to(t); }

}  // namespace
