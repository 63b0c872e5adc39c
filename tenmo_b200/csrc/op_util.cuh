// Shared by the transformer operators (layer norm, attention, linear cross-entropy).
#pragma once
#include "common.cuh"

// Makes the context's device current for the length of an entry point and puts the caller's back.
struct TenmoDeviceGuard {
    int before = -1;
    explicit TenmoDeviceGuard(const tenmo_ctx* ctx) {
        int now = -1;
        if (cudaGetDevice(&now) == cudaSuccess && now != ctx->device && cudaSetDevice(ctx->device) == cudaSuccess) before = now;
    }
    ~TenmoDeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
    TenmoDeviceGuard(const TenmoDeviceGuard&) = delete;
    TenmoDeviceGuard& operator=(const TenmoDeviceGuard&) = delete;
};

// A second workspace block, apart from the one of tenmo_workspace: these operators call the library's GEMMs while they
// hold intermediate results.  Grown on demand; a call that is being captured takes a block that has been used at its size before (else it is
// refused) and keeps it for its graph, so that a replay never meets a call outside of graphs.
int tenmo_op_workspace(tenmo_ctx* ctx, size_t bytes, void** out);
void tenmo_op_done(tenmo_ctx* ctx);

// Held by an entry point for its length: the context's device is current, and at the end it is noted how far the workspace is used.
struct TenmoOpCall {
    tenmo_ctx* const ctx;
    TenmoDeviceGuard device;
    explicit TenmoOpCall(tenmo_ctx* c) : ctx(c), device(c) {}
    ~TenmoOpCall() { tenmo_op_done(ctx); }
};
