// What the host sources of libgemma_hip share: the handle registry, the
// entry checks and the op-level helpers of a context (defined in model.cpp).
#pragma once

#include "common.h"

namespace gh {

using Lock = std::lock_guard<std::recursive_mutex>;

// Handle registry (see the notes on lifetimes and locking in model.cpp).
enum HandleKind { HK_CTX = 1, HK_MODEL, HK_KV, HK_Q4, HK_KV8 };
void handle_add(const void* h, int kind);
bool handle_live(const void* h, int kind);
// Unregisters an open handle of `kind`; false if it is not one.
bool handle_take(const void* h, int kind);
int dead_handle(const char* fn, int kind);

// Entry points taking a context handle: it must be open.
int ctx_bind(gh_ctx* ctx);
// Entry points taking a model / cache / tensor handle (checked open by the
// caller): its context is alive, released or not.
int dev_bind(gh_ctx* ctx);

// True when a released context has no open model, Q4_0 tensor or 8-bit cache
// left; the caller that sees this (once: `dying` is set, context mutex held)
// frees it with ctx_free after letting the mutex go.
bool ctx_dead(gh_ctx* ctx);
// Frees a context that ctx_dead selected.  No other thread holds a handle
// made from it, so nothing else can be waiting on its mutex.
void ctx_free(gh_ctx* ctx);

// Op-level calls are synchronous, except while the context stream is being
// captured (gh_capture_begin): then they only enqueue.
int op_sync(gh_ctx* ctx);
// Per-context device scratch for op-level temporaries; grows outside capture.
int ctx_scratch(gh_ctx* ctx, size_t bytes, void** out);

}  // namespace gh

#define GH_LIVE(h, kind)                                                  \
    do {                                                                  \
        if (!(h)) return set_error(GH_ERR_INVALID, "%s: null handle", __func__); \
        if (!handle_live((h), (kind))) return dead_handle(__func__, (kind)); \
    } while (0)

#define OP_ENTER(ctx)             \
    GH_CHECK(ctx_bind(ctx));      \
    Lock lk((ctx)->mu)
