// What the two addons over libbrik.so share: argument conversions, errors, and the context handle that both take.
#pragma once
#include <node_api.h>

#include <cstdint>
#include <cstring>
#include <string>

#include "brik.h"

namespace {

#define NAPI_CALL(env, call)                                                  \
    do {                                                                      \
        if ((call) != napi_ok) {                                              \
            napi_throw_error((env), "BRIK_NAPI", "N-API call failed: " #call); \
            return nullptr;                                                   \
        }                                                                     \
    } while (0)
// the same in a function returning bool
#define NAPI_CALL_B(env, call)                                                \
    do {                                                                      \
        if ((call) != napi_ok) {                                              \
            napi_throw_error((env), "BRIK_NAPI", "N-API call failed: " #call); \
            return false;                                                     \
        }                                                                     \
    } while (0)

inline const char* code_name(int rc)
{
    switch (rc) {
    case BRIK_EINVAL: return "BRIK_EINVAL";
    case BRIK_EALIGN: return "BRIK_EALIGN";
    case BRIK_EHIP: return "BRIK_EHIP";
    case BRIK_ENOMEM: return "BRIK_ENOMEM";
    case BRIK_ENODEV: return "BRIK_ENODEV";
    case BRIK_EMODULE: return "BRIK_EMODULE";
    default: return "BRIK_ERROR";
    }
}

// Throw for rc < 0. Returns true if an exception is pending.
inline bool check(napi_env env, brik_ctx* ctx, int rc)
{
    if (rc == BRIK_OK) return false;
    std::string msg = std::string(code_name(rc)) + ": " + (ctx ? brik_last_error(ctx) : brik_strerror(rc));
    napi_throw_error(env, code_name(rc), msg.c_str());
    return true;
}

struct Args {
    napi_value v[16];
    size_t n = 16;
};

inline bool get_args(napi_env env, napi_callback_info info, Args& a, size_t need)
{
    if (napi_get_cb_info(env, info, &a.n, a.v, nullptr, nullptr) != napi_ok) return false;
    if (a.n < need) {
        napi_throw_type_error(env, "BRIK_EINVAL", "too few arguments");
        return false;
    }
    return true;
}

inline bool get_i32(napi_env env, napi_value v, int32_t* out)
{
    if (napi_get_value_int32(env, v, out) != napi_ok) {
        napi_throw_type_error(env, "BRIK_EINVAL", "expected a number");
        return false;
    }
    return true;
}

inline bool get_f32(napi_env env, napi_value v, float* out)
{
    double d;
    if (napi_get_value_double(env, v, &d) != napi_ok) {
        napi_throw_type_error(env, "BRIK_EINVAL", "expected a number");
        return false;
    }
    *out = (float)d;
    return true;
}

// An element count: a non-negative integral Number (exact below 2^53).
inline bool get_size(napi_env env, napi_value v, size_t* out)
{
    double d;
    if (napi_get_value_double(env, v, &d) != napi_ok || !(d >= 0) || d != (double)(uint64_t)d || d > 9007199254740992.0) {
        napi_throw_type_error(env, "BRIK_EINVAL", "expected a non-negative integer count");
        return false;
    }
    *out = (size_t)d;
    return true;
}

// A device pointer: BigInt address, null/undefined (-> nullptr), or an object with a BigInt `ptr`.
inline bool get_ptr(napi_env env, napi_value v, void** out)
{
    napi_valuetype t;
    napi_typeof(env, v, &t);
    if (t == napi_null || t == napi_undefined) { *out = nullptr; return true; }
    if (t == napi_object) {
        napi_value p;
        if (napi_get_named_property(env, v, "ptr", &p) != napi_ok) return false;
        v = p;
        napi_typeof(env, v, &t);
    }
    if (t != napi_bigint) {
        napi_throw_type_error(env, "BRIK_EINVAL", "expected a device pointer (BigInt or {ptr: BigInt})");
        return false;
    }
    uint64_t u;
    bool lossless;
    if (napi_get_value_bigint_uint64(env, v, &u, &lossless) != napi_ok) return false;
    *out = reinterpret_cast<void*>(static_cast<uintptr_t>(u));
    return true;
}

// A context as JS holds it: the library context, and the count of the JS-side objects that keep it
// alive (the context handle itself, device buffers, plans). It is destroyed when the last one is
// finalized, so a buffer collected after its context never frees into a destroyed context.
struct CtxBox {
    brik_ctx* ctx;
    long refs;
    long live_buffers;   // device buffers allocated through allocBuffer and not yet freed
};

inline void box_release(CtxBox* b)
{
    if (--b->refs == 0) {
        brik_destroy(b->ctx);
        delete b;
    }
}

inline bool get_box(napi_env env, napi_value v, CtxBox** out)
{
    void* p = nullptr;
    if (napi_get_value_external(env, v, &p) != napi_ok || !p) {
        napi_throw_type_error(env, "BRIK_EINVAL", "expected a brik context");
        return false;
    }
    *out = static_cast<CtxBox*>(p);
    return true;
}

inline bool get_ctx(napi_env env, napi_value v, brik_ctx** out)
{
    CtxBox* b;
    if (!get_box(env, v, &b)) return false;
    *out = b->ctx;
    return true;
}

inline napi_value make_ptr(napi_env env, void* p)
{
    napi_value r;
    napi_create_bigint_uint64(env, static_cast<uint64_t>(reinterpret_cast<uintptr_t>(p)), &r);
    return r;
}

inline napi_value undefined(napi_env env)
{
    napi_value u;
    napi_get_undefined(env, &u);
    return u;
}

// An integer of the range of its C type: anything else is refused, not cut off.
inline bool get_whole(napi_env env, napi_value v, const std::string& what, double most, double* out)
{
    if (napi_get_value_double(env, v, out) != napi_ok || !(*out >= -most && *out <= most) || *out != (double)(int64_t)*out) {
        napi_throw_type_error(env, "BRIK_EINVAL", ("expected an integer: " + what).c_str());
        return false;
    }
    return true;
}

// Parse (ctx, p0 .. p{np-1}, i0 .. i{ni-1}). whole: numbers that are no 32-bit integers are refused, else converted as by ToInt32.
inline bool parse(napi_env env, napi_callback_info info, brik_ctx** ctx, void** p, int np, int32_t* iv, int ni, bool whole = false)
{
    Args a;
    if (!get_args(env, info, a, (size_t)(1 + np + ni))) return false;
    if (!get_ctx(env, a.v[0], ctx)) return false;
    for (int i = 0; i < np; ++i)
        if (!get_ptr(env, a.v[1 + i], &p[i])) return false;
    for (int i = 0; i < ni; ++i) {
        double d = 0;
        if (!whole) {
            if (!get_i32(env, a.v[1 + np + i], &iv[i])) return false;
        } else if (!get_whole(env, a.v[1 + np + i], "argument " + std::to_string(np + i + 1), 2147483647.0, &d)) return false;
        else iv[i] = (int32_t)d;
    }
    return true;
}

// A named property of `o`; absent, undefined and null leave `*has` false.
inline bool get_field(napi_env env, napi_value o, const char* name, napi_value* out, bool* has)
{
    napi_valuetype t;
    NAPI_CALL_B(env, napi_typeof(env, o, &t));
    if (t != napi_object) {
        napi_throw_type_error(env, "BRIK_EINVAL", "expected an object");
        return false;
    }
    NAPI_CALL_B(env, napi_get_named_property(env, o, name, out));
    NAPI_CALL_B(env, napi_typeof(env, *out, &t));
    *has = t != napi_undefined && t != napi_null;
    return true;
}

// Optional fields: as they are where absent.
inline bool opt_ptr(napi_env env, napi_value o, const char* name, void** out)
{
    napi_value f;
    bool has;
    return get_field(env, o, name, &f, &has) && (!has || get_ptr(env, f, out));
}
inline bool opt_f32(napi_env env, napi_value o, const char* name, float* out)
{
    napi_value f;
    bool has;
    return get_field(env, o, name, &f, &has) && (!has || get_f32(env, f, out));
}
inline bool opt_int(napi_env env, napi_value o, const char* name, double most, double* out)
{
    napi_value f;
    bool has;
    return get_field(env, o, name, &f, &has) && (!has || get_whole(env, f, name, most, out));
}
inline bool opt_i32(napi_env env, napi_value o, const char* name, int32_t* out)
{
    double d = *out;
    if (!opt_int(env, o, name, 2147483647.0, &d)) return false;
    *out = (int32_t)d;
    return true;
}
inline bool opt_i64(napi_env env, napi_value o, const char* name, int64_t* out)
{
    double d = (double)*out;
    if (!opt_int(env, o, name, 9007199254740991.0, &d)) return false;
    *out = (int64_t)d;
    return true;
}

}  // namespace
