// brik_experts.node — Node N-API binding of libbrik.so's experts and 8-bit products, on contexts that brik.node made. An addon of
// its own: brik.node's surface stays what callers compare. Thin as that one: arguments converted, one brik_* call, its error thrown.
#include "brik_napi.h"

namespace {

// {logits, tokens, experts, k, ids, weights[, bias, logitStride, rowOff, src, slot, flags, scale]}
bool get_route(napi_env env, napi_value o, brik_moe_route_args* r)
{
    std::memset(r, 0, sizeof *r);
    r->scale = 1.f;
    void* p[7] = {};
    const char* const names[7] = {"logits", "bias", "ids", "weights", "rowOff", "src", "slot"};
    for (int i = 0; i < 7; ++i)
        if (!opt_ptr(env, o, names[i], &p[i])) return false;
    r->logits = (const float*)p[0];
    r->bias = (const float*)p[1];
    r->ids = (int32_t*)p[2];
    r->weights = (float*)p[3];
    r->row_off = (int32_t*)p[4];
    r->src = (int32_t*)p[5];
    r->slot = (int32_t*)p[6];
    return opt_i32(env, o, "tokens", &r->tokens) && opt_i32(env, o, "experts", &r->experts) && opt_i32(env, o, "k", &r->k) &&
           opt_i32(env, o, "flags", &r->flags) && opt_f32(env, o, "scale", &r->scale) && opt_i64(env, o, "logitStride", &r->logit_stride);
}

napi_value MoeRoute(napi_env env, napi_callback_info info)   // (ctx, route)
{
    Args a;
    brik_ctx* c;
    brik_moe_route_args r;
    if (!get_args(env, info, a, 2) || !get_ctx(env, a.v[0], &c) || !get_route(env, a.v[1], &r)) return nullptr;
    return check(env, c, brik_moe_route(c, &r)) ? nullptr : undefined(env);
}

napi_value MoeRouteGrad(napi_env env, napi_callback_info info)   // (ctx, route, dweights, dlogits)
{
    Args a;
    brik_ctx* c;
    brik_moe_route_args r;
    void *dw, *dl;
    if (!get_args(env, info, a, 4) || !get_ctx(env, a.v[0], &c) || !get_route(env, a.v[1], &r) || !get_ptr(env, a.v[2], &dw) ||
        !get_ptr(env, a.v[3], &dl))
        return nullptr;
    return check(env, c, brik_moe_route_grad(c, &r, (const float*)dw, (float*)dl)) ? nullptr : undefined(env);
}

napi_value MoeSort(napi_env env, napi_callback_info info)   // (ctx, ids, rowOff, src, slot, tokens, k, experts)
{
    brik_ctx* c; void* p[4]; int32_t i[3];
    if (!parse(env, info, &c, p, 4, i, 3, true)) return nullptr;
    if (check(env, c, brik_moe_sort(c, (const int32_t*)p[0], i[0], i[1], i[2], (int32_t*)p[1], (int32_t*)p[2], (int32_t*)p[3]))) return nullptr;
    return undefined(env);
}

napi_value MoeDispatch(napi_env env, napi_callback_info info)   // (ctx, x, slot, weights, xSorted, tokens, k, width)
{
    brik_ctx* c; void* p[4]; int32_t i[3];
    if (!parse(env, info, &c, p, 4, i, 3, true)) return nullptr;
    if (check(env, c, brik_moe_dispatch(c, (const float*)p[0], (const int32_t*)p[1], (const float*)p[2], (float*)p[3], i[0], i[1], i[2])))
        return nullptr;
    return undefined(env);
}

napi_value MoeCombine(napi_env env, napi_callback_info info)   // (ctx, ySorted, slot, weights, res, out, tokens, k, width)
{
    brik_ctx* c; void* p[5]; int32_t i[3];
    if (!parse(env, info, &c, p, 5, i, 3, true)) return nullptr;
    if (check(env, c, brik_moe_combine(c, (const float*)p[0], (const int32_t*)p[1], (const float*)p[2], (const float*)p[3], (float*)p[4], i[0], i[1],
                                       i[2])))
        return nullptr;
    return undefined(env);
}

napi_value MoeCombineGrad(napi_env env, napi_callback_info info)   // (ctx, dout, ySorted, slot, weights, dySorted, dweights, tokens, k, width)
{
    brik_ctx* c; void* p[6]; int32_t i[3];
    if (!parse(env, info, &c, p, 6, i, 3, true)) return nullptr;
    if (check(env, c, brik_moe_combine_grad(c, (const float*)p[0], (const float*)p[1], (const int32_t*)p[2], (const float*)p[3], (float*)p[4],
                                            (float*)p[5], i[0], i[1], i[2])))
        return nullptr;
    return undefined(env);
}

napi_value QuantizeI8(napi_env env, napi_callback_info info)   // (ctx, {x, codes, scales, M, K[, gate, flags, xStride, gateStride]})
{
    Args a;
    brik_ctx* c;
    if (!get_args(env, info, a, 2) || !get_ctx(env, a.v[0], &c)) return nullptr;
    void* p[4] = {};
    const char* const names[4] = {"x", "gate", "codes", "scales"};
    for (int i = 0; i < 4; ++i)
        if (!opt_ptr(env, a.v[1], names[i], &p[i])) return nullptr;
    int32_t M = 0, K = 0, flags = 0;
    int64_t xs = 0, gs = 0;
    if (!opt_i32(env, a.v[1], "M", &M) || !opt_i32(env, a.v[1], "K", &K) || !opt_i32(env, a.v[1], "flags", &flags) ||
        !opt_i64(env, a.v[1], "xStride", &xs) || !opt_i64(env, a.v[1], "gateStride", &gs))
        return nullptr;
    if (check(env, c, brik_quantize_i8(c, (const float*)p[0], xs, (const float*)p[1], gs, flags, (int8_t*)p[2], (float*)p[3], M, K))) return nullptr;
    return undefined(env);
}

napi_value MatmulI8(napi_env env, napi_callback_info info)   // (ctx, x, xScales, w, wScales, res, y, M, K, N)
{
    brik_ctx* c; void* p[6]; int32_t i[3];
    if (!parse(env, info, &c, p, 6, i, 3, true)) return nullptr;
    if (check(env, c, brik_matmul_t_i8(c, (const int8_t*)p[0], (const float*)p[1], (const int8_t*)p[2], (const float*)p[3], (const float*)p[4],
                                       (float*)p[5], i[0], i[1], i[2])))
        return nullptr;
    return undefined(env);
}

// (ctx, x, xScales, src, rowOff, w, wScales, ySorted, xRows, k, E, rows, K, N)
napi_value MoeMatmulI8(napi_env env, napi_callback_info info)
{
    brik_ctx* c; void* p[7]; int32_t i[6];
    if (!parse(env, info, &c, p, 7, i, 6, true)) return nullptr;
    if (check(env, c, brik_moe_matmul_t_i8(c, (const int8_t*)p[0], (const float*)p[1], i[0], (const int32_t*)p[2], i[1], (const int32_t*)p[3],
                                           (const int8_t*)p[4], (const float*)p[5], (float*)p[6], i[2], i[3], i[4], i[5])))
        return nullptr;
    return undefined(env);
}

napi_value Init(napi_env env, napi_value exports)
{
    const napi_property_descriptor props[] = {
        {"moeRoute", nullptr, MoeRoute, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"moeRouteGrad", nullptr, MoeRouteGrad, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"moeSort", nullptr, MoeSort, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"moeDispatch", nullptr, MoeDispatch, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"moeCombine", nullptr, MoeCombine, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"moeCombineGrad", nullptr, MoeCombineGrad, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"quantizeI8", nullptr, QuantizeI8, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"matmulI8", nullptr, MatmulI8, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
        {"moeMatmulI8", nullptr, MoeMatmulI8, nullptr, nullptr, nullptr, napi_enumerable, nullptr},
    };
    napi_define_properties(env, exports, sizeof(props) / sizeof(props[0]), props);
    return exports;
}

}  // namespace

NAPI_MODULE(NODE_GYP_MODULE_NAME, Init)
