// readout_rows.hip -- operators of the read-out that work on a row at a time (pink_hip_readout_norm*, pink_hip_readout_distil* of
// include/pink_hip.h): layer norm and its gradients, and an image's loss against its teacher and its label.
#include "readout_handle.h"

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "readout_tile.inc"
#include "readout_norm.inc"
#include "readout_distil.inc"

namespace {

constexpr uint32_t kMaxRows = 0x7fffffffu;

bool is_bfloat(const pink_hip_readout *r) { return r->cfg.element == PINK_HIP_ELEMENT_BFLOAT; }

}  // namespace

extern "C" {

int pink_hip_readout_norm(pink_hip_readout *r, const void *x, uint32_t images, uint32_t width, uint64_t x_stride, const void *weight,
                          const void *bias, float epsilon, void *y, uint64_t y_stride, float *mean, float *scale)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, width == 0 || width > kMaxSize, "pink_hip_readout_norm: width must be between 1 and 1048576");
    REFUSE(r, !(epsilon >= 0.0f) || std::isinf(epsilon), "pink_hip_readout_norm: epsilon must be 0 or larger, and finite");
    x_stride = x_stride ? x_stride : width;
    y_stride = y_stride ? y_stride : width;
    REFUSE(r, x_stride < width || y_stride < width || (x == y && x_stride != y_stride && images > 1), "pink_hip_readout_norm: rows overlap");
    if (images == 0) return PINK_HIP_OK;
    REFUSE(r, !x || !y, "pink_hip_readout_norm: null argument");
    REFUSE(r, images > kMaxRows, "too many images for one call");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    NormArgs g = {};
    g.x = x;
    g.weight = weight;
    g.bias = bias;
    g.y = y;
    g.mean = mean;
    g.scale = scale;
    g.x_stride = x_stride;
    g.y_stride = y_stride;
    g.rows = images;
    g.width = width;
    g.epsilon = epsilon;
    g.over_width = 1.0f / (float)width;
    return is_bfloat(r) ? norm<Bfloat>(r, g) : norm<float>(r, g);
}

int pink_hip_readout_norm_reserve(pink_hip_readout *r, uint32_t images, uint32_t width)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, width == 0 || width > kMaxSize, "pink_hip_readout_norm: width must be between 1 and 1048576");
    REFUSE(r, images > kMaxRows, "too many images for one call");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    uint32_t parts = 0;                                    // (few rows may have a block each, and so more parts than more rows)
    for (const uint32_t rows : {images, std::min(images, kNormFewLong), std::min(images, kNormFew)}) parts = std::max(parts, norm_parts(rows, width));
    return grow(r, (size_t)parts * 2 * width * 4);
}

int pink_hip_readout_norm_backward(pink_hip_readout *r, const void *x, uint32_t images, uint32_t width, uint64_t x_stride,
                                   const void *weight, const float *mean, const float *scale, const void *dy, uint64_t dy_stride,
                                   const void *residual, uint64_t residual_stride, void *dx, uint64_t dx_stride, void *dweight, void *dbias)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, width == 0 || width > kMaxSize, "pink_hip_readout_norm: width must be between 1 and 1048576");
    x_stride = x_stride ? x_stride : width;
    dy_stride = dy_stride ? dy_stride : width;
    dx_stride = dx_stride ? dx_stride : width;
    residual_stride = residual_stride ? residual_stride : width;
    REFUSE(r, x_stride < width || dy_stride < width || dx_stride < width || residual_stride < width, "pink_hip_readout_norm_backward: rows overlap");
    REFUSE(r, images > 1 && dx && ((dx == dy && dx_stride != dy_stride) || (dx == residual && dx_stride != residual_stride)),
           "pink_hip_readout_norm_backward: rows overlap");
    REFUSE(r, images && (!x || !mean || !scale || !dy), "pink_hip_readout_norm_backward: null argument");
    REFUSE(r, images > kMaxRows, "too many images for one call");
    if (!dweight && !dbias && (!dx || images == 0)) return PINK_HIP_OK;
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    NormArgs g = {};
    g.x = x;
    g.weight = weight;
    g.dy = dy;
    g.residual = residual;
    g.y = dx;
    g.mean = const_cast<float *>(mean);
    g.scale = const_cast<float *>(scale);
    g.x_stride = x_stride;
    g.y_stride = dx_stride;
    g.dy_stride = dy_stride;
    g.residual_stride = residual_stride;
    g.rows = images;
    g.width = width;
    g.over_width = 1.0f / (float)width;
    return is_bfloat(r) ? norm_backward<Bfloat>(r, g, dweight, dbias) : norm_backward<float>(r, g, dweight, dbias);
}

int pink_hip_readout_distil(pink_hip_readout *r, const pink_hip_readout_distil_config *c, const void *logits, uint32_t images, uint64_t logit_stride,
                            const int32_t *teacher_class, const float *teacher_logits, const float *teacher_normaliser, const int32_t *label,
                            const float *image_weights, float *losses, void *gradients, uint64_t gradient_stride)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, !c, "pink_hip_readout_distil: null argument");
    REFUSE(r, c->classes == 0 || c->classes > kMaxSize, "pink_hip_readout_distil: classes must be between 1 and 1048576");
    REFUSE(r, c->places > kMaxPlaces, "pink_hip_readout_distil: at most 1024 places");
    // (of a subnormal one the inverse is past float32)
    REFUSE(r, !(c->temperature >= FLT_MIN) || std::isinf(c->temperature), "pink_hip_readout_distil: temperature must be 2^-126 or larger, and finite");
    REFUSE(r, !std::isfinite(c->teacher_weight) || !std::isfinite(c->label_weight), "pink_hip_readout_distil: weights must be finite");
    logit_stride = logit_stride ? logit_stride : c->classes;
    gradient_stride = gradient_stride ? gradient_stride : c->classes;
    REFUSE(r, logit_stride < c->classes || gradient_stride < c->classes, "pink_hip_readout_distil: rows overlap");
    if (images == 0) return PINK_HIP_OK;
    REFUSE(r, !logits || (c->places && (!teacher_class || !teacher_logits)), "pink_hip_readout_distil: null argument");
    REFUSE(r, images > kMaxRows, "too many images for one call");
    if (!losses && !gradients) return PINK_HIP_OK;
    if (gradients) {
        const uintptr_t from = (uintptr_t)logits, to = (uintptr_t)gradients;
        const size_t e = element_bytes(r), read = ((images - 1) * logit_stride + c->classes) * e, written = ((images - 1) * gradient_stride + c->classes) * e;
        REFUSE(r, from < to + written && to < from + read, "pink_hip_readout_distil: gradients may not lie where logits do");
    }
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    DistilArgs g = {};
    g.logits = logits;
    g.gradients = gradients;
    g.place_class = teacher_class;
    g.place_logits = teacher_logits;
    g.normaliser = teacher_normaliser;
    g.label = label;
    g.image_weights = image_weights;
    g.losses = losses;
    g.logit_stride = logit_stride;
    g.gradient_stride = gradient_stride;
    g.images = images;
    g.classes = c->classes;
    g.teacher_weight = c->teacher_weight;
    g.label_weight = c->label_weight;
    // (without a teacher powers are needed at temperature 1 alone)
    const bool teach = c->teacher_weight != 0.0f && (c->places || teacher_normaliser);
    g.places = teach ? c->places : 0;
    g.temperature = teach ? c->temperature : 1.0f;
    if (!teach) g.teacher_weight = 0.0f;
    return is_bfloat(r) ? distil<Bfloat>(r, g) : distil<float>(r, g);
}

int pink_hip_readout_distil_reserve(pink_hip_readout *r, uint32_t images, uint32_t classes)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, classes == 0 || classes > kMaxSize, "pink_hip_readout_distil: classes must be between 1 and 1048576");
    REFUSE(r, images > kMaxRows, "too many images for one call");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    size_t bytes = 0;                                      // (fewer images may be split where more are not)
    for (const uint32_t n : {images, std::min(images, kDistilFew)})
        bytes = std::max(bytes, is_bfloat(r) ? distil_bytes<Bfloat>(n, classes) : distil_bytes<float>(n, classes));
    return grow(r, bytes);
}

}  // extern "C"
