// block_quant.h -- matrices held in 8 bits: e4m3 payloads with a scale byte for every 128 columns
// of one row or of 128 rows.  Host checks and device helpers shared by their entry points.
#pragma once
#include "quant_cache.h"

namespace sandy_hip {

constexpr int kQuantBlock = 128;

// A matrix [batch, rows, k] in 8 bits, checked.
struct QuantMat {
    uint8_t* payload;
    uint8_t* scales;      // [batch, scale_rows, blocks], contiguous
    int64_t batch, rows, k;
    int64_t pitch;        // bytes from a row to the next
    int64_t batch_pitch;  // bytes from a matrix to the next
    int64_t scale_rows;   // rows, or one for every 128 of them
    int64_t blocks;       // ceil(k / 128)
    int32_t shift;        // row >> shift is its row of scales: 0 or 7
};

// Checks payload [.., rows, k] and scales [.., rows or ceil(rows / 128), ceil(k / 128)] (both U8, rank
// 2 or 3) and fills *m.  `what` begins every message.
inline int check_quant_matrix(const SandyTensor* payload, const SandyTensor* scales, const char* what, Err e, QuantMat* m) {
    if (!valid_rank(payload) || !valid_rank(scales)) return fail(e, SANDY_ERR_INVALID, "%s requires payloads and scales", what);
    const int r = payload->rank;
    if (payload->dtype != SANDY_U8 || scales->dtype != SANDY_U8 || (r != 2 && r != 3) || scales->rank != r)
        return fail(e, SANDY_ERR_INVALID, "%s payloads and scales must be u8 of rank 2 or 3", what);
    for (int i = 0; i < r; i++)
        if (payload->dims[i] < 0) return fail(e, SANDY_ERR_INVALID, "%s expects static dimensions", what);
    *m = QuantMat{};
    m->batch = r == 3 ? payload->dims[0] : 1;
    m->rows = payload->dims[r - 2];
    m->k = payload->dims[r - 1];
    if (m->batch > INT32_MAX || m->rows > INT32_MAX || m->k > (int64_t{1} << 30))
        return fail(e, SANDY_ERR_UNSUPPORTED, "%s matrix too large", what);
    m->blocks = (m->k + kQuantBlock - 1) / kQuantBlock;
    m->scale_rows = scales->dims[r - 2];
    const bool each = m->scale_rows == m->rows, tiled = m->scale_rows == (m->rows + kQuantBlock - 1) / kQuantBlock;
    if ((r == 3 && scales->dims[0] != m->batch) || scales->dims[r - 1] != m->blocks || !(each || tiled))
        return fail(e, SANDY_ERR_INVALID, "%s scales must be [.., rows or ceil(rows / 128), ceil(k / 128)]", what);
    m->shift = each ? 0 : 7;
    if (!contiguous(*scales)) return fail(e, SANDY_ERR_INVALID, "%s scales must be contiguous", what);
    if (m->batch == 0 || m->rows == 0 || m->k == 0) return SANDY_OK;
    if (!payload->data || !scales->data) return fail(e, SANDY_ERR_INVALID, "%s payloads or scales are null", what);
    m->payload = static_cast<uint8_t*>(base_ptr(*payload));
    m->scales = static_cast<uint8_t*>(base_ptr(*scales));
    if (m->k > 1 && payload->strides[r - 1] != 1) return fail(e, SANDY_ERR_INVALID, "%s payload rows must have unit inner stride", what);
    // a stride of a dimension of one element says nothing
    m->pitch = m->rows > 1 ? payload->strides[r - 2] : (m->k + 15) / 16 * 16;
    m->batch_pitch = m->batch > 1 ? payload->strides[0] : 0;
    if (m->pitch < m->k || m->pitch > (int64_t{1} << 40) ||
        (m->batch > 1 && (m->batch_pitch < (m->rows - 1) * m->pitch + m->k || m->batch_pitch > INT64_MAX / m->batch)))
        return fail(e, SANDY_ERR_INVALID, "%s payload rows must follow one another without overlap", what);
    return SANDY_OK;
}

// What the products ask for beyond that: 16-byte pieces of every row.
inline bool quant_rows_aligned(const QuantMat& m) {
    return ((reinterpret_cast<uintptr_t>(m.payload) | static_cast<uintptr_t>(m.rows > 1 ? m.pitch : 0) |
             static_cast<uintptr_t>(m.batch > 1 ? m.batch_pitch : 0)) & 15) == 0;
}

} // namespace sandy_hip
