// qm_beam_check.h -- what the host can tell of a call of beam search's step: a
// status code and its message before anything is enqueued.  Host code without
// HIP, so that it is tested on the CPU.
#pragma once
#include "qm_beam.h"
#include "qm_kv4_check.h"

namespace qm_beam {

using qm_kv4::Fault;
using qm_kv4::fault;
using qm_kv4::off_grid;

inline Fault check_select(int32_t groups, int32_t beams, int32_t take, int32_t vocab, const float* logits,
                          const float* scores, const int32_t* done, int32_t end_id, const int32_t* parents,
                          const int32_t* tokens, const float* out_scores, const int32_t* out_done) {
    if (groups <= 0 || vocab <= 0)
        return fault(QM_ERR_INVALID_ARG, "qm_beam_select: %d groups, vocab %d", groups, vocab);
    if (beams <= 0 || beams > QMK_BEAM_MAX || take <= 0 || take > QMK_BEAM_MAX)
        return fault(QM_ERR_INVALID_ARG, "qm_beam_select: %d beams, take %d (1 .. %d)", beams, take, QMK_BEAM_MAX);
    if (vocab > QMK_BEAM_VOCAB)
        return fault(QM_ERR_SHAPE, "qm_beam_select: vocab %d (at most %d)", vocab, QMK_BEAM_VOCAB);
    if (groups > QMK_STATE_ROWS / beams)
        return fault(QM_ERR_SHAPE, "qm_beam_select: %d groups of %d beams (at most %d sequences)", groups, beams, QMK_STATE_ROWS);
    if (!logits || !scores || !parents || !tokens || !out_scores)
        return fault(QM_ERR_INVALID_ARG, "qm_beam_select: null pointer");
    if (off_grid(4, {logits, scores, done, parents, tokens, out_scores, out_done}))
        return fault(QM_ERR_INVALID_ARG, "qm_beam_select: device pointers must be 4-byte aligned");
    if (end_id < -1 || end_id >= vocab || (done && end_id < 0))
        return fault(QM_ERR_INVALID_ARG, "qm_beam_select: end_id %d of a vocabulary of %d%s", end_id, vocab,
                     done ? ", with done" : "");
    if (take != beams && (out_scores == scores || (done && out_done == done)))
        return fault(QM_ERR_INVALID_ARG, "qm_beam_select: in place with %d beams, take %d", beams, take);
    return Fault{};
}
inline int32_t slices(int32_t vocab) { return (vocab + QMK_BEAM_SLICE - 1) / QMK_BEAM_SLICE; }
inline size_t select_ws(int64_t rows, int32_t vocab) { return static_cast<size_t>(rows) * slices(vocab) * sizeof(BeamSlice); }

inline Fault check_fork(int32_t buffers, const qm_state_rows* list, int32_t rows, int32_t count, const int32_t* src,
                        const int32_t* dst, const int32_t* result) {
    if (buffers <= 0 || buffers > QMK_STATE_BUFFERS || !list)
        return fault(QM_ERR_INVALID_ARG, "qm_state_fork: %d buffers (1 .. %d)", buffers, QMK_STATE_BUFFERS);
    if (rows <= 0 || rows > QMK_STATE_ROWS)
        return fault(QM_ERR_INVALID_ARG, "qm_state_fork: %d rows (1 .. %d)", rows, QMK_STATE_ROWS);
    if (count <= 0 || count > QMK_STATE_COUNT || count > rows)
        return fault(QM_ERR_INVALID_ARG, "qm_state_fork: %d pairs (1 .. %d, of %d rows)", count, QMK_STATE_COUNT, rows);
    if (!src || !result) return fault(QM_ERR_INVALID_ARG, "qm_state_fork: null pointer");
    if (off_grid(4, {src, dst, result}))
        return fault(QM_ERR_INVALID_ARG, "qm_state_fork: lists and result must be 4-byte aligned");
    for (int32_t i = 0; i < buffers; ++i) {
        const qm_state_rows& b = list[i];
        if (!b.rows_dev) return fault(QM_ERR_INVALID_ARG, "qm_state_fork: buffer %d is null", i);
        if (b.row_bytes <= 0 || b.row_bytes % 16 || b.stride_bytes < b.row_bytes || b.stride_bytes % 16 ||
            b.stride_bytes > INT64_MAX / QMK_STATE_ROWS || off_grid(16, {b.rows_dev}))
            return fault(QM_ERR_INVALID_ARG,
                         "qm_state_fork: buffer %d: rows of %lld bytes, %lld apart (multiples of 16, at a 16-byte aligned address)",
                         i, static_cast<long long>(b.row_bytes), static_cast<long long>(b.stride_bytes));
    }
    return Fault{};
}
// The kernel: rows in registers, up to 8, 32, 64 and 128, or in LDS.
inline int32_t fork_form(int32_t count) { return count <= 8 ? 0 : count <= 32 ? 1 : count <= 64 ? 2 : count <= 128 ? 3 : 4; }
// Bytes of a row that a workgroup takes at a time: what its 256 lanes hold, or
// all rows' fit its LDS.
inline int32_t fork_column(int32_t count) {
    const int32_t form = fork_form(count);
    if (form < 4) return form < 2 ? QMK_STATE_COLUMN : QMK_STATE_COLUMN >> (form - 1);
    int32_t wide = QMK_STATE_COLUMN;
    while (wide * count > QMK_STATE_LDS) wide /= 2;
    return wide;
}
static_assert(QMK_STATE_LDS / QMK_STATE_COUNT >= 16, "a column is at least a vector");

}  // namespace qm_beam
