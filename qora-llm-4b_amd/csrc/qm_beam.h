// qm_beam.h -- beam search's step: arguments of the kernels, and the host's
// checks of a call's arguments (host code without HIP, tested on the CPU).
#pragma once
#include <stdint.h>

#define QMK_BEAM_SLICE 1024         // logits of a row that a wave looks at
#define QMK_BEAM_MAX 64             // sequences, and continuations, of a request
#define QMK_BEAM_VOCAB 262144
#define QMK_STATE_BUFFERS 64        // buffers of one call
#define QMK_STATE_ROWS 65536        // rows of a buffer: the LDS bitmap of the destinations
#define QMK_STATE_COUNT 1024        // rows of one call
#define QMK_STATE_COLUMN 4096       // bytes of a row that a workgroup takes at a time, up to 32 rows
#define QMK_STATE_LDS 65536         // bytes that it holds of all rows, more than 128

// A slice's largest logit, the lowest token that has it, and the sum of
// exp(logit - largest).
struct BeamSlice {
    double sum;
    float top;
    int32_t token;
};
struct BeamArgs {
    const float* logits;     // [groups * beams][vocab]
    const float* scores;     // [groups * beams]
    const int32_t* done;     // null or [groups * beams]
    int32_t* parents;        // [groups][take]
    int32_t* tokens;
    float* out_scores;
    int32_t* out_done;       // or null
    BeamSlice* slices;       // workspace [groups * beams][ns]
    int32_t groups, beams, take, vocab, end_id;
    int32_t ns;              // slices of a row
};

struct StateBuffer {
    uint8_t* rows;
    int64_t bytes, stride;
};
struct StateForkArgs {
    const int32_t* src;
    const int32_t* dst;
    int32_t* result;
    int32_t rows, count, buffers;
    int32_t column;                             // bytes of a row taken at a time
    int64_t first[QMK_STATE_BUFFERS + 1];       // columns of the buffers before
    StateBuffer buffer[QMK_STATE_BUFFERS];
};
