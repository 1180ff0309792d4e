// q4_dev.h -- layout of the 4-bit read-out's records (readout.hip, classifier.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/htm_amd.h"

#define Q4_BLK 32          // outputs of one 16-byte block of codes
#define Q4_MAX_INPUTS 65536
#define Q4_MAX_SOFTMAX 1024

struct Q4Dims {
    int32_t nm, ni, nh, no, group;
    int32_t nblk;      // blocks per head
    int32_t ngrp;      // scales per head
    uint32_t pitch;    // bytes of one input's record
    uint32_t scales;   // offset of the scales in it
};

// HTM_OK and *d filled, or HTM_E_INVALID (message set)
int q4_dims(const htm_q4_shape* s, const char* who, Q4Dims* d);
int q4_quantise_launch(const Q4Dims& d, const void* w, int32_t dtype, int64_t ms, int64_t is, int64_t hs, void* rec,
                       int32_t* bad, hipStream_t st);
