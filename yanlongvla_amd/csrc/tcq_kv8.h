// The 8-bit key / value cache shared by its kernels (tcq_kv8.hip). Per sequence and KV head, blocks of 64 tokens:
//   k8    64 D bytes a block, token t, dim d at ((t / 16 * D / 16 + d / 16) * 16 + t % 16) * 16 + d % 16 (the token-block layout): the 16
//         bytes of a lane are the INT8 MFMA fragment of 16 keys x 64 dims, a wave's load one contiguous KiB;
//   v8    64 D bytes, dim d, token t at ((d / 16 * 4 + t % 16 / 4) * 16 + d % 16) * 16 + t / 16 * 4 + t % 4: the fragment of 16 dims x 64
//         keys, the keys in the order in which the score product leaves its rows in the lanes, so that neither the values nor the
//         probabilities ever cross lanes;
//   scale (K, V) FP32 a block;
//   tail  the 16-bit rows of the newest two blocks, (block % 2, K | V, 64, D).
#pragma once
#include "tcq_device.h"
#include "tcq_launch.h"

constexpr int KB = 64;           // tokens per block

__device__ __forceinline__ float kv_value(u16 b, bool bf16) { return bf16 ? bf16_to_f32(b) : f16_to_f32(b); }
