// Packed cross-attention of bf16 operands (a file a type: they compile side by side).
#define VFL_CROSS_KERNEL
#include "cross_attention.h"

int vfl::launch_cross_bf16(const CrossArgs &a, int ks, hipStream_t stream) {
  return launch_cross<VFL_BFLOAT16>(a, ks, stream);
}
