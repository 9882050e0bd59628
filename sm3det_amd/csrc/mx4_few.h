// mx4_few.h -- interface of mx4_few.hip
#pragma once
#include "common.h"

namespace sm3x {

struct Few {
  const void* x;  // (S, k), ldx elements between rows
  long ldx;
  const unsigned char* codes;
  const unsigned char* scales;
  int k, kp, cols, G, S;
  const int* offsets;
  const void* bias;
  int bias_type, act, out_type;
  void* out;
};
int launch_few(const Few& P, int type, long row_tiles, hipStream_t st);

}  // namespace sm3x
