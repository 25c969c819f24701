// The products of the dense layers on float32 operands: gradients in three bfloat16 planes, the rest in two of f16.
#include "gl_mm16_launch.h"

template int gl_mm16<gl_bf16, float, float, 6>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
template int gl_mm16<gl_f16, float, float, 3>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
