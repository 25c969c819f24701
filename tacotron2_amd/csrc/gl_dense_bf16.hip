// The 16-bit products of the dense layers on bf16 operands.
#include "gl_mm16_launch.h"

template int gl_mm16<gl_bf16, gl_bf16, gl_bf16, 1>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
template int gl_mm16<gl_bf16, float, gl_bf16, 1>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
template int gl_mm16<gl_bf16, gl_bf16, gl_bf16, 2>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
