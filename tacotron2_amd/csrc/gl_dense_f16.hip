// The 16-bit products of the dense layers on f16 operands.
#include "gl_mm16_launch.h"

template int gl_mm16<gl_f16, gl_f16, gl_f16, 1>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
template int gl_mm16<gl_f16, float, gl_f16, 1>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
template int gl_mm16<gl_f16, gl_f16, gl_f16, 2>(const gl_operand&, const gl_operand&, gl_epilogue, long long, int, long long, float*, hipStream_t);
