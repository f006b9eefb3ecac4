// The operations of the 8-bit cache called on their own (not from a step plan): everything a call needs in one array of 64-bit
// words, because a call's time on the host is what its caller waits for when the kernels are short.
//
// w0 operation (0 store, 1 attention), w1 stream, w2 status word, w3..w14 the step's first twelve symbols (gb_plan_op.h), w15
// partial tiles or 0, w16 their number, w17 their bias or 0, w18 the operation's floating operand (the bits of a double),
// w19..w38 its operands.  Returns what the operation does.
#include <cstring>

#include "kv8.cuh"

GB_OP(gb_op_kv8_store);
GB_OP(gb_op_kv8_attention);

GB_API int gb_kv8_run(const long long* w) {
  long long sym[GB_SYM_COUNT] = {}, a[24] = {};
  for (int i = 0; i < 12; ++i) sym[i] = w[3 + i];
  for (int i = 0; i < 20; ++i) a[i] = w[19 + i];
  double f[3] = {};
  memcpy(f, w + 18, sizeof(double));
  GbPlanCtx ctx = {};
  ctx.stream = reinterpret_cast<cudaStream_t>(w[1]);
  ctx.status = reinterpret_cast<int*>(w[2]);
  ctx.sym = sym;
  ctx.n_sym = GB_SYM_COUNT;
  ctx.part = reinterpret_cast<const float*>(w[15]);
  ctx.part_splits = (int)w[16];
  ctx.part_bias = reinterpret_cast<const float*>(w[17]);
  const int flags = ctx.part != nullptr ? GB_OP_TAKES_PARTIALS : 0;
  return w[0] == 0 ? gb_op_kv8_store(&ctx, a, f, flags) : gb_op_kv8_attention(&ctx, a, f, flags);
}
