// A step of stream_rows (paged_attention.hpp), which includes it in its loops: the scores of 16 keys, their weights, and what these add to the rows' results, with the next step's rows asked for on the way.
// STEP_FOLLOWS: whether there is a next step, a condition or a constant.  (In the loop's own scope: as a lambda or a function with references it costs 2 to 8 %.)
look(kb, k, v, missing);
f32x4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
for (int b = 0; b < 4 * BLOCKS; ++b) {
  f32x4 x = k[b];
  if (size != DPAD && 16 * b + 4 * g >= size) x = f32x4{0, 0, 0, 0};
  s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[0], q[b][0], s0, 0, 0, 0);
  s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[1], q[b][1], s1, 0, 0, 0);
  s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[2], q[b][2], s0, 0, 0, 0);
  s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[3], q[b][3], s1, 0, 0, 0);
}
f32x4 s = s0 + s1;
if constexpr (SHAPED) {
  float formed[4] = {s[0], s[1], s[2], s[3]};
  shape.apply(formed, kb + 4 * (int)g, [](int i) { return i; });
  s = f32x4{formed[0], formed[1], formed[2], formed[3]} * shape.unit;
}
const bool more = STEP_FOLLOWS;
const Held next_pages = pages_of();
if (more) load_keys(kb + STEP, next_pages);
const bool edge = __any(missing != 0) || kb < t.all_low || kb + 16 > t.all_high;
unsigned foreign = 0;  // values that are not finite, of keys that some row does not see
if (edge) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = kb + 4 * (int)g + i;
    const bool there = (missing >> i & 1) == 0;
    s[i] = there && key >= t.row_low && key < t.row_high ? s[i] : -INFINITY;
    const bool none = !there || key < t.low || key >= t.high;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool odd = (__float_as_uint(v[i][b][j]) & 0x7f800000u) == 0x7f800000u;
        foreign |= odd && !none ? 1u : 0u;
        v[i][b][j] = none || odd ? 0.0f : v[i][b][j];
      }
  }
}
const float top = across_groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
if (__any(top > m)) {
  const float next = fmaxf(m, top);
  const float f = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
  m = next;
  l *= f;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[b][j] *= f;
}
const float zero = m == -INFINITY ? 0.0f : m;
float e[4];
#pragma unroll
for (int i = 0; i < 4; ++i) {
  e[i] = __builtin_amdgcn_exp2f(s[i] - zero);
  l += e[i];
}
#pragma unroll
for (int i = 0; i < 4; ++i)
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][b][j], e[i], o[b][j], 0, 0, 0);
if (edge && __any(foreign != 0)) {
  // Rare: a key with an infinity or a NaN among its values that only some of the rows see.  A product over all rows would hand
  // 0 x infinity to the others, so it went in as zeros and is added here, to the rows that see it.
  for (int at = 0; at < 16; ++at) {
    const int key = kb + at;
    const unsigned from = c + 16 * (at / 4);
    const float e0 = __shfl(e[0], (int)from, 64), e1 = __shfl(e[1], (int)from, 64), e2 = __shfl(e[2], (int)from, 64), e3 = __shfl(e[3], (int)from, 64);
    const float weight = at % 4 == 0 ? e0 : at % 4 == 1 ? e1 : at % 4 == 2 ? e2 : e3;
    const unsigned index = p.cache.page_size.quotient((unsigned)key), inside = (unsigned)key - index * p.cache.page_size.d;
    const int held = page_of(p, table, index);
    if (held < 0 || key < t.row_low || key >= t.row_high) continue;
    const float* row = values + held * p.cache.page + inside * p.cache.row;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned d = 64 * b + 4 * (4 * g + i) + j;
          const float x = d < size ? row[d] : 0.0f;
          if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) o[b][j][i] += weight * x;
        }
  }
}
if (more) {
  load_values(kb + STEP, next_pages);
  if (kb + 2 * STEP < end) ask_pages(kb + 2 * STEP);
}
#undef STEP_FOLLOWS
