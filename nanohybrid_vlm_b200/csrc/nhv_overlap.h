// Whether two operands of a call share memory (on the host, from what the call was given).
#pragma once

// Rows of `bytes` bytes each, `pitch` bytes apart from `at` on.
struct NhvRows {
  long long at, rows, pitch, bytes;
};

// Exact: columns of one buffer side by side do not meet although their ranges do.  A handful of operations where the ranges are
// apart (nearly every call) or the pitches equal; else a turn for each row of the operand with fewer.
inline bool nhv_rows_meet(NhvRows a, NhvRows b) {
  if (a.rows <= 0 || b.rows <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
  if (a.pitch == 0) a.rows = 1;
  if (b.pitch == 0) b.rows = 1;
  // the first place of a whole step from `first` on that lies behind `behind`
  auto step_behind = [](long long first, long long pitch, long long behind) -> long long {
    const long long d = behind - first;
    return d < 0 ? -(-d - 1) / pitch : d / pitch + 1;
  };
  if (a.rows == 1) a.pitch = b.rows == 1 ? 1 : b.pitch;      // a single row's may be anything
  if (b.rows == 1) b.pitch = a.pitch;
  if (a.at + (a.rows - 1) * a.pitch + a.bytes <= b.at || b.at + (b.rows - 1) * b.pitch + b.bytes <= a.at) return false;
  if (a.pitch == b.pitch) {
    // row i of a and row i + k of b: their distance is b.at - a.at + k * pitch
    long long k = step_behind(b.at - a.at, a.pitch, -b.bytes);
    if (k < 1 - a.rows) k = 1 - a.rows;
    return k < b.rows && b.at - a.at + k * a.pitch < a.bytes;
  }
  if (b.rows < a.rows) {
    const NhvRows c = a;
    a = b;
    b = c;
  }
  for (long long i = 0; i < a.rows; ++i) {
    const long long from = a.at + i * a.pitch;
    long long j = step_behind(b.at, b.pitch, from - b.bytes);      // the first row of b that ends behind `from`
    if (j < 0) j = 0;
    if (j < b.rows && b.at + j * b.pitch < from + a.bytes) return true;
  }
  return false;
}
