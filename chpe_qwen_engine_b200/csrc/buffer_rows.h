// buffer_rows.h -- which bytes of a caller's strided buffer a call touches, and
// whether two such buffers share one.  Host code only.
#pragma once
#include <cstdint>

namespace chpe {

// A buffer as a call touches it: `n` rows of `width` bytes, `stride` bytes apart.
struct Rows {
  const char* name;
  const void* p;
  int64_t n, stride, width;
  uint64_t end;  // the address behind the last row (0: nothing is touched)

  // stride_: in elements of `size` bytes; not looked at where there is one row
  Rows(const char* name_, const void* p_, int64_t width_, int64_t n_ = 1, int64_t stride_ = 0, int64_t size = 1)
      : name(name_), p(p_), n(n_), stride(p_ && n_ > 1 ? stride_ * size : 0), width(width_) {
    if (stride == 0 && n > 1) n = 1;  // one row for all
    end = p && n > 0 && width > 0 ? first() + uint64_t(n - 1) * uint64_t(stride) + uint64_t(width) : 0;
  }
  uint64_t first() const { return reinterpret_cast<uintptr_t>(p); }

  // Whether a byte of one is a byte of the other.  Rows of one stride that lie side by side (q, k
  // and v of a token) share an extent but no byte.
  bool meets(const Rows& o) const { return first() < o.end && o.first() < end && shares(o); }

 private:
  bool shares(const Rows& o) const {  // of two whose extents meet
    if (n > o.n) return o.shares(*this);
    if (o.n == 1) return true;  // both are one stretch
    // row i here meets row j there if d + j S < i s + w and i s < d + j S + W: of all i at
    // once where the strides are one, else row by row
    typedef __int128 wide;
    const wide d = wide(o.first()) - wide(first());
    auto below = [](wide x, wide y) { return x / y - (x % y < 0); };  // floor of x / y
    const bool one = n == 1 || stride == o.stride;
    for (int64_t i = 0; i < (one ? 1 : n); i++) {
      const wide at = wide(i) * stride - d;  // this row from there's first
      const wide lo = below(at - o.width, o.stride) + 1, hi = below(at + width - 1, o.stride);
      const wide least = one ? 1 - wide(n) : 0, most = o.n - 1;
      if ((lo > least ? lo : least) <= (hi < most ? hi : most)) return true;
    }
    return false;
  }
};
// A pool's rows; one larger than any device's memory is a caller's way to give no limit: what lies in
// it is not known.
inline Rows pool(const char* name, const void* p, uint64_t rows, uint64_t row_bytes) {
  return Rows(name, p, rows <= (1ull << 40) / row_bytes ? int64_t(rows * row_bytes) : 0);
}

}  // namespace chpe
