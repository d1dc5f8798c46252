// What the translation units of libprosim_hip.so share on the host side.
#ifndef PS_INTERNAL_H
#define PS_INTERNAL_H

namespace ps {
// Store the message ps_last_error() returns (per thread; printf form, cut at 511 characters) and hand `code` back.  Never throws: a C entry
// may end with it.  Defined in prosim_hip.hip.
__attribute__((format(printf, 2, 3))) int set_error(int code, const char* fmt, ...) noexcept;
}  // namespace ps

#endif  // PS_INTERNAL_H
