// What norm.cu shares with the rest of the library.
#pragma once

namespace ksmm {

constexpr int kNormWaits = 96;  // codes of norm.cu's bounded waits: 96 to 98

}  // namespace ksmm
