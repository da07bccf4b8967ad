// OncePerDevice (tvq_once.h): on every device, until it has worked there.
#include <cstdio>

#include "../../tokenvector/inference_b200/csrc/tvq_once.h"

int main() {
    tvq::OncePerDevice once;
    int calls = 0, rc = 0;
    auto set = [&] {
        calls++;
        return rc;
    };
    auto expect = [&](int dev, int want_rc, int want_calls, const char* what) {
        const int got = once(dev, set);
        if (got == want_rc && calls == want_calls) return true;
        std::printf("%s: rc %d, %d calls\n", what, got, calls);
        return false;
    };
    bool ok = expect(0, 0, 1, "the first call") && expect(0, 0, 1, "again on the device") &&
              expect(1, 0, 2, "another device") && expect(1, 0, 2, "again there") && expect(0, 0, 2, "back");
    rc = 5;
    ok = ok && expect(2, 5, 3, "a failure") && expect(2, 5, 4, "is not kept");
    rc = 0;
    ok = ok && expect(2, 0, 5, "nor passed over") && expect(2, 0, 5, "after it worked") &&
         expect(64, 0, 6, "a device beyond the flags") && expect(64, 0, 7, "each time") && expect(-1, 0, 8, "no device");
    return ok ? 0 : 1;
}
