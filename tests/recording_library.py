"""A stand-in for the library that runs nothing: it hands out addresses and keeps what it was called with, so that what a network passes
to which entry point can be looked at without a GPU."""
import bisect
import ctypes as C

from parallelreverseautodiff_b200 import engine as E


class RecordingLibrary:
    def __init__(self):
        self.calls, self.live, self._starts, self._next = [], {}, [], 1 << 20

    def prad_alloc(self, ctx, size, out):
        out._obj.value = self._next
        self.live[self._next] = size
        self._starts.append(self._next)
        self._next += (size + 511) // 256 * 256        # (nothing follows directly behind an allocation)
        return 0

    def prad_free(self, ctx, p):
        del self.live[p.value]
        return 0

    def prad_selective_scan_saved_bytes(self, dt, scan, out):
        s = scan._obj
        out._obj.value = (s.tokens + 7) // 8 * s.dim * s.state * (8 if dt else 4)
        return 0

    def prad_capture_end(self, ctx, out):
        out._obj.value = 1
        return 0

    def __getattr__(self, name):
        if not name.startswith("prad_"):
            raise AttributeError(name)

        def call(*args):
            self.calls.append((name, args))
            return 0

        return call

    def taken(self):
        """The calls since the last look."""
        calls, self.calls = self.calls, []
        return calls

    def touched(self):
        """The allocations that the calls since the last look were given addresses in, in structs too."""
        found = set()
        for _, args in self.taken():
            for a in args[1:]:
                struct = getattr(a, "_obj", None)
                values = [getattr(struct, k) for k, _ in struct._fields_] if isinstance(struct, C.Structure) else [a]
                found.update(self._starts[bisect.bisect(self._starts, v) - 1] for v in values if isinstance(v, int) and v >= 1 << 20)
        return found


def recording_engine():
    e = E.Engine.__new__(E.Engine)
    e.lib, e.ctx, e.device, e.options = RecordingLibrary(), 1, 0, {}
    return e
