"""The child process of the scene's live schedule (``stylemesh_amd/schedule.py``)."""
import io
import sys
import time

from stylemesh_amd import schedule as SCH


def test_epoch_lines_are_shown_as_they_come():
    child = ("import sys, time\n"
             "print('set-up', flush=True)\n"
             "for e in range(3):\n"
             "    print(f'epoch {e}: {(e + 1) * 5460} steps, {(e + 1) * 26.0:.1f} s [train loop 25.0 s = 218.4 steps/s, validation + epoch-end hooks 1.0 s]', flush=True)\n"
             "    time.sleep(0.6)\n"
             "print('warning', file=sys.stderr)\n")

    class Clock(io.StringIO):
        def __init__(self):
            super().__init__()
            self.at = []

        def write(self, s):
            if s.startswith("epoch"):
                self.at.append(time.time())
            return super().write(s)
    out = Clock()
    stdout, stderr, rc, wall = SCH.run_cli([sys.executable, "-c", child], echo=out)
    end = time.time()
    assert rc == 0 and "warning" in stderr and stdout.startswith("set-up")
    assert out.getvalue().splitlines() == [s for s in stdout.splitlines() if s.startswith("epoch")] and len(out.at) == 3
    assert end - out.at[0] >= 1.2                       # not held back until the end
    assert [e["views_per_s"] for e in SCH.parse_epochs(stdout)[2]] == [210.0] * 3
    assert SCH.run_cli([sys.executable, "-c", child])[0] == stdout
