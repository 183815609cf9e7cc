"""A test that forces one of the library's kernels and fails before it lets go leaves nothing forced behind."""
import conftest


class Fake:
    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        return lambda *args: self.calls.__setitem__(name, args)


def test_every_hook_is_released():
    from yolo11_cu_b200 import runtime
    fake = Fake()
    conftest.release_hooks(fake)
    hooks = {n: len(runtime._SIGS[n][1]) for n in runtime._SIGS if n.startswith("yk_test_") and n != "yk_test_inject"}
    assert fake.calls == {n: (0,) * args for n, args in hooks.items()}


def test_the_release_runs_behind_every_test(request):
    assert "hooks_end_with_their_test" in request.fixturenames
