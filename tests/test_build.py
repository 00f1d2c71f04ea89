"""What the library's build needs: the default target neither torch nor Python, `python` alone does."""
import os
import subprocess

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mono-qwen27_amd")


def plan(*targets):
    """The commands that a build from scratch would run (nothing is run)."""
    return subprocess.run(["make", "-n", "-B", "-C", PKG, *targets], check=True, capture_output=True, text=True).stdout


def test_the_default_target_needs_no_torch():
    got = plan()
    for name in ("libm27q.so", "libm27q_stream.so", "libm27q_timeline.so"):
        assert "-o " + name in got
    assert "torch" not in got and "python" not in got


def test_the_python_target_builds_the_module():
    assert "-o m27q_torch.so" in plan("python")
