"""Building the oracle where the reference is not there."""
import oracle


def test_an_empty_reference_folder_is_no_reference(tmp_path, monkeypatch):
    """The oracle is built, the reference's own library is left alone, and nothing fails."""
    calls = []
    monkeypatch.setenv("MME_REFERENCE_ROOT", str(tmp_path))
    monkeypatch.setattr(oracle.subprocess, "check_call", calls.append)
    oracle.build(with_ref=True)
    assert [c[-1] for c in calls] == ["oracle"]
