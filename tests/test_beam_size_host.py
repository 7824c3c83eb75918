"""Beam sizes that are none are refused wherever one is given, before anything is read or run: no GPU needed."""
import pytest


class Untouched:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was asked for")


@pytest.mark.parametrize("bad", [0, -1, 65])
def test_prediction_and_evaluation_refuse_it(bad, tmp_path):
    from multimodal_seq2seq_gscan_amd.predict import beam_decode, evaluate, evaluate_sums, predict
    model, data = Untouched(), Untouched()
    for call in (lambda: next(predict(data, model, 5, 0, 1, 2, beam_size=bad)),
                 lambda: evaluate(data, model, 5, 0, 1, 2, beam_size=bad),
                 lambda: evaluate_sums(data, model, 5, 0, 1, 2, beam_size=bad),
                 lambda: beam_decode(model, data, [3], data, 1, 2, 5, bad)):
        with pytest.raises(ValueError, match="beam_size must be 1 to 64"):
            call()


@pytest.mark.parametrize("bad", [0, -1, 65])
@pytest.mark.parametrize("mode", ["train", "test"])
def test_the_command_line_refuses_it(bad, mode, tmp_path):
    from multimodal_seq2seq_gscan_amd.__main__ import main, parser
    flags = vars(parser.parse_args(["--mode", mode, "--synthetic_data", "--beam_size", str(bad), "--output_directory", str(tmp_path)]))
    with pytest.raises(ValueError, match="beam_size must be 1 to 64"):
        main(flags)


def test_training_refuses_it_before_it_reads_the_data():
    from multimodal_seq2seq_gscan_amd.train import train_on_dataset
    with pytest.raises(ValueError, match="beam_size must be 1 to 64"):
        train_on_dataset("no such file", "no such directory", False, "", "", 8, 1, 1, 1, 5, "", beam_size=0)
