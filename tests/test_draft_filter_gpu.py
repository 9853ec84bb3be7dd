"""Top-k on the scores of a drafted step: what ``Generator.generate_ragged`` draws behind the first token is among the k likeliest of the model's logits, up to what two
routes' logits differ (twice the tolerance of ``_close``, as in ``test_draft_model_gpu.py``)."""
import pytest
import torch

from test_core_gpu import DEV
from test_draft_model_gpu import ints
from test_paged_model_gpu import alone, generator, model_and_prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("record_steps", [False, True])
@pytest.mark.parametrize("k", [1, 3])
def test_drafted_steps_draw_from_what_a_filter_leaves(k, record_steps):
    model, prompts, _ = model_and_prompts([6], seed=2)
    B = 256
    g = torch.Generator(device=DEV).manual_seed(4)

    def drafts(seen, lens):
        return torch.randint(2, 96, (seen.size(0), 9), generator=g, device=DEV), ints(*[-1] * 4, *[0, 1, 2, 3, 4])
    gen = generator(model, temperature=1.5, top_k=k, seed=12)
    tokens = gen.generate_ragged([prompts[0]] * B, 3, record_steps=record_steps, drafts=drafts)
    beyond = 0.0                                         # draws that no filter would have sent elsewhere
    with torch.inference_mode():
        for line in tokens.unique(dim=0).tolist():
            times = int((tokens == torch.tensor(line, device=DEV)).all(1).sum())
            logits = alone(model, prompts[0], [torch.tensor(t, device=DEV) for t in line[:2]])
            for i, row in enumerate(logits[:3]):
                if 1 in line[:i]:
                    continue
                row = row[:96].float()
                least = float(row.topk(k).values[-1]) - 2 * 3e-2 * max(float(row.abs().max()), 1.0)
                assert float(row[line[i]]) >= least, (line, i)
                if i > 0:
                    beyond += times * float(torch.softmax(row / 1.5, -1)[row < least].sum())
    print(f"{beyond:.1f} of {2 * B} draws expected elsewhere without the filter", flush=True)
    assert beyond > 30
