"""Isolated-word classifier with the reference's interface
(src/loe_speech_recognition/model_collection.py): every word model scores the utterance with
its own left-to-right Viterbi pass and the best score wins.  All models of the collection run
side by side in one wavefront per utterance (lsr_decode_chain_batch with one start state per
model and no transitions between models)."""
from __future__ import annotations

import os
from dataclasses import dataclass, field
from typing import List, Optional, Tuple

import numpy as np

from . import _native
from .hidden_markov_model import HiddenMarkovModel, stack_gaussians
from .scores import sample_scores, top_scores
from .ti_digits import TI_DIGITS_LABELS


@dataclass
class ModelCollection:
    num_of_states: int = field(default=5)
    dim_of_feature: int = field(default=39)

    _models: List[HiddenMarkovModel] = field(default_factory=list)

    def __getstate__(self):
        state = dict(self.__dict__)
        state.pop("_dev_cache", None)
        return state

    def _bind(self):
        eng = _native.get_engine()
        cache = self.__dict__.get("_dev_cache")
        # the upload belongs to these very parameter objects: a replaced model (or a re-estimated one, which
        # gets new lists) invalidates it even when the number of models is unchanged
        srcs = [(m._multivariate_normals, m._log_transition_probs) for m in self._models]
        if cache is None or len(cache["srcs"]) != len(srcs) or \
                any(a[0] is not b[0] or a[1] is not b[1] for a, b in zip(cache["srcs"], srcs)):
            sizes = [m.num_of_states for m in self._models]
            if sum(sizes) > _native.NARROW_STATES:
                raise ValueError(f"{sum(sizes)} states in the collection; scoring all models side by side handles "
                                 f"{_native.NARROW_STATES}")
            band = np.concatenate([m._log_transition_probs.band() for m in self._models], axis=1)
            ends = np.cumsum(sizes)
            start = np.zeros(int(ends[-1]), dtype=np.uint8)
            start[np.concatenate([[0], ends[:-1]])] = 1
            cache = {"srcs": srcs, "token": _native.new_token(),
                     "model": stack_gaussians([g for m in self._models for g in m._multivariate_normals]),
                     "band": band, "start": start, "last": ends - 1}
            self.__dict__["_dev_cache"] = cache
        eng.set_model(cache["token"], *cache["model"])
        return eng, cache

    def scores_device(self, signals):
        """Device tensor float32 [B, n_models]: each model's Viterbi score, left on the device."""
        eng, c = self._bind()
        fb = signals if isinstance(signals, _native.FeatureBatch) else eng.feature_batch(signals)
        n = c["start"].shape[0]
        d_off, total, d_ids, d_band, d_start = eng.uniform_chains(c["token"], fb.n, np.arange(n, dtype=np.int32), c["band"],
                                                                  c["start"])
        _, _, final = eng.decode_chain_device(fb, d_off, total, d_ids, d_band, d_start, want_paths=False, want_final=True)
        if "d_last" not in c:
            c["d_last"] = eng.to_device(np.asarray(c["last"], dtype=np.int64))
        return final[:, c["d_last"]]

    def scores_batch(self, signals) -> np.ndarray:
        """float32 [B, n_models]: each model's Viterbi score (hidden_markov_model.py:160-198)."""
        return self.scores_device(signals).cpu().numpy()

    def predict_batch(self, signals) -> List[str]:
        scores = self.scores_batch(signals)
        # model_collection.py:26-28 sorts (label, score) pairs with a stable sort, reverse=True:
        # among equal scores the model that comes first in the collection wins = first argmax
        names = [str(m) for m in self._models]
        return [names[i] for i in np.argmax(scores, axis=1).tolist()]

    def predict(self, signal: np.ndarray) -> str:
        return self.predict_batch([signal])[0]

    def nbest_batch(self, signals, n: int) -> List[List[Tuple[str, np.float32]]]:
        """The ``n`` best (label, score) pairs of every utterance, best first, models with equal scores in the order of
        the collection: the head of the sorted list of which ``predict`` returns the first label (model_collection.py:26-28).
        A model that cannot score an utterance (-inf) is left out."""
        values, index, _ = top_scores(self.scores_device(signals), n)
        names = [str(m) for m in self._models]
        return [[(names[i], v) for i, v in zip(row_i, row_v) if i >= 0]
                for row_i, row_v in zip(index.cpu().numpy().tolist(), values.cpu().numpy())]

    def sample_batch(self, signals, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> List[Optional[str]]:
        """A label per utterance drawn in proportion to ``exp(score / temperature)`` among the models that the cuts leave
        (see ``sample_scores``), with the uniform numbers given - for instance pseudo-labels that keep the recogniser's
        doubt.  Scores are log-likelihoods of whole utterances; a temperature of the order of the utterances' frames makes
        them comparable per frame.  None where no model can score the utterance."""
        scores = self.scores_device(signals)
        uniform = _native.get_engine().to_device(np.asarray(uniform, dtype=np.float32))
        index, _ = sample_scores(scores, uniform, temperature, top_k, top_p, min_p)
        names = [str(m) for m in self._models]
        return [names[i] if i >= 0 else None for i in index.cpu().numpy().tolist()]

    @classmethod
    def load_from_files(cls, folder_path: str):
        mc = cls()
        for label in TI_DIGITS_LABELS:
            mc._models.append(HiddenMarkovModel.from_folder(os.path.join(folder_path, f"{label}")))
        return mc
