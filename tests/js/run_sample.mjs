/**
 * Sampled generation through HipPetitGPT with given random numbers.
 *   node run_sample.mjs <model.pgw> <spec.json>   -> prints one JSON line
 * spec: { prompt: [...], maxNewTokens, temperature, topK, topP, minP, numbers: [...] }
 */
import fs from "fs";
import { parsePgw } from "../../microllm-lab_amd/js/weights.mjs";
import { HipPetitGPT } from "../../microllm-lab_amd/js/engine.mjs";

async function main() {
  const [, , pgwPath, specPath] = process.argv;
  const spec = JSON.parse(fs.readFileSync(specPath, "utf8"));
  const model = new HipPetitGPT(parsePgw(fs.readFileSync(pgwPath)));
  let at = 0;
  const res = await model.generate(spec.prompt, Object.assign({}, spec, {
    mode: "sample",
    random: () => spec.numbers[at++],
  }));
  model.forwardPrompt(spec.prompt);
  const drawn = model.draw(spec.numbers[0], spec);
  model.decodeChain(1, 1, -1, null);
  let refused = null;
  try {
    model.draw(0.5);
  } catch (e) {
    refused = String(e.message);
  }
  model.destroy();
  console.log(JSON.stringify({ generatedIds: res.generatedIds, mode: res.mode, used: at, drawn, refused }));
}

main().catch((e) => {
  console.error(e && e.stack ? e.stack : String(e));
  process.exit(1);
});
